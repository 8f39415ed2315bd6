"""The training operators on the device (include/wc_learn.h), through the binding, against plain float64 code.

Tolerances. Statistics and sums are float32: with logits up to 16 in magnitude a row's log-sum is off by a few ulps of 16
(2^-20 each), so log-probabilities, ratios and probabilities are held to 2e-5 (relative, or of the output's largest). An
output in a 16-bit type adds its own rounding: 2^-11 of the value in f16 (2^-24 at least: half its smallest step twice),
2^-8 in bf16. Sums over R rows in float32 add at most 2^-24 of the sum of magnitudes for each of the (tree's) additions:
2e-5 of that sum covers 300. The 8-bit checkpoint is exact: its integers, exponents and values are compared for equality.
"""
import math

import pytest
import torch

import learn_ref as R
import warchest_learn as wl
import warchest_wave as ww

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def float32_by_default():
    """Other test modules set torch's default type to float64 for the whole process."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
STEP = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}


def say(text):
    print(text, flush=True)


def near(got, want, what, scale=None):
    """Every element within its type's rounding and 2e-5 of the largest (or of `scale`)."""
    got64, want = got.detach().cpu().double(), want.double()
    assert got64.shape == want.shape, (what, got64.shape, want.shape)
    if not want.numel():
        return
    top = want.abs().max() if scale is None else scale
    bound = want.abs() * ROUND[got.dtype] + STEP[got.dtype] + 2e-5 * top
    bad = (got64 - want).abs() > bound
    assert not bad.any(), (what, int(bad.sum()), float((got64 - want).abs().max()), float(torch.as_tensor(top)))


def gen(seed):
    return torch.Generator().manual_seed(seed)


def strided(x, extra, fill=float("nan")):
    """x on the device with `extra` columns more per row in memory (holding `fill`), at an offset of one element."""
    rows, width = x.shape
    buf = torch.full((rows * (width + extra) + 1,), fill, dtype=x.dtype, device=DEV)
    v = buf[1:].view(rows, width + extra)[:, :width]
    v.copy_(x)
    return v


def to(x):
    return None if x is None else x.to(DEV)


# ------------------------------------------------------------------ policy loss

def policy_inputs(rows, vocab, dtype, seed, legal, ref):
    g = gen(seed)
    k = {"logits": (2 * torch.randn(rows, vocab, generator=g)).to(dtype),
         "actions": torch.randint(0, vocab, (rows,), generator=g),
         "advantages": torch.randn(rows, generator=g), "weights": torch.rand(rows, generator=g) + 0.1,
         "legal": None, "ref_logp": None, "ref_logits": None}
    if legal:
        k["legal"] = torch.rand(rows, vocab, generator=g) < 0.5
        k["legal"][torch.arange(rows), k["actions"]] = True
    x = k["logits"].double()
    if legal:
        x = x.masked_fill(~k["legal"], -math.inf)
    lp = torch.log_softmax(x, 1)[torch.arange(rows), k["actions"]].float()
    k["behaviour_logp"] = lp + 0.3 * torch.randn(rows, generator=g)
    if ref == "token":
        k["ref_logp"] = lp + 0.5 * torch.randn(rows, generator=g)
    if ref == "full":
        k["ref_logits"] = (k["logits"].float() + torch.randn(rows, vocab, generator=g)).to(dtype)
    return k


def check_policy(got, k, coefs):
    want = R.policy(**k, **coefs)
    for n in ("logp", "kl", "entropy"):
        near(getattr(got, n), want[n], n, scale=max(1.0, float(want[n].abs().max())) if len(want[n]) else None)
    near(got.loss, want["loss"], "loss", scale=1.0)
    near(got.grad, want["grad"], "grad", scale=max(1e-3, float(want["grad"].abs().max())))


COEFS = dict(inv_temperature=0.7, clip_low=0.2, clip_high=0.3, kl_coef=0.1, entropy_coef=0.02)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 8), (3, 22), (65, 7), (2, 64), (5, 63), (5, 65), (130, 97), (7, 511), (4, 513),
                                        (7, 1000), (3, 2049), (4, 4099), (300, 567), (2, 20011)])
def test_policy_loss_over_sizes(rows, vocab, dtype):
    for i, (legal, ref) in enumerate([(False, "none"), (True, "token"), (True, "full"), (False, "full")]):
        if rows * vocab > 50000 and i not in (0, 2):
            continue
        say(f"case policy: {rows} x {vocab} {dtype}, legal {legal}, ref {ref}")
        k = policy_inputs(rows, vocab, TYPES[dtype], rows + vocab, legal, ref)
        got = wl.policy_loss(**{n: to(v) for n, v in k.items()}, **COEFS)
        check_policy(got, k, COEFS)


@pytest.mark.parametrize("rows,vocab,dtype", [(2, 131072, "f32"), (2, 131072, "bf16"), (3, 70001, "f16"), (300, 33001, "bf16"),
                                              (257, 8200, "f32")])
def test_policy_loss_with_a_large_vocabulary(rows, vocab, dtype):
    """Against float64 torch over whole rows (the row-by-row code is for small ones)."""
    say(f"case policy: {rows} x {vocab} {dtype}")
    k = policy_inputs(rows, vocab, TYPES[dtype], vocab, False, "full")
    got = wl.policy_loss(**{n: to(v) for n, v in k.items()}, **COEFS)
    some = torch.randperm(rows, generator=gen(1))[:3]
    part = {n: v if v is None else v[some] for n, v in k.items()}
    want = R.policy(**part, **COEFS)
    for n in ("logp", "kl", "entropy"):
        near(getattr(got, n)[some.to(DEV)], want[n], n, scale=max(1.0, float(want[n].abs().max())))
    near(got.grad[some.to(DEV)], want["grad"], "grad")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [22, 700, 9001])
def test_policy_rows_left_out_and_what_lies_in_masked_places(vocab, dtype):
    """Weight 0 over NaN logits, actions out of range or illegal, rows with nothing legal, NaN and infinities in illegal
    columns, a row at the type's lowest value, columns at -infinity; strided rows with NaN between them; 32-bit actions."""
    say(f"case policy: rows left out, vocab {vocab} {dtype}")
    t = TYPES[dtype]
    k = policy_inputs(9, vocab, t, 5, True, "full")
    low = torch.finfo(t).min
    k["weights"][0], k["logits"][0] = 0.0, math.nan
    k["actions"][1], k["actions"][2] = -1, vocab
    k["legal"][3] = False
    k["legal"][4, k["actions"][4]] = False
    k["logits"][5] = torch.where(k["legal"][5], k["logits"][5], torch.tensor(math.nan, dtype=t))
    k["logits"][6] = torch.where(k["legal"][6], k["logits"][6], torch.tensor(math.inf, dtype=t))
    k["ref_logits"][5] = torch.where(k["legal"][5], k["ref_logits"][5], torch.tensor(-math.inf, dtype=t))
    k["logits"][7], k["ref_logits"][7] = low, low
    other = (torch.arange(vocab) != k["actions"][8]) & (torch.arange(vocab) % 3 == 0)
    k["logits"][8] = torch.where(other, torch.tensor(-math.inf, dtype=t), k["logits"][8])
    k["behaviour_logp"][7] = -math.log(float(k["legal"][7].sum()))
    want = R.policy(**k, **COEFS)
    dev = {n: to(v) for n, v in k.items()}
    dev["logits"], dev["ref_logits"] = strided(k["logits"], 5), strided(k["ref_logits"], 3)
    dev["actions"] = dev["actions"].int()
    got = wl.policy_loss(**dev, **COEFS)
    for n in ("logp", "kl", "entropy"):
        near(getattr(got, n), want[n], n, scale=max(1.0, float(want[n].abs().max())))
    near(got.grad, want["grad"], "grad")
    near(got.loss, want["loss"], "loss", scale=1.0)
    assert not got.grad[:5].any() and not got.logp[:5].any()


def test_policy_nan_in_a_counted_row_shows():
    k = policy_inputs(4, 40, torch.float32, 6, False, "none")
    k["logits"][2, 7] = math.nan
    got = wl.policy_loss(**{n: to(v) for n, v in k.items()}, **COEFS)
    assert got.loss.isnan() and got.logp[2].isnan() and got.grad[2].isnan().any()
    assert got.grad[[0, 1, 3]].isfinite().all()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("ref", ["none", "full"])
@pytest.mark.parametrize("vocab", [13, 60, 600, 5003, 20001, 90001])
def test_policy_gradient_of_illegal_columns_is_zero_whatever_the_row(vocab, ref, dtype):
    """A legal NaN or infinity, and an advantage that is NaN or infinite, show in the row's legal columns only."""
    for entropy_coef in (0.0, 0.02):
        k = policy_inputs(6, vocab, TYPES[dtype], vocab, True, ref)
        k["legal"][:, :4] = torch.tensor([False, True, True, True])
        k["actions"][:] = 2
        k["logits"][:, 2] = 1.0
        coefs = {**COEFS, "entropy_coef": entropy_coef}
        before = wl.policy_loss(**{n: to(v) for n, v in k.items()}, **coefs).grad
        k["logits"][1, 1], k["logits"][2, 1], k["logits"][2, 0] = math.nan, math.inf, math.nan
        k["advantages"][3], k["advantages"][4] = math.nan, math.inf
        got = wl.policy_loss(**{n: to(v) for n, v in k.items()}, **coefs).grad
        on, x = to(k["legal"]), to(k["logits"])
        assert not got[~on].any()
        for r in (1, 2):
            assert got[r][on[r] & (x[r] != -math.inf)].isnan().all(), r
        assert torch.equal(got[[0, 5]], before[[0, 5]])


@pytest.mark.parametrize("rows,vocab,dtype", [(5, 22, "f32"), (6, 3001, "bf16"), (2, 40000, "f16")])
def test_policy_in_place_without_gradient_scaled_and_again(rows, vocab, dtype):
    """grad written over the logits, not at all, or scaled by what arrives; the same bits every time."""
    say(f"case policy: ways to call, {rows} x {vocab} {dtype}")
    k = {n: to(v) for n, v in policy_inputs(rows, vocab, TYPES[dtype], 8, False, "token").items()}
    first = wl.policy_loss(**k, **COEFS)
    second = wl.policy_loss(**k, **COEFS)
    only = wl.policy_loss(**k, **COEFS, grad=False)
    assert only.grad is None
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    for a, b in zip(first[:4], only[:4]):
        near(a, b.cpu(), "without gradient", scale=1.0)
    scaled = wl.policy_loss(**k, **COEFS, grad_out=torch.tensor(2.0, device=DEV))
    near(scaled.grad, 2 * wl.policy_loss(**k, **COEFS).grad.double().cpu(), "twice")
    x = k.pop("logits").clone()
    over = wl.policy_loss(x, grad=x, **k, **COEFS)
    assert over.grad is x and torch.equal(x, first.grad)


def test_policy_no_rows_and_even_weights():
    z = torch.zeros(0, device=DEV)
    got = wl.policy_loss(torch.zeros(0, 5, device=DEV), z.long(), z, z)
    assert float(got.loss) == 0 and got.grad.shape == (0, 5)
    k = policy_inputs(6, 9, torch.float32, 9, False, "none")
    k["weights"] = None
    check_policy(wl.policy_loss(**{n: to(v) for n, v in k.items()}, **COEFS), k, COEFS)


def test_policy_gradient_against_differences_of_the_loss():
    """Float32 losses: steps of 0.05 leave 2e-3 of a unit gradient's curvature and 1e-5 of rounding."""
    k = policy_inputs(3, 6, torch.float32, 11, True, "full")
    dev = {n: to(v) for n, v in k.items()}
    grad = wl.policy_loss(**dev, **COEFS).grad.cpu()
    for i in range(18):
        step = []
        for s in (0.02, -0.02):
            x = k["logits"].clone()
            x.view(-1)[i] += s
            step.append(float(wl.policy_loss(**{**dev, "logits": x.to(DEV)}, **COEFS, grad=False).loss))
        assert abs((step[0] - step[1]) / 0.04 - float(grad.view(-1)[i])) < 2e-3


# -------------------------------------------------------------- preference loss

def preference_inputs(lengths, vocab, dtype, seed, lead=0, tail=0):
    g = gen(seed)
    ends = [lead]
    for n in lengths:
        ends.append(ends[-1] + n)
    rows = ends[-1] + tail
    logits = (2 * torch.randn(rows, vocab, generator=g)).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    lp = torch.log_softmax(logits.double(), 1)[torch.arange(rows), tokens].float()
    return {"logits": logits, "tokens": tokens, "offsets": torch.tensor(ends),
            "ref_logp": lp + 0.5 * torch.randn(rows, generator=g), "weights": (torch.rand(rows, generator=g) < 0.8).float()}


def check_preference(got, k, **kw):
    want = R.preference(**k, **kw)
    for n in ("margins", "ratios", "logp"):
        near(getattr(got, n), want[n], n, scale=max(1.0, float(want[n].abs().max())) if len(want[n]) else None)
    near(got.loss, want["loss"], "loss", scale=max(1.0, abs(float(want["loss"]))))
    near(got.grad, want["grad"], "grad", scale=max(1e-3, float(want["grad"].abs().max())) if len(want["grad"]) else None)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind,average", [("logistic", False), ("logistic", True), ("squared", True), ("hinge", False)])
@pytest.mark.parametrize("lengths,vocab", [([1, 1], 8), ([0, 3], 22), ([0, 0], 5), ([4, 0, 7, 2], 63), ([5, 6, 1, 0, 0, 9], 513),
                                           ([3, 300], 65), ([2, 3], 4099), ([1, 2], 20011)])
def test_preference_loss_over_sizes(lengths, vocab, dtype, kind, average):
    say(f"case preference: {lengths} x {vocab} {dtype} {kind} average {average}")
    k = preference_inputs(lengths, vocab, TYPES[dtype], sum(lengths) + vocab)
    kw = dict(beta=0.3, smoothing=0.1, kind=kind, average=average, inv_temperature=0.8)
    check_preference(wl.preference_loss(**{n: to(v) for n, v in k.items()}, **kw), k, **kw)


@pytest.mark.parametrize("vocab", [22, 3000])
def test_preference_rows_that_do_not_count(vocab):
    """Rows before and after the sequences (NaN logits), tokens out of range, weight 0 over NaN, a row at -infinity;
    32-bit indices; offsets beyond the rows and backwards; strided logits."""
    say(f"case preference: rows that do not count, vocab {vocab}")
    k = preference_inputs([4, 3, 5, 2], vocab, torch.float32, 3, lead=2, tail=3)
    k["logits"][0] = k["logits"][1] = k["logits"][-1] = math.nan
    k["tokens"][3], k["tokens"][6] = -1, vocab + 7
    k["weights"][:] = 1.0
    k["weights"][4], k["logits"][4] = 0.0, math.nan
    k["logits"][8] = -math.inf
    kw = dict(beta=0.5, kind="logistic", average=True)
    quiet = {**k, "logits": k["logits"].clone()}
    for r in (0, 1, len(quiet["logits"]) - 1):
        quiet["logits"][r] = 0.0
    want = R.preference(**quiet, **kw)
    dev = {n: to(v) for n, v in k.items()} | {"logits": strided(k["logits"], 3), "tokens": k["tokens"].int().to(DEV),
                                              "offsets": k["offsets"].int().to(DEV)}
    got = wl.preference_loss(**dev, **kw)
    near(got.grad, want["grad"], "grad")
    near(got.margins, want["margins"], "margins", scale=1.0)
    assert not got.grad[[0, 1, 3, 4, 6, 8, -1]].any()
    dev["offsets"] = torch.tensor([-5, 4, 1000, 900, 2000], dtype=torch.int32, device=DEV)
    quiet["offsets"] = torch.tensor([-5, 4, 1000, 900, 2000])
    quiet["logits"] = k["logits"].nan_to_num(nan=0.0, neginf=0.0)
    dev["logits"] = to(quiet["logits"])
    got = wl.preference_loss(**dev, **kw)
    want = R.preference(**quiet, **kw)
    near(got.margins, want["margins"], "margins", scale=1.0)
    near(got.grad, want["grad"], "grad")


def test_preference_far_margins_and_no_pairs():
    """Margins of +-1e4: the loss is linear or 0 there and its slope exact; no pairs: 0."""
    k = preference_inputs([2, 2, 2, 2], 9, torch.float32, 5)
    k["weights"][:] = 1.0
    k["ref_logp"][:2] += 5e3
    k["ref_logp"][4:6] -= 5e3
    got = wl.preference_loss(**{n: to(v) for n, v in k.items()}, beta=1.0)
    assert got.loss.isfinite() and got.grad.isfinite().all()
    assert not got.grad[4:].any() and got.grad[:4].any()
    assert abs(float(got.loss) - 5e3) < 10
    k["offsets"] = torch.zeros(1, dtype=torch.int64)
    got = wl.preference_loss(**{n: to(v) for n, v in k.items()})
    assert float(got.loss) == 0 and not got.grad.any()


def test_preference_again_in_place_and_without_gradient():
    k = {n: to(v) for n, v in preference_inputs([40, 3, 17, 60], 2001, torch.bfloat16, 6).items()}
    a, b = wl.preference_loss(**k), wl.preference_loss(**k)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert torch.equal(wl.preference_loss(**k, grad=False).margins, a.margins)
    x = k.pop("logits").clone()
    assert torch.equal(wl.preference_loss(x, grad=x, **k).grad, a.grad)


# ---------------------------------------------------------------- residual norm

def norm_inputs(rows, width, dtype, seed, kind, gate, pdtype=None):
    g = gen(seed)
    pdtype = pdtype or dtype
    k = {"block": (1.5 * torch.randn(rows, width, generator=g) + 0.2).to(dtype),
         "stream": (2 * torch.randn(rows, width, generator=g)).to(dtype),
         "post_gain": (1 + 0.1 * torch.randn(width, generator=g)).to(pdtype),
         "pre_gain": (1 + 0.1 * torch.randn(width, generator=g)).to(pdtype), "post_bias": None, "pre_bias": None,
         "gate": None}
    if kind == "layer":
        k["post_bias"], k["pre_bias"] = ((0.1 * torch.randn(width, generator=g)).to(pdtype) for _ in range(2))
    if gate == "vector":
        k["gate"] = (0.5 + 0.3 * torch.randn(width, generator=g)).to(pdtype)
    if gate == "token":
        k["gate"] = (0.5 + 0.3 * torch.randn(rows, width, generator=g)).to(dtype)
    d = [torch.randn(rows, width, generator=g).to(dtype) for _ in range(2)]
    return k, d


def check_norm(k, d, kw, dev=None):
    v = {n: None if t is None else t.double().requires_grad_(True) for n, t in k.items()}
    new, out = R.residual_norm(**v, **kw)
    dev = dev or {n: to(t) for n, t in k.items()}
    f = wl.residual_norm(**dev, **kw)
    # a row's normed values are as well known as its variance: widths of a few channels can leave little of it
    near(f.stream, new.detach(), "stream", scale=max(4.0, float(new.abs().max())) if new.numel() else None)
    near(f.out, out.detach(), "out", scale=8.0)
    given = [(o, t) for o, t in ((out, d[0]), (new, d[1])) if t is not None]
    if given:
        torch.autograd.backward([o for o, _ in given], [t.double() for _, t in given])
    b = wl.residual_norm_backward(to(d[0]), to(d[1]), dev["block"], dev["stream"], f.stats, *(
        dev[n] for n in ("post_gain", "post_bias", "gate", "pre_gain", "pre_bias")), **kw)
    for n, t in v.items():
        got = getattr(b, n)
        if t is None:
            assert got is None
            continue
        want = t.grad if t.grad is not None else torch.zeros_like(t)
        # sums over the rows of terms of about 1: 2e-5 of their magnitudes' sum
        near(got, want, n, scale=max(8.0, float(want.abs().max())) if want.numel() else None)
    return f, b


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,width", [(1, 8), (2, 7), (3, 65), (37, 96), (300, 33), (5, 129), (2, 512), (67, 513), (3, 1153),
                                        (2, 2049), (3, 4096), (2, 5000), (2, 8191), (1, 16384), (2, 9001)])
def test_residual_norm_over_sizes(rows, width, kind, dtype):
    for gate, act in (("none", "none"), ("vector", "none"), ("token", "sigmoid"), ("vector", "tanh")):
        if width > 1000 and gate == "none":
            continue
        say(f"case norm: {rows} x {width} {dtype} {kind} gate {gate} {act}")
        k, d = norm_inputs(rows, width, TYPES[dtype], rows + width, kind, gate)
        check_norm(k, d, dict(scale=0.7, eps=1e-3, norm=kind, gate_act=act))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_other_arguments(kind):
    """No rows; no parameters at all; float32 parameters beside 16-bit matrices; one of the two gradients missing;
    strided rows; a broadcast stream."""
    say(f"case norm: other arguments, {kind}")
    kw = dict(scale=-1.3, eps=1e-4, norm=kind)
    k, d = norm_inputs(0, 40, torch.float32, 1, kind, "vector")
    _, b = check_norm(k, d, kw)
    assert not b.post_gain.any() and not b.gate.any()
    k, d = norm_inputs(9, 40, torch.float32, 2, kind, "none")
    check_norm({n: t if n in ("block", "stream") else None for n, t in k.items()}, d, kw)
    k, d = norm_inputs(9, 200, torch.bfloat16, 3, kind, "vector", torch.float32)
    check_norm(k, d, kw)
    check_norm(k, [d[0], None], kw)
    check_norm(k, [None, d[1]], kw)
    k, d = norm_inputs(11, 51, torch.float16, 4, kind, "token")
    dev = {n: to(t) for n, t in k.items()} | {n: strided(k[n], 3) for n in ("block", "stream", "gate")}
    check_norm(k, d, kw, dev)
    k, d = norm_inputs(6, 72, torch.float32, 5, kind, "vector")
    k["stream"] = k["stream"][:1].expand(6, 72).contiguous()
    dev = {n: to(t) for n, t in k.items()} | {"stream": to(k["stream"][:1]).expand(6, 72)}
    check_norm(k, d, kw, dev)


def test_residual_norm_of_a_constant_row_and_one_channel():
    """A row without variance: normed values are 0, gradients stay finite."""
    x = torch.full((3, 24), 5.0, device=DEV)
    f = wl.residual_norm(x, torch.full_like(x, -5.0), norm="layer")
    assert not f.out.any() and torch.equal(f.stream, torch.full_like(x, -5.0))
    b = wl.residual_norm_backward(x, x, x, torch.full_like(x, -5.0), f.stats, norm="layer")
    assert b.block.isfinite().all() and b.stream.isfinite().all()
    one = torch.tensor([[3.0], [-2.0]], device=DEV)
    f = wl.residual_norm(one, one, norm="rms", eps=0.0)
    near(f.out, torch.tensor([[1.0], [-1.0]]), "one channel")


def test_residual_norm_many_rows_and_the_same_bits_twice():
    """More rows than workgroups: every workgroup's column sums hold several rows."""
    for rows, width, kind in ((3001, 96, "layer"), (1500, 1153, "rms"), (700, 4096, "layer")):
        say(f"case norm: {rows} x {width} {kind}")
        k, d = norm_inputs(rows, width, torch.float32, 7, kind, "vector")
        kw = dict(scale=0.5, eps=1e-5, norm=kind)
        _, b = check_norm(k, d, kw)
        _, c = check_norm(k, d, kw)
        for x, y in zip(b, c):
            assert (x is None and y is None) or torch.equal(x, y)


# ------------------------------------------------------- activations in 8 bits

SPECIAL = [0.0, -0.0, 1.0, -1.0, 127.0, 127.4999, 128.0, 0.5, 1.5, 2.5, -2.5, 3e-5, -6e4, 6.5e4, 1e-7, 255.0, 254.0]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (2, 31), (2, 32), (5, 33), (3, 64), (2, 100), (17, 257), (1, 1000)])
def test_checkpoint_writes_and_reads_exactly(rows, width, dtype):
    say(f"case checkpoint: {rows} x {width} {dtype}")
    t = TYPES[dtype]
    g = gen(rows * width)
    x = torch.randn(rows, width, generator=g) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float())
    x.view(-1)[: min(x.numel(), len(SPECIAL))] = torch.tensor(SPECIAL)[: x.numel()]
    if rows > 2:
        x[2] = 0.0
    x = x.to(t)
    q, e, value = R.keep8(x)
    for dev in (x.to(DEV), strided(x, 5)):
        ck = wl.checkpoint8(dev)
        assert torch.equal(ck.q.cpu(), q) and torch.equal(ck.exps.cpu(), e)
        got = wl.checkpoint8_read(ck, torch.float32)
        assert torch.equal(got.cpu().double(), value)
        assert torch.equal(wl.checkpoint8_read(ck, torch.bfloat16).cpu().double(), value)  # 8 bits fit bf16


def test_checkpoint_extremes():
    """Subnormals, the type's largest, infinities and NaN (whose group reads back as NaN, the next one untouched)."""
    for t in (torch.float32, torch.bfloat16):
        x = torch.zeros(6, 64, dtype=t)
        x[0, :3] = torch.tensor([1e-39, -3e-39, 2e-41])
        x[1, 0], x[1, 40] = torch.finfo(t).max, -torch.finfo(t).max
        x[2, 5], x[2, 33] = math.inf, 1.0
        x[3, 5], x[3, 33] = math.nan, 1.0
        x[4, 63] = -math.inf
        x[5, :32] = 2.0 ** -126
        q, e, value = R.keep8(x)
        ck = wl.checkpoint8(x.to(DEV))
        assert torch.equal(ck.q.cpu(), q) and torch.equal(ck.exps.cpu(), e)
        got = wl.checkpoint8_read(ck, torch.float32).cpu().double()
        # the largest number is kept as 64 * 2^122 = 2^128, which a read gives as float32's largest
        value = value.clamp(-torch.finfo(torch.float32).max, torch.finfo(torch.float32).max)
        assert torch.equal(got.isnan(), value.isnan())
        assert torch.equal(got.nan_to_num(), value.nan_to_num())
    empty = wl.checkpoint8(torch.zeros(0, 40, device=DEV))
    assert wl.checkpoint8_read(empty).shape == (0, 40)


@pytest.mark.parametrize("name", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width", [(1, 5), (3, 96), (40, 333)])
def test_checkpoint_activations_forward_and_backward(rows, width, dtype, name):
    say(f"case checkpoint {name}: {rows} x {width} {dtype}")
    t, g = TYPES[dtype], gen(width)
    x = (3 * torch.randn(rows, width, generator=g)).to(t)
    x.view(-1)[:4] = torch.tensor([0.0, -30.0, 30.0, 1e-3])
    d = torch.randn(rows, width, generator=g).to(t)
    _, _, value = R.keep8(x)
    z = value.requires_grad_(True)
    R.act(z, name).backward(d.double())
    ck, y = wl.checkpoint8_act(strided(x, 3), name)
    near(y, R.act(x.double(), name), "value", scale=4.0)
    near(wl.checkpoint8_act_backward(ck, strided(d, 1), name), z.grad, "slope", scale=4.0)
    near(wl.checkpoint8_read(ck, t, act=name), R.act(value.detach(), name), "read", scale=4.0)


def test_activation_tails_are_finite():
    x = torch.tensor([[-3e38, -1e20, -1e4, -90.0, 90.0, 1e4, 1e20, 3e38]], device=DEV)
    for name in ("relu", "gelu", "silu"):
        for i in range(8):
            ck, y = wl.checkpoint8_act(x[:, i:i + 1].contiguous(), name)
            d = wl.checkpoint8_act_backward(ck, torch.ones(1, 1, device=DEV), name)
            want = (max(float(x[0, i]), 0.0), 1.0 if i > 3 else 0.0)
            assert abs(float(y) - want[0]) <= 1e-6 * abs(want[0]) and abs(float(d) - want[1]) < 1e-6, (name, i)


# ----------------------------------------------------------------- weight gradient

def weight_case(rows, width, out, dtype, name, wdtype, seed=0, dev=None):
    t, g = TYPES[dtype], gen(rows + width + out + seed)
    x = 1.5 * torch.randn(rows, width, generator=g)
    d = torch.randn(rows, out, generator=g).to(t)
    ck = wl.checkpoint8(x.to(DEV))
    value = wl.checkpoint8_read(ck, torch.float32).cpu().double()
    weight, bias = wl.checkpoint8_weight_grad(ck, dev(d) if dev else to(d), act=name, bias=True, dtype=wdtype)
    a = R.act(value, name)
    want = a.t() @ d.double()
    size = a.abs().t() @ d.double().abs()  # the sum of the products' magnitudes
    # exact products: 2e-5 of the magnitudes for the float32 sums; a recomputed activation is rounded to grad's type
    bound = size * (2e-5 + (ROUND[t] if name in ("gelu", "silu") else 0.0)) + want.abs() * ROUND[weight.dtype] + 1e-30
    bound = bound + STEP[weight.dtype]
    off = (weight.cpu().double() - want).abs()
    assert not (off > bound).any(), (float(off.max()), float(bound.min()))
    near(bias, d.double().sum(0), "bias", scale=max(1.0, float(d.double().abs().sum(0).max())) if rows else 1.0)
    return weight, bias, ck


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width,out", [(0, 5, 3), (1, 1, 1), (1, 40, 9), (31, 33, 65), (32, 64, 64), (33, 130, 7), (300, 65, 129),
                                            (1000, 96, 22), (2500, 256, 200), (700, 1, 300), (130, 515, 260)])
def test_weight_gradient_over_sizes(rows, width, out, dtype):
    for name in ("none", "relu", "gelu", "silu"):
        if dtype == "f32" and name in ("gelu", "silu"):
            continue
        say(f"case weight: {rows} x {width} x {out} {dtype} {name}")
        weight_case(rows, width, out, dtype, name, torch.float32)
        weight_case(rows, width, out, dtype, name, TYPES[dtype])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_weight_gradient_long_sums_strides_and_the_same_bits(dtype):
    """A long sum over few tiles (split into runs), rows of grad at an odd stride and offset, twice the same bits."""
    say(f"case weight: long sum {dtype}")
    w, b, ck = weight_case(20011, 70, 50, dtype, "none", torch.float32, dev=lambda d: strided(d, 3))
    g = gen(1)
    d = torch.randn(20011, 50, generator=g).to(TYPES[dtype]).to(DEV)
    one, two = (wl.checkpoint8_weight_grad(ck, d, bias=True) for _ in range(2))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,width,out,name,pad", [
    (9000, 1500, 1504, "gelu", 0),     # 256-wide tiles past both ends, several runs of rows, rows past the last step
    (9001, 1500, 1501, "silu", 0),     # the gradient's rows at odd places: copied first
    (9000, 1500, 1504, "gelu", 8),     # its rows apart in memory
    (16384, 4096, 2048, "none", 0),    # whole tiles, whole steps
    (16411, 2050, 4090, "relu", 2),
])
def test_weight_gradient_of_large_products(rows, width, out, name, pad, dtype):
    """Sizes of the large tiles, or near where they begin, against a float64 product on the device."""
    say(f"case weight: {rows} x {width} x {out} {dtype} {name}, {pad} between rows")
    t = TYPES[dtype]
    g = torch.Generator(device=DEV).manual_seed(rows + out)
    x = 1.5 * torch.randn(rows, width, generator=g, device=DEV)
    d = torch.full((rows, out + pad), math.nan, dtype=t, device=DEV)[:, :out]
    d.copy_(torch.randn(rows, out, generator=g, device=DEV))
    ck = wl.checkpoint8(x)
    a = R.act(wl.checkpoint8_read(ck, torch.float32).double(), name)
    want = a.t().contiguous() @ d.double()
    size = a.abs().t().contiguous() @ d.double().abs()
    for wdtype in (torch.float32, t):
        weight, bias = wl.checkpoint8_weight_grad(ck, d, act=name, bias=True, dtype=wdtype)
        again, _ = wl.checkpoint8_weight_grad(ck, d, act=name, bias=True, dtype=wdtype)
        assert torch.equal(weight, again)
        bound = size * (2e-5 + (ROUND[t] if name in ("gelu", "silu") else 0.0)) + want.abs() * ROUND[wdtype] + STEP[wdtype]
        assert not ((weight.double() - want).abs() > bound).any()
        near(bias, d.double().sum(0).cpu(), "bias", scale=float(d.double().abs().sum(0).max()))


def test_weight_gradient_of_a_sliced_checkpoint_and_nan_groups():
    """A checkpoint's rows may be a slice of a larger one; a group held as NaN reaches its own channels only."""
    x = torch.randn(64, 96, generator=gen(2))
    x[20, 40] = math.inf
    ck = wl.checkpoint8(x.to(DEV))
    d = torch.randn(50, 8, generator=gen(3)).bfloat16().to(DEV)
    part = wl.Checkpoint8(ck.q[10:60], ck.exps[10:60])
    w, _ = wl.checkpoint8_weight_grad(part, d)
    assert w[32:64].isnan().all() and w[:32].isfinite().all() and w[64:].isfinite().all()


def test_f16_weight_gradient_at_the_ends_of_its_range():
    """A kept value just beyond f16's largest (65504 is kept as 65536) is held there."""
    x = torch.full((4, 32), 65504.0)
    ck = wl.checkpoint8(x.to(DEV))
    d = torch.ones(4, 3, dtype=torch.float16, device=DEV)
    w, _ = wl.checkpoint8_weight_grad(ck, d)
    assert torch.equal(w, torch.full_like(w, 4 * 65504.0))


# ------------------------------------------------------------------- streams, graphs

def everything(s):
    p = wl.policy_loss(**s["policy"], **COEFS)
    f = wl.preference_loss(**s["preference"])
    n = wl.residual_norm(**s["norm"])
    b = wl.residual_norm_backward(*s["d"], s["norm"]["block"], s["norm"]["stream"], n.stats, *(
        s["norm"][i] for i in ("post_gain", "post_bias", "gate", "pre_gain", "pre_bias")))
    ck, y = wl.checkpoint8_act(s["norm"]["block"], "gelu")
    z = wl.checkpoint8_act_backward(ck, s["d"][0], "gelu")
    w, c = wl.checkpoint8_weight_grad(ck, s["d"][1], act="relu", bias=True)
    return [t for t in (*p, *f, *n, *b, *ck, y, z, w, c) if t is not None]


def all_inputs(seed):
    k, d = norm_inputs(300, 96, torch.bfloat16, seed, "layer", "vector")
    return {"policy": {n: to(v) for n, v in policy_inputs(40, 700, torch.bfloat16, seed, False, "token").items()},
            "preference": {n: to(v) for n, v in preference_inputs([5, 9, 0, 3], 333, torch.float16, seed).items()},
            "norm": {n: to(v) for n, v in k.items()}, "d": [to(x) for x in d]}


def test_operators_on_another_stream():
    s = all_inputs(1)
    want = everything(s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = everything(s)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_operators_in_a_captured_graph():
    """Captured once, replayed over new inputs with eager work between: every replay equals the eager result."""
    held = all_inputs(1)
    everything(held)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = everything(held)
    for seed in (2, 3, 4):
        fresh = all_inputs(seed)
        want = [t.clone() for t in everything(fresh)]
        for part in ("policy", "preference", "norm"):
            for n, t in held[part].items():
                if t is not None:
                    t.copy_(fresh[part][n])
        for a, b in zip(held["d"], fresh["d"]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_refusals_of_the_binding():
    """Shapes, types and layouts that do not fit raise before anything is queued."""
    x = torch.zeros(4, 8, device=DEV)
    i = torch.zeros(4, dtype=torch.int64, device=DEV)
    v = torch.zeros(4, device=DEV)
    for call in (lambda: wl.policy_loss(x, i[:3], v, v), lambda: wl.policy_loss(x, v, v, v),
                 lambda: wl.policy_loss(x.t(), i, v, v), lambda: wl.policy_loss(x.double(), i, v, v),
                 lambda: wl.policy_loss(x, i, v.half(), v), lambda: wl.policy_loss(x, i, v, v, legal=x),
                 lambda: wl.policy_loss(x, i, v, v, ref_logp=v, ref_logits=x),
                 lambda: wl.policy_loss(x, i, v, v, grad=x.half()), lambda: wl.policy_loss(x, i, v.cpu(), v),
                 lambda: wl.preference_loss(x, i, i, v), lambda: wl.preference_loss(x, i, i[:3].int(), v),
                 lambda: wl.preference_loss(x, i, i[:3], None), lambda: wl.preference_loss(x, i, i[:3], v, kind="odd"),
                 lambda: wl.preference_loss(x, i, i[:3], v, beta=0.0),
                 lambda: wl.residual_norm(x, x.half()), lambda: wl.residual_norm(x, x[:, :4]),
                 lambda: wl.residual_norm(x, x, torch.ones(7, device=DEV)), lambda: wl.residual_norm(x, x, norm="batch"),
                 lambda: wl.residual_norm(x, x, gate=x[:1].expand(4, 8)),
                 lambda: wl.residual_norm(torch.zeros(1, 16385, device=DEV), torch.zeros(1, 16385, device=DEV)),
                 lambda: wl.residual_norm_backward(x, x, x, x, None), lambda: wl.checkpoint8(x.int()),
                 lambda: wl.checkpoint8_act(x, "tan"), lambda: wl.checkpoint8(x[0]),
                 lambda: wl.checkpoint8_read(wl.Checkpoint8(x, x)),
                 lambda: wl.checkpoint8_weight_grad(wl.checkpoint8(x), x, act="gelu"),
                 lambda: wl.checkpoint8_weight_grad(wl.checkpoint8(x), x[:3])):
        with pytest.raises(ww.WaveError):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("width", [24, 65, 513, 1025, 4097, 9001])
def test_residual_norm_in_place(width):
    """The new stream over the old one, and the stream's gradient over what arrived, through the C ABI: the same bits as
    apart. At 513, 1025 and 4097 columns the last chunk's first columns are another wavefront's too."""
    say(f"case norm in place: 2000 x {width}")
    k, d = norm_inputs(2000, width, torch.bfloat16, width, "layer", "vector")
    v = {n: to(t) for n, t in k.items()}
    f = wl.residual_norm(**v)
    b = wl.residual_norm_backward(to(d[0]), to(d[1]), v["block"], v["stream"], f.stats, *(
        v[n] for n in ("post_gain", "post_bias", "gate", "pre_gain", "pre_bias")))
    p = [v[n].data_ptr() for n in ("post_gain", "post_bias", "gate")]
    q = [v[n].data_ptr() for n in ("pre_gain", "pre_bias")]
    x, out = v["stream"].clone(), torch.empty_like(v["stream"])
    wl._call("wc_residual_norm", wl._NORM.pack(
        wl._NORM.size, 0, 2, 2, 0, 2000, width, v["block"].data_ptr(), width, x.data_ptr(), width, *p, 0, *q, 1.0, 1e-5, 1, 0,
        x.data_ptr(), width, out.data_ptr(), width, 0), x.device)
    assert torch.equal(x, f.stream) and torch.equal(out, f.out)
    g, block = to(d[1]), torch.empty_like(x)
    need = wl._norm_scratch(0, 2, 2000, width)
    work = torch.empty(need, dtype=torch.uint8, device=DEV)
    d_out = to(d[0])
    wl._call("wc_residual_norm_backward", wl._NORM_BACK.pack(
        wl._NORM_BACK.size, 0, 2, 2, 0, 2000, width, v["block"].data_ptr(), width, v["stream"].data_ptr(), width, *p, 0, q[0],
        1.0, 1, 0, 0, f.stats.data_ptr(), d_out.data_ptr(), width, g.data_ptr(), width, block.data_ptr(), width,
        g.data_ptr(), width, 0, 0, 0, 0, 0, 0, work.data_ptr(), need), x.device)
    assert torch.equal(g, b.stream) and torch.equal(block, b.block)


def far_rows(x, stride):
    """x's rows `stride` elements apart in memory that is otherwise left as it comes."""
    buf = torch.empty((x.shape[0] - 1) * stride + x.shape[1], dtype=x.dtype, device=DEV)
    v = buf.as_strided(x.shape, (stride, 1))
    v.copy_(x)
    return v


def test_rows_past_32_bit_offsets():
    """Rows a billion elements apart: the last one's offset passes what a signed 32-bit number holds in elements, and any
    32-bit number in bytes. The same bits as from rows side by side."""
    say("case far rows")
    far = (1 << 30) + 8
    k = {n: to(v) for n, v in policy_inputs(4, 900, torch.bfloat16, 3, False, "none").items()}
    want = wl.policy_loss(**k, **COEFS)
    g = far_rows(torch.zeros(4, 900, dtype=torch.bfloat16), far)
    got = wl.policy_loss(**{**k, "logits": far_rows(k["logits"], far)}, **COEFS, grad=g)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.grad, want.grad)
    del g, got
    k, d = norm_inputs(4, 200, torch.bfloat16, 4, "layer", "none")
    v = {n: to(t) for n, t in k.items()}
    want = wl.residual_norm(**v)
    got = wl.residual_norm(**{**v, "block": far_rows(v["block"], far)})
    assert torch.equal(got.stream, want.stream) and torch.equal(got.out, want.out)
    x = far_rows(v["block"], far)
    ck, plain = wl.checkpoint8(x), wl.checkpoint8(v["block"])
    assert torch.equal(ck.q, plain.q) and torch.equal(ck.exps, plain.exps)
    del got, x
    for out in (40, 41):
        dy = torch.randn(4, out, generator=gen(out)).bfloat16().to(DEV)
        want, _ = wl.checkpoint8_weight_grad(ck, dy)
        got, _ = wl.checkpoint8_weight_grad(ck, far_rows(dy, far))
        assert torch.equal(got, want)
    q = far_rows(ck.q, 1 << 31)
    got, _ = wl.checkpoint8_weight_grad(wl.Checkpoint8(q, ck.exps), dy)
    assert torch.equal(got, want)
    assert torch.equal(wl.checkpoint8_read(wl.Checkpoint8(q, ck.exps)), wl.checkpoint8_read(ck))


@pytest.mark.parametrize("rows,width", [(64, 9), (100, 15), (64, 17), (33, 31), (65, 33), (70, 100), (90, 257), (200, 321),
                                        (300, 505), (64, 3), (64, 511)])
def test_column_sums_of_odd_widths_count_every_row_once(rows, width):
    """Rows of one wavefront, whose last chunk of columns lies over the one before: whole numbers, so that a column's sum
    over the rows is exact and a row counted twice shows."""
    say(f"case norm column sums: {rows} x {width}")
    g = gen(rows + width)
    d = torch.randint(-50, 51, (rows, width), generator=g).float()
    u, x = torch.randn(rows, width, generator=g).to(DEV), torch.randn(rows, width, generator=g).to(DEV)
    one, zero = torch.ones(width, device=DEV), torch.zeros(width, device=DEV)
    for kind in ("layer", "rms"):
        f = wl.residual_norm(u, x, one, zero, None, one, zero, norm=kind)
        b = wl.residual_norm_backward(to(d), None, u, x, f.stats, one, zero, None, one, zero, norm=kind)
        assert torch.equal(b.pre_bias.cpu(), d.sum(0))
        # with no d_out the update's factor is 1: post_bias gets what arrives at the stream
        b = wl.residual_norm_backward(None, to(d), u, x, f.stats, one, zero, None, one, zero, norm=kind)
        assert torch.equal(b.post_bias.cpu(), d.sum(0)) and not b.pre_bias.any()


def test_preference_more_pairs_than_a_launch_has_workgroups():
    """Pairs whose threads, 256 each, pass 32 bits: the first, one in between and the last with rows, the others empty
    (margin 0). Margins and ratios as of the three alone, and the loss log 2 but for three parts in 2^24."""
    pairs = (1 << 24) + 3
    say(f"case preference: {pairs} pairs")
    k = preference_inputs([2, 1, 1, 2, 3, 1], 8, torch.float32, 12)
    small = wl.preference_loss(**{n: to(v) for n, v in k.items()}, beta=0.3)
    offsets = torch.zeros(2 * pairs + 1, dtype=torch.int32, device=DEV)
    at = [0, 1 << 23, pairs - 1]
    ends = k["offsets"].int().tolist()
    for i, p in enumerate(at):  # sequences before a pair end where it starts
        offsets[2 * p + 1:] = ends[2 * i + 1]
        offsets[2 * p + 2:] = ends[2 * i + 2]
    dev = {n: to(v) for n, v in k.items()} | {"offsets": offsets, "tokens": k["tokens"].int().to(DEV)}
    got = wl.preference_loss(**dev, beta=0.3)
    where = torch.tensor(at, device=DEV)
    assert torch.equal(got.margins[where], small.margins)
    assert torch.equal(got.ratios.view(-1, 2)[where], small.ratios.view(-1, 2))
    assert int(got.margins.count_nonzero()) <= 3
    assert abs(float(got.loss) - math.log(2)) < 2e-5
    # every row's coefficient is 3 / pairs of what it is among three
    near(got.grad * (pairs / 3), small.grad.cpu(), "grad")


@pytest.mark.parametrize("rows,vocab,dtype", [(3, 22, "f32"), (3, 567, "f32"), (3, 4099, "f16"), (2, 33001, "f32"),
                                              (2, 70001, "bf16")])
def test_policy_kl_does_not_depend_on_where_the_reference_lies(rows, vocab, dtype):
    """Rows that registers hold, and rows in chunks (float32 beyond 32,768 columns, 16 bits beyond 65,536): a constant
    added to the reference's logits, or to the policy's, changes nothing but their rounding, which the oracle shares; a
    reference row at the type's lowest value is an even one; columns of the policy at its lowest value (whole chunks of
    them among these) weigh nothing, whatever the reference holds there."""
    say(f"case policy kl: {rows} x {vocab} {dtype}")
    t = TYPES[dtype]
    low = torch.finfo(t).min
    k = policy_inputs(rows, vocab, t, vocab, False, "full")

    def check(**edit):
        e = {**k, **edit}
        lp = torch.log_softmax(e["logits"].double() * COEFS["inv_temperature"], 1)[torch.arange(rows), e["actions"]]
        e["behaviour_logp"] = lp.float() + 0.1  # ratios near 1: the loss is as well known as the log-probabilities
        want = R.policy(**e, **COEFS)
        got = wl.policy_loss(**{n: to(v) for n, v in e.items()}, **COEFS)
        for n in ("logp", "kl", "entropy"):
            near(getattr(got, n), want[n], n, scale=max(1.0, float(want[n].abs().max())))
        near(got.loss, want["loss"], "loss", scale=1.0)
        near(got.grad, want["grad"], "grad")
        assert all(v.isfinite().all() for v in got)

    for far in (1e4, -3e4, 6e4):
        check(ref_logits=(k["ref_logits"].float() + far).clamp(low, torch.finfo(t).max).to(t))
    y = k["ref_logits"].clone()
    y[0] = low
    check(ref_logits=y)
    x = k["logits"].clone()
    x[:, vocab // 3:] = low
    a = k["actions"] % (vocab // 3)
    check(logits=x, actions=a)
    check(logits=x.flip(1), actions=vocab - 1 - a)
    check(logits=(x.float() + 5000).clamp(min=low).to(t), actions=a)


@pytest.mark.parametrize("rows", [2, 64, 200])
def test_float32_weight_gradient_of_infinite_and_very_large_values(rows):
    """Infinities, NaN and float32's largest values (past bf16's) in single rows: each product as in float32, the other
    columns untouched. The one row that holds them has no kept value of 0."""
    say(f"case weight: float32 ends, {rows} rows")
    top = torch.finfo(torch.float32).max
    row = torch.tensor([math.inf, -math.inf, math.nan, top, -3.4e38, 3.39e38, 1.5, -2.0 ** 100])
    at = rows // 2
    x = torch.zeros(rows, 40)
    x[at] = torch.tensor([1.0, -0.5, 0.25, 127 / 256] * 10)
    x[:at, ::2] = 1.0
    d = torch.randint(-3, 4, (rows, 8), generator=gen(rows)).float()
    d[at] = row
    ck = wl.checkpoint8(x.to(DEV))
    kept = wl.checkpoint8_read(ck, torch.float32).cpu()
    assert kept[at].all() and torch.equal(kept[:at], x[:at])
    small = d.clone()
    small[at] = 0.0
    # the sums of the other rows are small whole numbers: added to the row's exact products
    want = (kept.double().t() @ small.double()) + kept[at].double()[:, None] * row.double()
    weight, bias = wl.checkpoint8_weight_grad(ck, d.to(DEV), bias=True)
    total = small.double().sum(0) + row.double()
    for got, exact in ((weight, want), (bias, total)):
        got, exact = got.cpu().double(), exact.clamp(-2.0 * top, 2.0 * top)
        assert torch.equal(got.isnan(), exact.isnan())
        ends = exact.abs() > top
        assert torch.equal(got[ends].isinf(), torch.ones_like(got[ends], dtype=torch.bool))
        assert torch.equal(got[ends] > 0, exact[ends] > 0)
        fine = ~ends & ~exact.isnan()
        assert ((got - exact)[fine].abs() <= 2e-6 * exact[fine].abs() + 1e-6).all()


@pytest.mark.parametrize("kind", ["logistic", "hinge"])
def test_preference_at_infinite_margins(kind):
    """A token of no probability: the margin is infinite. Without smoothing the loss is 0 where it is the rejected one's
    and infinite where it is the chosen one's, and the slope finite either way."""
    say(f"case preference: infinite margins, {kind}")
    x = torch.randn(4, 6, generator=gen(2))
    tokens, offsets = torch.tensor([0, 1, 2, 3], device=DEV), torch.tensor([0, 1, 2], device=DEV)
    v = torch.full((4,), -1.5, device=DEV)
    for lost, loss, slope in ((1, 0.0, 0.0), (0, math.inf, -0.3)):
        y = x.clone()
        y[lost, lost] = -math.inf
        got = wl.preference_loss(y.to(DEV), tokens, offsets, v, beta=0.3, kind=kind)
        assert float(got.loss) == loss and math.isinf(float(got.margins))
        p = torch.softmax(y.double(), 1)
        want = torch.zeros(4, 6, dtype=torch.float64)
        for r, sign in ((0, 1.0), (1, -1.0)):
            want[r] = -sign * slope * p[r]
            want[r, r] += sign * slope
        near(got.grad, want, "grad", scale=1.0)
    for smoothing, lost in ((0.1, 0), (0.1, 1), (1.0, 1)):
        y = x.clone()
        y[lost, lost] = -math.inf
        got = wl.preference_loss(y.to(DEV), tokens, offsets, v, beta=0.3, smoothing=smoothing)
        assert float(got.loss) == math.inf and got.grad.isfinite().all()
    y = x.clone()
    y[0, 0] = -math.inf
    assert float(wl.preference_loss(y.to(DEV), tokens, offsets, v, smoothing=1.0).loss) == 0.0


@pytest.mark.parametrize("rows,vocab,dtype", [(3, 50, "f32"), (3, 4099, "bf16"), (2, 33001, "f32"), (2, 70001, "f16")])
def test_policy_an_infinite_kl_without_a_coefficient_has_no_effect(rows, vocab, dtype):
    """A reference that gives a column no probability, a reference without any, and an action of no probability: the KL
    is infinite (undefined without a reference's column), loss and gradient with a coefficient of 0 those without a
    reference, and with one the loss infinite."""
    say(f"case policy infinite kl: {rows} x {vocab} {dtype}")
    coefs = {**COEFS, "kl_coef": 0.0}
    k = policy_inputs(rows, vocab, TYPES[dtype], vocab, False, "full")
    k["ref_logits"][0, vocab - 3] = -math.inf
    dev = {n: to(v) for n, v in k.items()}
    plain = wl.policy_loss(**{**dev, "ref_logits": None}, **coefs)

    def as_plain(got, plain):
        near(got.loss, plain.loss.cpu(), "loss", scale=1.0)
        near(got.grad, plain.grad.cpu(), "grad")
        near(got.entropy, plain.entropy.cpu(), "entropy")
        assert got.loss.isfinite() and got.grad.isfinite().all() and got.entropy.isfinite().all()

    got = wl.policy_loss(**dev, **coefs)
    as_plain(got, plain)
    assert float(got.kl[0]) == math.inf and got.kl[1:].isfinite().all()
    assert float(wl.policy_loss(**dev, **COEFS).loss) == math.inf
    dev["ref_logits"][0] = -math.inf
    as_plain(wl.policy_loss(**dev, **coefs), plain)

    token = policy_inputs(rows, vocab, TYPES[dtype], vocab, False, "token")
    token["logits"][0, token["actions"][0]] = -math.inf
    dev = {n: to(v) for n, v in token.items()}
    plain = wl.policy_loss(**{**dev, "ref_logp": None}, **coefs)
    got = wl.policy_loss(**dev, **coefs)
    as_plain(got, plain)
    assert float(got.kl[0]) == math.inf and float(wl.policy_loss(**dev, **COEFS).loss) == math.inf


@pytest.mark.parametrize("stride", [8192, (1 << 29) - 8, 1 << 29, (1 << 29) + 8])
def test_weight_gradient_scratch_of_rows_far_apart(stride):
    """One row, which a view may give any stride: the scratch that the binding asks for is what the call takes. The same
    bits as from a plain row."""
    say(f"case weight: row stride {stride}")
    g = gen(9)
    ck = wl.checkpoint8(torch.randn(1, 8192, generator=g).to(DEV))
    d = torch.randn(1, 8192, generator=g).bfloat16().to(DEV)
    want, _ = wl.checkpoint8_weight_grad(ck, d, dtype=torch.bfloat16)
    got, _ = wl.checkpoint8_weight_grad(ck, d.as_strided((1, 8192), (stride, 1)), dtype=torch.bfloat16)
    assert torch.equal(got, want)


# ---------------------------------------------------------- rows in chunks

def held_to(got, want, what, scale=None):
    """near, and no NaN where the definition has none."""
    assert torch.equal(got.isnan().cpu(), want.isnan()), what
    near(got, want, what, scale)


@pytest.mark.parametrize("ref", ["none", "token", "full"])
@pytest.mark.parametrize("vocab,dtype", [(70001, "f32"), (140001, "f16"), (140001, "bf16")])
def test_policy_rows_in_chunks(vocab, dtype, ref):
    """Rows past what registers hold, read in chunks of 8,192 columns: legal columns with a whole chunk of them illegal
    (NaN and infinities there), a row whose only legal columns are in the last chunk, rows left out of each kind, strided
    rows with NaN between; without a gradient, and with the gradient over the logits."""
    say(f"case policy in chunks: {vocab} {dtype} ref {ref}")
    t = TYPES[dtype]
    k = policy_inputs(9, vocab, t, vocab, True, ref)
    row = torch.arange(9)
    k["legal"][:, 16384:24576] = False
    k["actions"] = torch.where(k["legal"][row, k["actions"]], k["actions"], k["legal"].int().argmax(1))
    k["weights"][0], k["logits"][0] = 0.0, math.nan
    k["actions"][1], k["actions"][2] = -3, vocab
    k["legal"][3] = False
    k["legal"][4, k["actions"][4]] = False
    k["legal"][5, : vocab - 40] = False
    k["legal"][5, vocab - 9] = True
    k["actions"][5] = vocab - 9
    k["logits"][6] = torch.where(k["legal"][6], k["logits"][6], torch.tensor(math.nan, dtype=t))
    k["logits"][7] = torch.where(k["legal"][7], k["logits"][7], torch.tensor(math.inf, dtype=t))
    k["logits"][8, :8192] = -math.inf
    k["actions"][8] = 8192 + int(k["legal"][8, 8192:].int().argmax())
    # (where a row has no legal column, or an action none, any number does)
    lp = torch.log_softmax(k["logits"].double().masked_fill(~k["legal"], -math.inf) * COEFS["inv_temperature"], 1)
    lp = lp[row, k["actions"].clamp(0, vocab - 1)].nan_to_num(neginf=0.0).float()
    k["behaviour_logp"] = lp + 0.1
    if ref == "token":
        k["ref_logp"] = lp - 0.3
    want = R.policy(**k, **COEFS)
    dev = {n: to(v) for n, v in k.items()} | {"logits": strided(k["logits"], 3)}
    got = wl.policy_loss(**dev, **COEFS)
    for n in ("logp", "kl", "entropy"):
        held_to(getattr(got, n), want[n], n, scale=max(1.0, float(want[n].abs().max())))
    held_to(got.loss, want["loss"], "loss", scale=max(1.0, abs(float(want["loss"]))))
    held_to(got.grad, want["grad"], "grad")
    assert not got.grad[:5].any() and not got.logp[:5].any()
    only = wl.policy_loss(**dev, **COEFS, grad=False)
    assert only.grad is None
    for a, b in zip(got[1:4], only[1:4]):
        assert torch.equal(a, b)
    held_to(only.loss, got.loss.cpu(), "loss without a gradient", scale=max(1.0, abs(float(want["loss"]))))
    over = wl.policy_loss(**dev, **COEFS, grad=dev["logits"])
    assert torch.equal(over.loss, got.loss) and torch.equal(dev["logits"], got.grad)


@pytest.mark.parametrize("kind,average", [("logistic", True), ("squared", False), ("hinge", True)])
@pytest.mark.parametrize("vocab,dtype", [(70001, "f32"), (140001, "f16"), (140001, "bf16")])
def test_preference_rows_in_chunks(vocab, dtype, kind, average):
    """Rows past what registers hold: ragged pairs, a row left out of each kind, a chunk at -infinity; without a gradient,
    and with the gradient over the logits."""
    say(f"case preference in chunks: {vocab} {dtype} {kind} average {average}")
    k = preference_inputs([2, 3, 0, 4], vocab, TYPES[dtype], vocab, lead=1, tail=1)
    k["weights"][:] = torch.linspace(0.5, 1.5, len(k["weights"]))
    k["weights"][2], k["logits"][2] = 0.0, math.nan
    k["tokens"][4] = vocab
    k["logits"][5] = -math.inf
    k["logits"][6, 8192:16384] = -math.inf
    k["tokens"][6] = vocab - 1
    k["ref_logp"][6] = -10.0
    kw = dict(beta=0.3, smoothing=0.1, kind=kind, average=average, inv_temperature=0.8)
    want = R.preference(**k, **kw)
    dev = {n: to(v) for n, v in k.items()} | {"logits": strided(k["logits"], 5)}
    got = wl.preference_loss(**dev, **kw)
    for n in ("margins", "ratios", "logp"):
        held_to(getattr(got, n), want[n], n, scale=max(1.0, float(want[n].abs().max())))
    held_to(got.loss, want["loss"], "loss", scale=max(1.0, abs(float(want["loss"]))))
    held_to(got.grad, want["grad"], "grad", scale=max(1e-3, float(want["grad"].abs().max())))
    assert not got.grad[[0, 2, 4, 5, -1]].any()
    only = wl.preference_loss(**dev, **kw, grad=False)
    for a, b in zip(got[1:4], only[1:4]):
        assert torch.equal(a, b)
    held_to(only.loss, got.loss.cpu(), "loss without a gradient", scale=1.0)
    over = wl.preference_loss(**dev, **kw, grad=dev["logits"])
    assert torch.equal(over.loss, got.loss) and torch.equal(dev["logits"], got.grad)


@pytest.mark.parametrize("step", [0.02, 0.05])
def test_policy_gradient_against_differences_of_the_loss_per_row(step):
    """Rows of weight 1. Differences of the float64 loss are off by 2.2e-6 at 0.02 and 1.3e-5 at 0.05 here; a float32 loss
    of up to 4 adds 2^-22 twice over 2 steps, 1.2e-5 at 0.02, and its own terms' rounding as much: 1e-4."""
    k = policy_inputs(3, 6, torch.float32, 11, True, "full")
    k["weights"] = torch.ones(3)
    dev = {n: to(v) for n, v in k.items()}
    grad = wl.policy_loss(**dev, **COEFS).grad.cpu()
    for i in range(18):
        ends = []
        for s in (step, -step):
            x = k["logits"].clone()
            x.view(-1)[i] += s
            ends.append(float(wl.policy_loss(**{**dev, "logits": x.to(DEV)}, **COEFS, grad=False).loss))
        assert abs((ends[0] - ends[1]) / (2 * step) - float(grad.view(-1)[i])) < 1e-4


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 8), (2, 31), (65, 100), (33, 513), (5, 1153), (9, 4099), (2, 9001)])
def test_finite_inputs_give_finite_outputs(rows, width, dtype):
    """A comparison with a bound lets a NaN pass: every output of every operator, over sizes of each kernel."""
    say(f"case finite: {rows} x {width} {dtype}")
    t = TYPES[dtype]
    outs = []
    for legal, ref in ((False, "none"), (True, "token"), (True, "full")):
        k = policy_inputs(rows, width, t, rows + width, legal, ref)
        outs += wl.policy_loss(**{n: to(v) for n, v in k.items()}, **COEFS)
    k = preference_inputs([rows, rows // 2, 0, 1], width, t, rows)
    for kind in ("logistic", "squared", "hinge"):
        outs += wl.preference_loss(**{n: to(v) for n, v in k.items()}, kind=kind, average=True)
    for kind, gate, act in (("rms", "none", "none"), ("layer", "vector", "tanh"), ("layer", "token", "sigmoid")):
        k, d = norm_inputs(rows, width, t, rows + width, kind, gate)
        v = {n: to(x) for n, x in k.items()}
        f = wl.residual_norm(**v, norm=kind, gate_act=act)
        b = wl.residual_norm_backward(to(d[0]), to(d[1]), v["block"], v["stream"], f.stats, *(
            v[n] for n in ("post_gain", "post_bias", "gate", "pre_gain", "pre_bias")), norm=kind, gate_act=act)
        outs += [x for x in (*f, *b) if x is not None]
    x = to(norm_inputs(rows, width, t, 1, "rms", "none")[0]["block"])
    for act in ("none", "relu", "gelu", "silu"):
        ck, y = wl.checkpoint8_act(x, act)
        outs += [y, wl.checkpoint8_read(ck, t, act), wl.checkpoint8_act_backward(ck, x, act)]
        if dtype != "f32" or act in ("none", "relu"):
            outs += wl.checkpoint8_weight_grad(ck, x[:, : (width + 1) // 2], act=act, bias=True)
    for i, o in enumerate(outs):
        assert o.isfinite().all(), i
