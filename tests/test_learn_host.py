"""CPU checks of the training operators' C ABI and binding: exports, structure layouts, refusals, and the float64
references' gradients against differences of the losses they belong to."""
import ctypes as C
import os
import re
import struct
import subprocess

import pytest
import torch

import learn_ref as R
import warchest_learn as wl
import warchest_wave as ww


@pytest.fixture(autouse=True)
def float32_by_default():
    """Other test modules set torch's default type to float64 for the whole process."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "wc_learn.h")
STRUCTS = {"wc_policy_args": wl._POLICY, "wc_preference_args": wl._PREFERENCE, "wc_norm_args": wl._NORM,
           "wc_norm_back_args": wl._NORM_BACK, "wc_ckpt_args": wl._CKPT, "wc_ckpt_weight_args": wl._WEIGHT}


def test_every_declared_symbol_is_exported():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\b(wc_[a-z0-9_]+)\s*\(", text))
    assert names == set(wl.EXPORTS)
    for n in names:
        assert hasattr(ww.lib(), n)


def test_structures_are_packed_as_c_lays_them_out(tmp_path):
    """Sizes, and every field's offset: the header's fields in order against the packing's."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    lines, want = [], {}
    for name, packed in STRUCTS.items():
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        fields = [re.search(r"(\w+)$", f.strip().rstrip("*").strip()).group(1)
                  for d in body.split(";") if d.strip() for f in d.split(",")]
        assert len(fields) == len(packed.unpack(bytes(packed.size))), name
        lines += ['printf("%%zu ", sizeof(%s));' % name] + ['printf("%%zu ", offsetof(%s, %s));' % (name, f)
                                                           for f in fields]
        offsets, fmt = [], packed.format.replace(" ", "")
        for i in range(1, len(fmt)):
            at = struct.calcsize(fmt[:i] + "0" + fmt[i]) if i > 1 else 0
            offsets.append(at)
        want[name] = [packed.size] + offsets
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "%s"\nint main(void) { %s return 0; }\n' % (HEADER, " ".join(lines)))
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.check_output([str(tmp_path / "sizes")]).split()]
    assert got == [x for name in STRUCTS for x in want[name]]


P = 256  # an address that passes for one; refused calls read nothing

POLICY = dict(bytes=216, device=0, dtype=0, rows=4, vocab=10, logits=P, logits_stride=10, legal=0, legal_stride=0, ref=0,
              ref_stride=0, actions=P, behaviour=P, advantages=P, weights=0, ref_logp=0, grad_out=0, inv=1.0, low=0.2,
              high=0.2, kl=0.0, ent=0.0, bits=64, loss=P, logp=P, klo=P, entropy=P, grad=P, grad_stride=10, work=P,
              work_bytes=1 << 30)
PREFERENCE = dict(bytes=184, device=0, dtype=1, rows=4, vocab=10, pairs=1, logits=P, logits_stride=10, tokens=P, offsets=P,
                  ref_logp=P, weights=0, grad_out=0, inv=1.0, beta=0.1, smoothing=0.0, kind=0, average=0, bits=32, loss=P,
                  margins=P, ratios=P, logp=P, grad=P, grad_stride=10, work=P, work_bytes=1 << 30)
NORM = dict(bytes=176, device=0, dtype=2, pdtype=2, pad=0, rows=4, width=16, block=P, block_stride=16, stream=P,
            stream_stride=16, pg=P, pb=P, gate=0, gate_stride=0, ng=P, nb=P, scale=1.0, eps=1e-5, norm=0, act=0, new=P,
            new_stride=16, out=P, out_stride=16, stats=P)
NORM_BACK = dict(bytes=264, device=0, dtype=2, pdtype=2, pad0=0, rows=4, width=16, block=P, block_stride=16, stream=P,
                 stream_stride=16, pg=P, pb=P, gate=0, gate_stride=0, ng=P, scale=1.0, norm=0, act=0, pad=0, stats=P,
                 d_out=P, d_out_stride=16, d_new=P, d_new_stride=16, d_block=P, d_block_stride=16, d_stream=P,
                 d_stream_stride=16, dpg=P, dpb=P, dng=P, dnb=P, d_gate=0, d_gate_stride=0, work=P, work_bytes=1 << 30)
CKPT = dict(bytes=104, device=0, dtype=0, rows=4, width=40, act=0, pad=0, q=P, q_stride=40, exps=P, exps_stride=2, x=P,
            x_stride=40, y=P, y_stride=40)
WEIGHT = dict(bytes=136, device=0, dtype=1, rows=4, width=40, out=8, act=0, wdtype=0, q=P, q_stride=40, exps=P,
              exps_stride=2, grad=P, grad_stride=8, weight=P, weight_stride=8, bias=P, work=P, work_bytes=1 << 30)


@pytest.mark.parametrize("entry,packed,base,edit,word", [
    ("wc_policy_loss", wl._POLICY, POLICY, dict(bytes=208), "size"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(dtype=3), "dtype"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(rows=-1), "rows"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(vocab=0), "width"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(logits=0), "logits"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(logits=P + 2), "logits"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(logits_stride=9), "logits"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(grad_stride=0), "grad"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(bits=16), "index_bits"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(actions=0), "actions"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(loss=0), "loss"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(inv=0.0), "inv_temperature"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(inv=float("nan")), "inv_temperature"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(low=-0.1), "clip"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(ref=P, ref_stride=10, ref_logp=P), "exclude"),
    ("wc_policy_loss", wl._POLICY, POLICY, dict(device=-1), "device"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(pairs=-1), "pairs"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(beta=0.0), "beta"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(smoothing=1.5), "smoothing"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(kind=3), "kind"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(offsets=0), "offsets"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(ref_logp=0), "ref_logp"),
    ("wc_preference_loss", wl._PREFERENCE, PREFERENCE, dict(tokens=P + 1), "tokens"),
    ("wc_residual_norm", wl._NORM, NORM, dict(width=16385, block_stride=16385, stream_stride=16385), "MAX_WIDTH"),
    ("wc_residual_norm", wl._NORM, NORM, dict(norm=2), "norm"),
    ("wc_residual_norm", wl._NORM, NORM, dict(act=-1), "gate_act"),
    ("wc_residual_norm", wl._NORM, NORM, dict(out=0), "out"),
    ("wc_residual_norm", wl._NORM, NORM, dict(pdtype=7), "dtype"),
    ("wc_residual_norm", wl._NORM, NORM, dict(new_stride=8), "new_stream"),
    ("wc_residual_norm", wl._NORM, NORM, dict(stats=P + 8), "stats"),
    ("wc_residual_norm", wl._NORM, NORM, dict(eps=-1.0), "eps"),
    ("wc_residual_norm_backward", wl._NORM_BACK, NORM_BACK, dict(stats=0), "stats"),
    ("wc_residual_norm_backward", wl._NORM_BACK, NORM_BACK, dict(d_gate=P), "d_gate"),
    ("wc_residual_norm_backward", wl._NORM_BACK, NORM_BACK, dict(d_block=0), "d_block"),
    ("wc_residual_norm_backward", wl._NORM_BACK, NORM_BACK, dict(scale=float("inf")), "scale"),
    ("wc_ckpt_write", wl._CKPT, CKPT, dict(act=4), "act"),
    ("wc_ckpt_write", wl._CKPT, CKPT, dict(x=0), "x"),
    ("wc_ckpt_write", wl._CKPT, CKPT, dict(exps_stride=1), "exps"),
    ("wc_ckpt_read", wl._CKPT, CKPT, dict(y=0), "y"),
    ("wc_ckpt_act_backward", wl._CKPT, CKPT, dict(q=0), "q"),
    ("wc_ckpt_weight_grad", wl._WEIGHT, WEIGHT, dict(wdtype=2), "weight_dtype"),
    ("wc_ckpt_weight_grad", wl._WEIGHT, WEIGHT, dict(dtype=0, act=2), "float32"),
    ("wc_ckpt_weight_grad", wl._WEIGHT, WEIGHT, dict(out=0), "width"),
    ("wc_ckpt_weight_grad", wl._WEIGHT, WEIGHT, dict(weight=0), "weight"),
    ("wc_ckpt_weight_grad", wl._WEIGHT, WEIGHT, dict(grad=P + 1), "grad"),
])
def test_refusals_name_their_reason(entry, packed, base, edit, word):
    """Every refusal comes from the host's checks, before any device call."""
    fields = {**base, **edit}
    assert base["bytes"] == packed.size
    rc = wl._entry(entry)(packed.pack(*fields.values()), None)
    assert rc in (-1, -4)
    assert word in ww.lib().wc_last_error().decode(), ww.lib().wc_last_error()


def test_null_descriptions_are_refused():
    for n in wl.EXPORTS:
        f = getattr(ww.lib(), n)
        f.argtypes, f.restype = [C.c_char_p, C.c_void_p], C.c_int
        wl._fn.pop(n, None)
        assert f(None, None) == -1
        assert b"null" in ww.lib().wc_last_error()


def test_the_binding_refuses_tensors_that_are_not_on_a_gpu():
    x = torch.zeros(2, 3)
    with pytest.raises(ww.WaveError, match="not on a GPU"):
        wl.policy_loss(x, torch.zeros(2, dtype=torch.int64), x[:, 0], x[:, 0])
    with pytest.raises(ww.WaveError, match="not on a GPU"):
        wl.checkpoint8(x)
    with pytest.raises(ww.WaveError, match="not on a GPU"):
        wl.residual_norm(x, x)


def central(f, x, eps=1e-5):
    """Central differences of f at x, element by element."""
    g = torch.zeros_like(x)
    for i in range(x.numel()):
        hi, lo = x.clone().reshape(-1), x.clone().reshape(-1)
        hi[i] += eps
        lo[i] -= eps
        g.view(-1)[i] = (f(hi.view_as(x)) - f(lo.view_as(x))) / (2 * eps)
    return g


@pytest.mark.parametrize("ref", ["none", "token", "full"])
def test_the_reference_policy_gradient_is_the_slope_of_its_loss(ref):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 6, generator=g, dtype=torch.float64)
    legal = torch.rand(4, 6, generator=g) < 0.8
    legal[:, 2] = True
    kw = dict(actions=torch.tensor([2, 2, 2, -1]), behaviour_logp=torch.full((4,), -1.5), advantages=torch.randn(4, generator=g),
              weights=torch.tensor([0.5, 1.0, 0.25, 1.0]), legal=legal, inv_temperature=0.7, kl_coef=0.3, entropy_coef=0.2)
    if ref == "token":
        kw["ref_logp"] = torch.randn(4, generator=g) - 1.5
    if ref == "full":
        kw["ref_logits"] = torch.randn(4, 6, generator=g)
    want = central(lambda t: float(R.policy(t, **kw)["loss"]), x)
    # central differences of step 1e-5: 1e-10 of the third derivative, and 1e-16 / 1e-5 of rounding
    torch.testing.assert_close(R.policy(x, **kw)["grad"], want, rtol=0, atol=1e-8)


@pytest.mark.parametrize("kind", ["logistic", "squared", "hinge"])
@pytest.mark.parametrize("average", [False, True])
def test_the_reference_preference_gradient_is_the_slope_of_its_loss(kind, average):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(9, 5, generator=g, dtype=torch.float64)
    kw = dict(tokens=torch.tensor([0, 1, 4, 2, -1, 3, 3, 1, 0]), offsets=torch.tensor([1, 4, 6, 6, 8]),
              ref_logp=torch.randn(9, generator=g) - 1.5, weights=torch.tensor([1.0, 0.5, 0, 1, 1, 2, 1, 1, 1]), beta=0.3,
              smoothing=0.1, kind=kind, average=average, inv_temperature=1.3)
    want = central(lambda t: float(R.preference(t, **kw)["loss"]), x)
    torch.testing.assert_close(R.preference(x, **kw)["grad"], want, rtol=0, atol=1e-8)
