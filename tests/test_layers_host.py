"""CPU checks of the layer, update and log-probability operators: structure layouts, refusals, and the float64
references' gradients against differences."""
import os
import re
import struct
import subprocess

import pytest
import torch

import layer_ref as R
import warchest_learn as wl
import warchest_wave as ww

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "wc_learn.h")
STRUCTS = {"wc_linear_args": wl._LINEAR, "wc_linear_back_args": wl._LINEAR_BACK, "wc_orthogonalise_args": wl._ORTHO,
           "wc_logp_args": wl._LOGP, "wc_logp_back_args": wl._LOGP_BACK}


@pytest.fixture(autouse=True)
def float32_by_default():
    """Other test modules set torch's default type to float64 for the whole process."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)


def fields_of(name):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    return [re.search(r"(\w+)$", f.strip().rstrip("*").strip()).group(1)
            for d in body.split(";") if d.strip() for f in d.split(",")]


def test_structures_are_packed_as_c_lays_them_out(tmp_path):
    lines, want = [], []
    for name, packed in STRUCTS.items():
        fields = fields_of(name)
        assert len(fields) == len(packed.unpack(bytes(packed.size))), name
        lines += ['printf("%%zu ", sizeof(%s));' % name] + ['printf("%%zu ", offsetof(%s, %s));' % (name, f)
                                                           for f in fields]
        fmt = packed.format.replace(" ", "")
        want += [packed.size] + [struct.calcsize(fmt[:i] + "0" + fmt[i]) if i > 1 else 0 for i in range(1, len(fmt))]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "%s"\nint main(void) { %s return 0; }\n' % (HEADER, " ".join(lines)))
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "sizes")], check=True)
    assert [int(x) for x in subprocess.check_output([str(tmp_path / "sizes")]).split()] == want


P = 256  # an address that passes for one; refused calls read nothing
WORK = dict(workspace=P, workspace_bytes=1 << 40)
LINEAR = dict(bytes=wl._LINEAR.size, device=0, dtype=2, bias_dtype=0, weight_layout=0, rows=4, width=16, out=8, x=P,
              x_stride=16, weight=P, weight_stride=8, bias=P, residual=P, residual_stride=8, act=2, pad=0, pre=P,
              pre_stride=8, y=P, y_stride=8, **WORK)
BACK = dict(bytes=wl._LINEAR_BACK.size, device=0, dtype=2, weight_layout=1, act=2, grad_dtype=2, pad=0, rows=4, width=16,
            out=8, d_out=P, d_out_stride=8, pre=P, pre_stride=8, x=P, x_stride=16, weight=P, weight_stride=16, d_x=P,
            d_x_stride=16, d_weight=P, d_weight_stride=16, d_bias=P, **WORK)
ORTHO = dict(bytes=wl._ORTHO.size, device=0, dtype=0, out_dtype=2, steps=5, batch=2, rows=4, width=16, update=P,
             update_stride=16, update_batch=64, out=P, out_stride=16, out_batch=64, a=3.4445, b=-4.775, c=2.0315,
             eps=1e-7, scale=1.0, pad=0, **WORK)
LOGP = dict(bytes=wl._LOGP.size, device=0, dtype=0, rows=4, vocab=10, logits=P, logits_stride=10, legal=P,
            legal_stride=10, tokens=P, inv_temperature=1.0, index_bits=64, top=3, pad=0, logp=P, entropy=P, rank=P,
            top_logp=P, top_index=P, stats=P, **WORK)
LOGP_BACK = dict(bytes=wl._LOGP_BACK.size, device=0, dtype=0, rows=4, vocab=10, logits=P, logits_stride=10, legal=0,
                 legal_stride=0, tokens=P, inv_temperature=1.0, index_bits=32, stats=P, d_logp=P, d_entropy=P, grad=P,
                 grad_stride=10)
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("entry,name,packed,base,edit,word", [
    (e, n, p, b, edit, word)
    for e, n, p, b, cases in [
        ("wc_linear", "wc_linear_args", wl._LINEAR, LINEAR, [
            (dict(bytes=8), "size"), (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(width=0), "width"),
            (dict(out=0), "width"), (dict(out=(1 << 20) + 1), "2^20"), (dict(rows=1 << 31), "2^31"),
            (dict(weight_layout=2), "weight_layout"), (dict(act=4), "act"), (dict(act=-1), "act"), (dict(x=0), "x "),
            (dict(x=P + 1), "x "), (dict(x_stride=15), "x:"), (dict(weight=0), "weight"), (dict(weight_stride=7), "weight"),
            (dict(weight_layout=1, weight_stride=15), "weight"), (dict(bias_dtype=1), "bias_dtype"), (dict(bias=P + 2), "bias"),
            (dict(residual_stride=-8), "residual"), (dict(y=0), "y "), (dict(y_stride=0), "y:"), (dict(pre_stride=4), "pre"),
            (dict(device=-1), "device")]),
        ("wc_linear_backward", "wc_linear_back_args", wl._LINEAR_BACK, BACK, [
            (dict(bytes=8), "size"), (dict(grad_dtype=1), "grad_dtype"), (dict(d_out=0), "d_out"), (dict(pre=0), "pre"),
            (dict(x=0), "x "), (dict(weight=0), "weight"), (dict(d_weight_stride=8), "d_weight"), (dict(d_x_stride=8), "d_x"),
            (dict(d_bias=P + 1), "d_bias"), (dict(rows=-2), "rows")]),
        ("wc_orthogonalise", "wc_orthogonalise_args", wl._ORTHO, ORTHO, [
            (dict(bytes=8), "size"), (dict(dtype=9), "dtype"), (dict(out_dtype=-1), "dtype"), (dict(batch=-1), "batch"),
            (dict(batch=65536), "batch"), (dict(rows=0), "rows"), (dict(width=0), "rows and width"),
            (dict(width=1 << 21, update_stride=1 << 21, out_stride=1 << 21), "2^20"), (dict(steps=0), "steps"),
            (dict(steps=65), "steps"), (dict(a=NAN), "coefficients"), (dict(c=INF), "coefficients"),
            (dict(scale=INF), "scale"), (dict(eps=-1.0), "eps"), (dict(eps=NAN), "eps"), (dict(update=0), "update"),
            (dict(update_stride=15), "update"), (dict(update_batch=-1), "update_batch"), (dict(out=0), "out "),
            (dict(out_stride=15), "out:"), (dict(out_batch=63), "overlap")]),
        ("wc_token_logp", "wc_logp_args", wl._LOGP, LOGP, [
            (dict(bytes=8), "size"), (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "width"),
            (dict(rows=1 << 31), "launch"), (dict(index_bits=8), "index_bits"), (dict(inv_temperature=0.0), "inv_temperature"),
            (dict(inv_temperature=INF), "inv_temperature"), (dict(logits=0), "logits"), (dict(logits_stride=5), "logits"),
            (dict(legal_stride=9), "legal"), (dict(tokens=P + 4), "tokens"), (dict(top=65), "top"), (dict(top=-1), "top"),
            (dict(logp=0), "logp"), (dict(rank=0), "rank"), (dict(entropy=0), "entropy"), (dict(top_logp=0), "top_logp"),
            (dict(top_index=0), "top_index"), (dict(stats=P + 4), "stats")]),
        ("wc_token_logp_backward", "wc_logp_back_args", wl._LOGP_BACK, LOGP_BACK, [
            (dict(bytes=8), "size"), (dict(stats=0), "stats"), (dict(grad=0), "grad"), (dict(grad_stride=9), "grad"),
            (dict(d_logp=P + 1), "d_logp"), (dict(d_entropy=P + 2), "d_entropy")])]
    for edit, word in cases])
def test_refusals_name_their_reason(entry, name, packed, base, edit, word):
    """Every refusal comes from the host's checks, before any device call."""
    assert list(base) == fields_of(name)
    rc = wl._entry(entry)(packed.pack(*{**base, **edit}.values()), None)
    assert rc in (-1, -4)
    assert word in ww.lib().wc_last_error().decode(), ww.lib().wc_last_error()


OVER = 1 << 16  # another address: what is written over itself


@pytest.mark.parametrize("entry,packed,fields,edit,allowed", [
    ("wc_linear", wl._LINEAR, LINEAR, dict(residual=OVER, y=OVER, residual_stride=8, y_stride=9), dict(y_stride=8)),
    ("wc_linear", wl._LINEAR, LINEAR, dict(residual=OVER, y=OVER, residual_stride=0), dict(rows=1)),
    ("wc_orthogonalise", wl._ORTHO, ORTHO, dict(update=OVER, out=OVER), dict(out_dtype=0)),
    ("wc_orthogonalise", wl._ORTHO, ORTHO, dict(update=OVER, out=OVER, out_dtype=0, out_stride=17, out_batch=68), dict(batch=1)),
    ("wc_orthogonalise", wl._ORTHO, ORTHO, dict(update=OVER, out=OVER, out_dtype=0, out_batch=65), dict(batch=1)),
    ("wc_token_logp_backward", wl._LOGP_BACK, LOGP_BACK, dict(logits=OVER, grad=OVER, grad_stride=11), dict(grad_stride=10))])
def test_an_output_over_an_input_has_its_layout(entry, packed, fields, edit, allowed):
    """Other strides or another type would be written where rows are still to be read: refused. What is allowed passes these
    checks, and is stopped by the one of the device."""
    for more, word in ((edit, "itself needs"), ({**edit, **allowed, "device": -1}, "device")):
        assert wl._entry(entry)(packed.pack(*{**fields, **more}.values()), None) == -1
        assert word in ww.lib().wc_last_error().decode(), ww.lib().wc_last_error()


def test_the_binding_refuses_tensors_that_are_not_on_a_gpu():
    x = torch.zeros(2, 3)
    for call in (lambda: wl.linear(x, x.t()), lambda: wl.linear_backward(x, x, x.t()), lambda: wl.orthogonalise(x),
                 lambda: wl.token_logp(x), lambda: wl.token_logp_backward(None, None, x, None, None)):
        with pytest.raises(ww.WaveError, match="not on a GPU"):
            call()


def test_dense_keeps_pre_activations_only_for_gradients_that_read_them(monkeypatch):
    """Not under no_grad or inference_mode, whatever requires a gradient, nor for the residual's, which does not read them."""
    kept = []

    def linear(x, weight, bias=None, *, act="none", residual=None, keep=False):
        kept.append(keep)
        out = x @ weight
        return wl.Linear(out if residual is None else out + residual, out.clone() if keep else None)
    monkeypatch.setattr(wl, "linear", linear)
    x, w, b, r = torch.randn(3, 4), torch.randn(4, 5), torch.randn(5), torch.randn(3, 5)
    parameters = [torch.nn.Parameter(t.clone()) for t in (w, b)]
    with torch.no_grad():
        wl.dense(x, *parameters, act="gelu")
    with torch.inference_mode():
        wl.dense(x, *parameters, act="gelu")
    wl.dense(x, w, b, act="gelu")
    wl.dense(x, w, b, act="gelu", residual=r.clone().requires_grad_(True)).sum().backward()
    assert kept == [False] * 4
    for one in range(3):
        wl.dense(*(t.clone().requires_grad_(i == one) for i, t in enumerate((x, w, b))), act="gelu")
    assert kept[4:] == [True] * 3


def test_muon_refuses_vectors():
    with pytest.raises(ww.WaveError, match="dimensions"):
        wl.Muon([torch.nn.Parameter(torch.zeros(3))])


def central(f, x, eps=1e-5):
    g = torch.zeros_like(x)
    for i in range(x.numel()):
        hi, lo = x.clone().reshape(-1), x.clone().reshape(-1)
        hi[i] += eps
        lo[i] -= eps
        g.view(-1)[i] = (f(hi.view_as(x)) - f(lo.view_as(x))) / (2 * eps)
    return g


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_the_reference_layer_gradients_are_differences(act):
    """Central differences of step 1e-5: 1e-10 of the third derivative, and 1e-16 / 1e-5 of rounding."""
    g = torch.Generator().manual_seed(1)
    x, w, b, d = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((3, 4), (4, 5), (5,), (3, 5)))
    f = lambda x, w, b: float((R.linear(x, w, b, act)[0] * d).sum())  # noqa: E731
    dx, dw, db, _ = R.linear_backward(d, x, w, R.linear(x, w, b, act)[1], act)
    for got, want in ((dx, central(lambda t: f(t, w, b), x)), (dw, central(lambda t: f(x, t, b), w)),
                      (db, central(lambda t: f(x, w, t), b))):
        torch.testing.assert_close(got, want, rtol=0, atol=1e-8)


def test_the_reference_logp_gradient_is_a_difference():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(5, 7, generator=g, dtype=torch.float64)
    legal = torch.rand(5, 7, generator=g) < 0.7
    legal[:4, 2] = True
    legal[4, 3] = False
    tokens, d1, d2 = torch.tensor([2, 2, -1, 2, 2]), torch.randn(5, generator=g), torch.randn(5, generator=g)

    def f(t):
        r = R.token_logp(t, tokens, legal, 0.75)
        return float((r["logp"].clamp(min=-1e9) * d1).sum() + (r["entropy"] * d2).sum())
    got = R.token_logp(x, tokens, legal, 0.75, d_logp=d1, d_entropy=d2)["grad"]
    torch.testing.assert_close(got, central(f, x), rtol=0, atol=1e-8)


def test_the_reference_orthogonalise_acts_on_singular_values():
    """Its result has the update's singular vectors, and the polynomial's values of the normalised singular values."""
    g = torch.Generator().manual_seed(3)
    for shape in ((4, 9), (9, 4), (5, 5)):
        x = torch.randn(*shape, generator=g, dtype=torch.float64)
        u, s, v = torch.linalg.svd(x, full_matrices=False)
        t = s / (s.square().sum().sqrt() + 1e-7)
        for _ in range(5):
            t = 3.4445 * t - 4.7750 * t ** 3 + 2.0315 * t ** 5
        torch.testing.assert_close(R.orthogonalise(x), (u * t) @ v, rtol=0, atol=1e-5)  # float32 coefficients: 1e-7 each


def test_muon_keeps_its_momentum_in_float32_over_a_checkpoint():
    """torch casts what it loads to the parameter's type: of a bf16 weight's momentum 16 bits would be lost."""
    def optimiser():
        w = [torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.bfloat16)), torch.nn.Parameter(torch.zeros(5, 4))]
        return w, wl.Muon(w)

    (a, b), one = optimiser()
    one.state[a]["momentum"] = torch.randn(3, 4, dtype=torch.float32)
    held = one.state_dict()
    (c, d), two = optimiser()
    two.load_state_dict(held)
    got = two.state[c]["momentum"]
    assert got.dtype is torch.float32 and torch.equal(got, one.state[a]["momentum"])
    assert got.data_ptr() != one.state[a]["momentum"].data_ptr() and not two.state[d]
