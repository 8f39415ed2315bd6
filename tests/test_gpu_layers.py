"""The layer, update and log-probability operators on the device (include/wc_learn.h), through the binding, against plain
float64 code.

Tolerances. A product's sum over K is made of matrix instructions of 16 terms, added one after the other, in up to 64 runs
that are added at the end: (K / 16 + 80) additions of half a float32 ulp of the sum of magnitudes S = |x| |W|, and within an
instruction and for the parts of float32 operands as much again: 2^-23 (K / 16 + 80) S. The activation's slope is at most
1.2, its value off by 4e-6 of its argument. An output adds its type's rounding U of the value. The gradient at the
pre-activations is rounded to U before its products: U (|d_pre| |W|). Singular values: see there. Log-probabilities: a row's
log-sum is off by a few float32 ulps of the largest logit, 2e-5 as in the losses' tests. Indices and ranks are exact.
"""
import math

import pytest
import torch

import layer_ref as R
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


def say(text):
    print(text, flush=True)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def to(x):
    return None if x is None else x.to(DEV)


def within(got, want, bound, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (what, int(bad.sum()), float(off.max()), float(torch.as_tensor(bound).max()))


def strided(x, extra, fill=float("nan")):
    """x on the device with `extra` columns more per row in memory (holding `fill`), at an offset of one element."""
    rows, width = x.shape
    buf = torch.full((rows * (width + extra) + 1,), fill, dtype=x.dtype, device=DEV)
    v = buf[1:].view(rows, width + extra)[:, :width]
    v.copy_(x)
    return v


# ------------------------------------------------------------------ layers

def layer_inputs(rows, width, out, dtype, seed, bias=True, residual=True):
    g = gen(seed)
    k = {"x": torch.randn(rows, width, generator=g).to(dtype),
         "weight": (torch.randn(width, out, generator=g) * width ** -0.5).to(dtype),
         "bias": (0.3 * torch.randn(out, generator=g)).to(dtype) if bias else None,
         "residual": torch.randn(rows, out, generator=g).to(dtype) if residual else None}
    return k, torch.randn(rows, out, generator=g).to(dtype)


def rounding(want, dtype):
    return R.U[dtype] * want.abs() + R.LEAST[dtype]


def sums(k):
    return 2.0 ** -23 * (k / 16 + 80)


def check_forward(got, k, act):
    out, pre = R.linear(k["x"], k["weight"], k["bias"], act, k["residual"])
    s = k["x"].double().abs() @ k["weight"].double().abs() + (0 if k["bias"] is None else k["bias"].double().abs())
    off = sums(k["x"].shape[1]) * s
    dt = k["x"].dtype
    if got.pre is not None:
        assert got.pre.dtype == torch.float32
        within(got.pre, pre, rounding(pre, torch.float32) + off, "pre")
    # a residual's own addition: a float32 rounding of either
    more = 2.0 ** -22 * (out.abs() + pre.abs()) + 4e-6 * pre.abs()
    within(got.out, out, rounding(out, dt) + 1.2 * off + more, "out")


def check_backward(got, d, k, pre, act, dtype=None):
    x, w, dt = k["x"], k["weight"], k["x"].dtype
    dx, dw, db, dp = R.linear_backward(d, x, w, pre, act)
    # d_pre: its slope off by 4e-6, and rounded to its type for the products
    each = (4e-6 * d.double().abs() + rounding(dp, dt)) if act != "none" else torch.zeros_like(dp)
    wa, xa, da = w.double().abs(), x.double().abs(), dp.abs() + each
    if got.x is not None:
        within(got.x, dx, rounding(dx, dt) + each @ wa.t() + sums(w.shape[1]) * (da @ wa.t()), "d_x")
    if got.weight is not None:
        within(got.weight, dw, rounding(dw, dtype or dt) + xa.t() @ each + sums(len(x)) * (xa.t() @ da), "d_weight")
    if got.bias is not None:
        within(got.bias, db, 2.0 ** -24 * 300 * da.sum(0) + 4e-6 * d.double().abs().sum(0), "d_bias")


SIZES = [(1, 1, 1), (1, 8, 8), (3, 7, 5), (8, 16, 64), (5, 129, 128), (64, 64, 64), (65, 33, 67), (63, 72, 136), (2, 1000, 24),
         (130, 256, 257), (257, 65, 31), (300, 128, 567), (33, 512, 1024), (700, 40, 264), (1, 2048, 333), (9, 300, 4000)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width,out", SIZES)
def test_linear_over_sizes(rows, width, out, dtype):
    for i, act in enumerate(("none", "relu", "gelu", "silu")):
        for transposed in (False, True):
            k, d = layer_inputs(rows, width, out, TYPES[dtype], rows + width + out + i, bias=i != 0, residual=i % 2 == 0)
            say(f"case linear: {rows} x {width} x {out} {dtype} {act} transposed {transposed}")
            v = {n: to(t) for n, t in k.items()}
            if transposed:
                v["weight"] = v["weight"].t().contiguous().t()
            got = wl.linear(v["x"], v["weight"], v["bias"], act=act, residual=v["residual"], keep=i != 1)
            assert (got.pre is None) == (act in ("none", "relu"))
            check_forward(got, k, act)
            if act == "relu":
                got = got._replace(pre=wl.linear(v["x"], v["weight"], v["bias"], act="silu", keep=True).pre)
            pre = None if got.pre is None else got.pre.cpu()
            back = wl.linear_backward(to(d), v["x"], v["weight"], got.pre, act=act, bias=True)
            assert back.weight.stride() == v["weight"].stride() or 1 in (width, out)
            check_backward(back, d, k, pre, act)


@pytest.mark.parametrize("rows,width,out,dtype", [(1030, 520, 776, "bf16"), (2500, 264, 520, "f16"), (600, 333, 401, "f32"),
                                                  (20000, 96, 192, "bf16"), (20001, 97, 31, "f16"), (5000, 64, 128, "f32"),
                                                  (16, 4096, 512, "bf16"), (1, 8192, 1024, "f32"), (31, 20000, 40, "f16"),
                                                  (1, 4099, 16391, "bf16"), (7, 3001, 2057, "f16"), (13, 2500, 1029, "f32"),
                                                  (3, 70000, 65, "bf16"), (4, 512, 13000, "f32")])
def test_linear_with_larger_sizes(rows, width, out, dtype):
    k, d = layer_inputs(rows, width, out, TYPES[dtype], 7)
    say(f"case linear: {rows} x {width} x {out} {dtype}")
    v = {n: to(t) for n, t in k.items()}
    other = wl.linear(v["x"], v["weight"].t().contiguous().t(), v["bias"], residual=v["residual"], act="silu", keep=True)
    check_forward(other, k, "silu")
    got = wl.linear(**{n: v[n] for n in ("x", "weight", "bias")}, residual=v["residual"], act="silu", keep=True)
    check_forward(got, k, "silu")
    back = wl.linear_backward(to(d), v["x"], v["weight"], got.pre, act="silu", bias=True)
    check_backward(back, d, k, got.pre.cpu(), "silu")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_with_strides_and_what_lies_between_rows(dtype):
    """Rows at any stride, at an offset of one element, with NaN between them; a broadcast row; a residual in a view."""
    say(f"case linear: strides {dtype}")
    for extra in (1, 7, 8):
        k, d = layer_inputs(37, 83, 45, TYPES[dtype], extra)
        v = {n: t if t is None or n == "bias" else strided(t, extra) for n, t in k.items()}
        v["bias"] = to(k["bias"])
        got = wl.linear(v["x"], v["weight"], v["bias"], act="gelu", residual=v["residual"], keep=True)
        check_forward(got, k, "gelu")
        back = wl.linear_backward(strided(d, extra), v["x"], v["weight"], strided(got.pre.cpu(), extra), act="gelu", bias=True)
        check_backward(back, d, k, got.pre.cpu(), "gelu")
    k, _ = layer_inputs(40, 64, 64, TYPES[dtype], 3)
    for n in ("x", "residual"):
        k[n] = k[n][:1].expand(40, -1)
    got = wl.linear(to(k["x"][:1]).expand(40, -1), to(k["weight"]), to(k["bias"]), residual=to(k["residual"][:1]).expand(40, -1))
    check_forward(got, k, "none")


def test_linear_bias_and_weight_gradient_in_float32():
    k, d = layer_inputs(200, 72, 88, torch.bfloat16, 5)
    k["bias"] = k["bias"].float() + 1e-3
    v = {n: to(t) for n, t in k.items()}
    check_forward(wl.linear(v["x"], v["weight"], v["bias"], residual=v["residual"]), k, "none")
    for transposed in (False, True):
        w = v["weight"].t().contiguous().t() if transposed else v["weight"]
        back = wl.linear_backward(to(d), v["x"], w, dtype=torch.float32, bias=True)
        assert back.weight.dtype == torch.float32
        check_backward(back, d, k, None, "none", torch.float32)
        only = wl.linear_backward(to(d), v["x"], w, d_x=False, d_weight=False, bias=True)
        assert only.x is None and only.weight is None
        assert torch.equal(only.bias, back.bias)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_without_rows(dtype):
    x, w = torch.empty(0, 24, dtype=TYPES[dtype], device=DEV), torch.ones(24, 40, dtype=TYPES[dtype], device=DEV)
    assert wl.linear(x, w).out.shape == (0, 40)
    b = wl.linear_backward(torch.empty(0, 40, dtype=TYPES[dtype], device=DEV), x, w, bias=True)
    assert b.x.shape == (0, 24)
    assert torch.equal(b.weight, torch.zeros_like(w)) and torch.equal(b.bias, torch.zeros(40, device=DEV))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_keeps_infinities_and_nan_in_their_rows(dtype):
    """A row with an infinity or a NaN gives a row that is not finite, and no other; a float32 near the largest is exact."""
    say(f"case linear: infinities {dtype}")
    k, _ = layer_inputs(70, 96, 80, TYPES[dtype], 8, residual=False)
    want = wl.linear(*(to(k[n]) for n in ("x", "weight", "bias"))).out
    x = k["x"].clone()
    x[3, 5], x[40, 95] = math.inf, math.nan
    got = wl.linear(to(x), to(k["weight"]), to(k["bias"])).out
    assert not got[[3, 40]].isfinite().any()
    rest = [i for i in range(70) if i not in (3, 40)]
    assert torch.equal(got[rest], want[rest])
    top = torch.finfo(TYPES[dtype]).max
    x = torch.zeros(2, 32, dtype=TYPES[dtype])
    x[0, 0], x[1, 31] = top, -top
    got = wl.linear(to(x), torch.eye(32, dtype=TYPES[dtype], device=DEV)).out.cpu()
    assert torch.equal(got, x)


def test_linear_is_the_same_from_run_to_run_and_in_a_graph():
    """Split sums are added in a fixed order; a captured call replays on new inputs."""
    k, d = layer_inputs(300, 1153, 72, torch.bfloat16, 9)
    v = {n: to(t) for n, t in k.items()}
    d = to(d)

    def step():
        f = wl.linear(v["x"], v["weight"], v["bias"], act="gelu", residual=v["residual"], keep=True)
        return (*f, *wl.linear_backward(d, v["x"], v["weight"], f.pre, act="gelu", bias=True))

    first = [t.clone() for t in step()]
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        v["x"].copy_(to(layer_inputs(300, 1153, 72, torch.bfloat16, 20 + i)[0]["x"]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows,width,out", [(1, 40, 24), (70, 96, 80), (257, 333, 72), (1030, 520, 776), (70, 6000, 61)])
def test_linear_gradients_of_float16_past_its_largest(rows, width, out, act):
    """Of |d_out| up to 65,504 by a slope of 1.1: d_pre leaves f16's range, its products do not. Halved and doubled it is off
    by half a step of 2^-23 where it is small, 2^-24, which the bound has."""
    say(f"case linear: {rows} x {width} x {out} f16 {act}, gradients past 65,504")
    k, d = layer_inputs(rows, width, out, torch.float16, 14, residual=False)
    k["x"], k["weight"] = (1e-3 * k["x"].float()).half(), (1e-2 * k["weight"].float()).half()
    pre = torch.randn(rows, out, generator=gen(15))
    for r, j, v in ((0, 0, 65504.0), (rows // 2, out - 1, -65504.0), (rows - 1, out // 2, 61000.0)):
        d[r, j], pre[r, j] = v, {"gelu": 1.4, "silu": 2.4}[act]
    assert float((d.double() * R.slope(pre, act)).abs().max()) > 70000
    for transposed in (False, True):
        w = to(k["weight"].t().contiguous()).t() if transposed else to(k["weight"])
        for kw in ({"bias": True}, {"d_x": False}, {"d_weight": False}, {"dtype": torch.float32}):
            back = wl.linear_backward(to(d), to(k["x"]), w, to(pre), act=act, **kw)
            check_backward(back, d, k, pre, act, kw.get("dtype"))
    # what is infinite already stays so, in its own row and column
    d[rows - 1, out // 2] = math.inf
    back = wl.linear_backward(to(d), to(k["x"]), to(k["weight"]), to(pre), act=act)
    rest, columns = [i for i in range(rows - 1)], [j for j in range(out) if j != out // 2]
    assert not back.x[rows - 1].isfinite().any() and not back.weight[:, out // 2].isfinite().any()
    assert back.x[rest].isfinite().all() and back.weight[:, columns].isfinite().all()


def test_linear_gradients_of_float16_past_its_largest_in_a_graph():
    """Whether any is past is found anew in every replay."""
    k, d = layer_inputs(300, 72, 264, torch.float16, 16, residual=False)
    x, w, pre = to((1e-3 * k["x"].float()).half()), to(k["weight"]), torch.full((300, 264), 1.4, device=DEV)
    small, large = to(d), to(d)
    large = large.clone()
    large[7, 9] = 65504.0
    held_d = small.clone()

    def step():
        return wl.linear_backward(held_d, x, w, pre, act="gelu")

    want = []
    for v in (small, large):
        held_d.copy_(v)
        want.append([t.clone() for t in step()[:2]])
    assert want[1][0].isfinite().all() and want[1][1].isfinite().all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in (1, 0, 0, 1, 0):
        held_d.copy_((small, large)[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.x, want[i][0]) and torch.equal(got.weight, want[i][1])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_linear_gradients_next_to_the_largest(dtype):
    """3.4e38, which float32 holds and bf16 rounds to infinity: cut, less than a step of 2^-8 of it."""
    k, d = layer_inputs(70, 96, 80, TYPES[dtype], 17, residual=False)
    k["x"], k["weight"] = 1e-10 * k["x"], 1e-10 * k["weight"]
    pre = torch.randn(70, 80, generator=gen(18))
    # the place on the way up to the slope's maximum where it makes 3.4e38 of bf16's largest
    d[3, 5] = 3.3895313892515355e38
    lo, hi = 0.0, 1.4
    for _ in range(60):
        mid = (lo + hi) / 2
        lo, hi = (mid, hi) if float(R.slope(torch.tensor(mid), "gelu")) * float(d[3, 5]) < 3.4e38 else (lo, mid)
    pre[3, 5] = lo
    assert 3.3962e38 < float(d[3, 5]) * float(R.slope(pre[3, 5], "gelu")) < 3.4028e38
    back = wl.linear_backward(to(d), to(k["x"]), to(k["weight"]), to(pre), act="gelu", bias=True)
    assert back.x.isfinite().all() and back.weight.isfinite().all()
    check_backward(back, d, k, pre, "gelu")


@pytest.mark.parametrize("rows,width,out,dtype", [(1, 96, 200, "bf16"), (2, 4096, 40, "f16"), (300, 128, 264, "bf16"),
                                                  (1030, 520, 776, "f16"), (64, 9000, 72, "bf16"), (70, 50, 90, "f32"),
                                                  (40, 4096, 40, "f32"), (1201, 1027, 1103, "f32")])
def test_linear_over_its_residual(rows, width, out, dtype):
    """y may be the residual itself: one row, split sums, tiles, straight from memory and in parts, as into another matrix."""
    say(f"case linear: {rows} x {width} x {out} {dtype} over its residual")
    k, _ = layer_inputs(rows, width, out, TYPES[dtype], 12)
    for extra in (0, 3):
        x, w, b = to(k["x"]), to(k["weight"]), to(k["bias"])
        r = strided(k["residual"], extra)
        want = wl.linear(x, w, b, act="gelu", residual=r).out
        need = wl._linear_scratch(0, wl.DTYPES[x.dtype], 0, rows, width, out, width, out, x.data_ptr() % 16 == 0,
                                  w.data_ptr() % 16 == 0)
        work = torch.empty(need + 1, dtype=torch.uint8, device=DEV)
        s = r.stride(0) if rows > 1 else out
        wl._call("wc_linear", wl._LINEAR.pack(
            wl._LINEAR.size, 0, wl.DTYPES[x.dtype], wl.DTYPES[x.dtype], 0, rows, width, out, x.data_ptr(), width, w.data_ptr(),
            out, b.data_ptr(), r.data_ptr(), s, wl.ACTS["gelu"], 0, 0, out, r.data_ptr(), s, work.data_ptr(), need), x.device)
        assert torch.equal(r, want)


def test_linear_refuses_what_does_not_fit():
    x, w = torch.zeros(4, 16, device=DEV), torch.zeros(16, 8, device=DEV)
    for bad, word in ((lambda: wl.linear(x[0], w), "rows x width"), (lambda: wl.linear(x, w[:15]), "weight"),
                      (lambda: wl.linear(x, w.half()), "weight"), (lambda: wl.linear(x, w[:, ::2]), "weight"),
                      (lambda: wl.linear(x, w, torch.zeros(7, device=DEV)), "bias"),
                      (lambda: wl.linear(x, w, torch.zeros(8, device=DEV).half()), "bias"),
                      (lambda: wl.linear(x, w, act="tanh"), "act"), (lambda: wl.linear(x, w, residual=x), "residual"),
                      (lambda: wl.linear(x, w.cpu()), "weight"), (lambda: wl.linear(x.double(), w), "x:"),
                      (lambda: wl.linear_backward(x, x, w), "d_out"),
                      (lambda: wl.linear_backward(torch.zeros(4, 8, device=DEV), x, w, act="gelu"), "pre"),
                      (lambda: wl.linear_backward(torch.zeros(4, 8, device=DEV), x, w, dtype=torch.float16), "dtype")):
        with pytest.raises(ww.WaveError, match=word):
            bad()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_dense_under_automatic_differentiation(dtype):
    """Gradients of all four inputs, the residual and the bias broadcast, against float64 and the calls themselves."""
    k, d = layer_inputs(50, 40, 56, TYPES[dtype], 11)
    v = {n: to(t).requires_grad_(True) for n, t in k.items()}
    row = v["residual"].detach()[:1].clone().requires_grad_(True)
    y = wl.dense(v["x"], v["weight"], v["bias"], act="silu", residual=row.expand(50, -1))
    y.backward(to(d))
    pre = wl.linear(*(v[n].detach() for n in ("x", "weight", "bias")), act="silu", keep=True).pre
    got = wl.LinearGrads(v["x"].grad, v["weight"].grad, None)
    check_backward(got, d, k, pre.cpu(), "silu")
    assert v["bias"].grad.dtype == TYPES[dtype] and row.grad.shape == (1, 56)
    within(row.grad, d.double().sum(0, keepdim=True), 60 * rounding(d.double().abs().sum(0, keepdim=True), TYPES[dtype]), "row")
    x, w = (torch.randn(*s, device=DEV, requires_grad=True) for s in ((6, 5), (5, 4)))
    g, = torch.autograd.grad(wl.dense(x, w).sum(), x, create_graph=True)
    with pytest.raises(ww.WaveError, match="second"):
        g.sum().backward()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("held", ["f32", "bf16"])
@pytest.mark.parametrize("bias,residual,act", [(True, False, "gelu"), (False, True, "none"), (True, True, "silu")])
def test_dense_module_of_parameters_in_their_own_type(dtype, held, bias, residual, act):
    """Dense takes its products in x's type; the parameters' gradients come in the parameters', a float32 weight's to
    float32's own rounding."""
    dt, own = TYPES[dtype], TYPES[held]
    layer = wl.Dense(72, 88, bias=bias, act=act, gain=1.5, device=DEV, dtype=own)
    assert layer.weight.dtype == own and (layer.bias is None) == (not bias)
    assert abs(float(layer.weight.detach().float().std()) / (1.5 * 72 ** -0.5) - 1) < 0.06  # 6,336 normal values: 0.9% each
    k, d = layer_inputs(60, 72, 88, dt, 19)
    with torch.no_grad():
        k["weight"] = layer.weight.detach().cpu().to(dt)
        if bias:
            layer.bias.copy_(k["bias"])
            k["bias"] = layer.bias.detach().cpu()
            if own != torch.float32:
                k["bias"] = k["bias"].to(dt)
        else:
            k["bias"] = None
        if not residual:
            k["residual"] = None
    x = to(k["x"]).requires_grad_(True)
    r = to(k["residual"]).requires_grad_(True) if residual else None
    y = layer(x, r)
    check_forward(wl.Linear(y, None), k, act)
    y.backward(to(d))
    pre = None if act == "none" else wl.linear(to(k["x"]), to(k["weight"]), to(k["bias"]), act=act, keep=True).pre.cpu()
    assert x.grad.dtype == dt and layer.weight.grad.dtype == own
    check_backward(wl.LinearGrads(x.grad, None, None), d, k, pre, act)
    check_backward(wl.LinearGrads(None, layer.weight.grad, None), d, k, pre, act, own)
    if bias:
        assert layer.bias.grad.dtype == own
        # its sums' bound (which call makes them decides their order), and the roundings to x's type and to its own
        db = R.linear_backward(d, k["x"], k["weight"], pre, act)[2]
        size = d.double().abs().sum(0)
        off = (2.0 ** -24 * 300 * 1.2 + 4e-6) * size + (R.U[own] + (R.U[dt] if own != torch.float32 else 0.0)) * 1.01 * db.abs()
        within(layer.bias.grad, db, off, "d_bias")
    if residual:
        assert torch.equal(r.grad, to(d))


def test_dense_of_a_cast_weight_has_no_second_derivative():
    x, w = torch.randn(6, 5, device=DEV).bfloat16(), torch.randn(5, 4, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(wl.dense(x, w, act="gelu").sum(), w, create_graph=True)
    assert g.dtype == torch.float32
    with pytest.raises(ww.WaveError, match="second"):
        g.sum().backward()
    for bad in (w.double(), w.detach().int()):
        with pytest.raises(ww.WaveError, match="weight"):
            wl.dense(x, bad)


# ------------------------------------------------------------------ updates

def check_ortho(got, u, dtype, **kw):
    """Of a bf16 result beyond 128 rows and columns A (up to 1.5, which X' has times |b + 2 c A|, up to 4.8) and B (up to
    2.8) are rounded to 11 bits, 2^-12 of them: up to 10 2^-12 of X's scale in each of five steps. An element is off by no
    more than all of that, three times for one above the root mean square; as independent errors, sqrt(5) 10 2^-12 /
    sqrt(3) = 3.2e-3 of the norm, and with the result's own 2^-8 / sqrt(6) less than 2^-8. With 22 bits, 15 products'
    float32 sums over K: 15 2^-23 (K / 16 + 80) of the root mean square. And what rounds X (2^-23 of its largest element,
    and as much in a product's sum) in a direction that has no singular value grows a-fold in each step: 3.4445^5 = 485,
    times 2^-22 of the largest element of the normalised update."""
    want = R.orthogonalise(u, **kw)
    rms = want.square().mean((-2, -1), keepdim=True).sqrt()
    k = max(u.shape[-2:])
    one = dtype == torch.bfloat16 and min(u.shape[-2:]) > 128
    x = u.double().abs()
    grown = 485 * kw.get("scale", 1.0) * 2.0 ** -22 * (x.amax((-2, -1), keepdim=True) / x.square().sum((-2, -1), keepdim=True).sqrt())
    off = rounding(want, dtype) + (150 * 2.0 ** -12 if one else 15 * sums(k)) * rms + grown
    within(got, want, off, "orthogonalise")
    if one:
        assert float((got.cpu().double() - want).norm()) < 2.0 ** -8 * float(want.norm())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (17, 1), (3, 5), (8, 8), (64, 64), (63, 65), (40, 200), (200, 40), (96, 192),
                                   (3, 96, 192), (5, 33, 17), (2, 130, 70), (256, 264), (300, 700), (1, 70, 70), (0, 4, 4), (128, 128), (130, 128), (97, 161), (128, 160),
                                   (32, 1200), (1000, 30), (64, 570), (1030, 257), (131, 2000), (6, 140, 333), (500, 512),
                                   (513, 700)])
def test_orthogonalise_over_sizes(shape, dtype):
    say(f"case orthogonalise: {shape} {dtype}")
    u = (0.01 * torch.randn(*shape, generator=gen(sum(shape)))).to(TYPES[dtype])
    got = wl.orthogonalise(to(u))
    assert got.shape == u.shape and got.dtype == u.dtype
    check_ortho(got, u, u.dtype)


@pytest.mark.parametrize("shape,dtype", [((1100, 530), "bf16"), ((520, 1400), "bf16"), ((600, 600), "f32"), ((4, 520, 260), "f16")])
def test_orthogonalise_with_larger_sizes(shape, dtype):
    say(f"case orthogonalise: {shape} {dtype}")
    u = torch.randn(*shape, generator=gen(1)).to(TYPES[dtype])
    check_ortho(wl.orthogonalise(to(u)), u, u.dtype)
    # small directions beside three large ones
    g = gen(2)
    u = 1e-3 * torch.randn(*shape, generator=g)
    for _ in range(3):
        u += 0.02 * torch.randn(*shape[:-1], 1, generator=g) * torch.randn(*shape[:-2], 1, shape[-1], generator=g)
    check_ortho(wl.orthogonalise(to(u), dtype=TYPES[dtype]), u, TYPES[dtype])


def test_orthogonalise_types_strides_and_arguments():
    say("case orthogonalise: strides")
    u = torch.randn(3, 50, 90, generator=gen(2))
    wide = torch.full((3, 55, 97), math.nan, device=DEV)
    wide[:, :50, 3:93] = to(u)
    view = wide[:, :50, 3:93]
    for out in TYPES.values():
        got = wl.orthogonalise(view, dtype=out, steps=3, coefficients=(2.0, -1.5, 0.5), scale=1.7)
        assert got.dtype == out and got.is_contiguous()
        check_ortho(got, u, out, steps=3, coefficients=(2.0, -1.5, 0.5), scale=1.7)
    same = to(u[:1]).expand(4, -1, -1)
    got = wl.orthogonalise(same)
    assert torch.equal(got[0], got[3])
    # a row, a rank of one, a norm beyond float32's squares, and nothing at all
    for v in (torch.outer(torch.arange(1.0, 20), torch.arange(1.0, 33)), 1e30 * torch.randn(30, 20, generator=gen(3)),
              1e-30 * torch.randn(20, 30, generator=gen(3)).bfloat16()):
        eps = 0.0 if v.abs().max() < 1e-20 else 1e-7
        check_ortho(wl.orthogonalise(to(v), eps=eps), v, v.dtype, eps=eps)
    assert torch.equal(wl.orthogonalise(torch.zeros(9, 12, device=DEV)), torch.zeros(9, 12, device=DEV))


@pytest.mark.parametrize("shape", [(40, 60), (60, 40), (300, 700), (700, 300), (600, 700), (700, 600), (3, 20, 30)])
def test_orthogonalise_close_to_what_its_parts_hold(shape):
    """One element, and so a singular value that is an element of X, A and B: A at 62.41 and the result there, B at -62.
    X, A and B are held to 2^-22, a product leaves out as much: 62 (3 roundings + X's two + 3 of float32) 2^-22 at most. A
    bf16 result of more than 128 rows and columns has A, B and X's large part to 2^-11 each."""
    say(f"case orthogonalise: {shape} near the largest that is held")
    u = torch.zeros(shape)
    at = (*(n // 2 for n in shape),) if len(shape) == 2 else (1, 7, 29)
    u[at] = 3.0
    for out in (torch.float32, torch.bfloat16):
        one = out == torch.bfloat16 and min(shape[-2:]) > 128
        for coefficients, steps, want in (((7.9, 0.0, 0.0), 2, 62.41), ((63.0, -62.0, 0.0), 1, 1.0)):
            got = wl.orthogonalise(to(u), coefficients=coefficients, steps=steps, eps=0.0, dtype=out).cpu().double()
            off = 62 * (3 * 2.0 ** -11 if one and steps == 1 else 12 * 2.0 ** -22) + R.U[out] * want
            assert abs(float(got[at]) - want) <= off, (coefficients, out, float(got[at]))
            got[at] = 0
            if len(shape) == 2:
                assert not got.any()
            else:
                assert got[[0, 2]].isnan().all() and not got[1].any()  # 0 / 0, eps being 0


@pytest.mark.parametrize("shape,out", [((5, 33, 70), "f32"), ((70, 33), "bf16"), ((3, 140, 333), "f32"), ((3, 333, 140), "f32"),
                                       ((2, 520, 600), "bf16"), ((600, 700), "f32"), ((2050, 1, 4104), "f32")])
def test_orthogonalise_over_its_update(shape, out):
    """out may be update itself: of one type and strides, or a single matrix, as into another tensor."""
    say(f"case orthogonalise: {shape} {out} over its update")
    batch, rows, width = shape if len(shape) == 3 else (1, *shape)
    same = TYPES[out] if batch > 1 else torch.float32
    u = torch.randn(batch, rows, width, generator=gen(13)).to(same).to(DEV)
    want = wl.orthogonalise(u, dtype=TYPES[out])
    code, to_code = wl.DTYPES[same], wl.DTYPES[TYPES[out]]
    need = wl._ortho_scratch(0, code, to_code, batch, rows, width)
    work = torch.empty(need + 1, dtype=torch.uint8, device=DEV)
    wl._call("wc_orthogonalise", wl._ORTHO.pack(
        wl._ORTHO.size, 0, code, to_code, 5, batch, rows, width, u.data_ptr(), width, rows * width, u.data_ptr(), width,
        rows * width, *wl.NEWTON_SCHULZ, 1e-7, 1.0, 0, work.data_ptr(), need), u.device)
    got = u if same == TYPES[out] else u.view(-1).view(TYPES[out])[: rows * width].view(1, rows, width)
    assert torch.equal(got, want)


def test_orthogonalise_keeps_matrices_apart():
    """A NaN in one matrix of a batch makes that one NaN and leaves the others as they are alone."""
    u = torch.randn(3, 24, 40, generator=gen(4))
    u[1, 3, 3] = math.nan
    got = wl.orthogonalise(to(u))
    assert got[1].isnan().all()
    for i in (0, 2):
        check_ortho(got[i], u[i], torch.float32)
    with pytest.raises(ww.WaveError, match="columns"):
        wl.orthogonalise(torch.zeros(4, 6, device=DEV).t())
    with pytest.raises(ww.WaveError, match="steps"):
        wl.orthogonalise(torch.zeros(4, 6, device=DEV), steps=0)
    with pytest.raises(ww.WaveError, match="update"):
        wl.orthogonalise(torch.zeros(0, 6, device=DEV))


# -------------------------------------------------------- log-probabilities

def logp_inputs(rows, vocab, dtype, seed, legal):
    g = gen(seed)
    k = {"logits": (2 * torch.randn(rows, vocab, generator=g)).to(dtype),
         "tokens": torch.randint(0, vocab, (rows,), generator=g), "legal": None}
    if legal:
        k["legal"] = torch.rand(rows, vocab, generator=g) < 0.5
        k["legal"][torch.arange(rows), k["tokens"]] = True
    return k, torch.randn(rows, generator=g), torch.randn(rows, generator=g)


def check_values(got, want, what, scale=1.0):
    """2e-5 of the larger of 1 and the value; infinities and NaN alike."""
    got, want = got.detach().cpu().double(), want.double()
    odd = ~want.isfinite()
    assert torch.equal(torch.nan_to_num(got[odd], nan=7.0), torch.nan_to_num(want[odd], nan=7.0)), what
    within(torch.where(odd, 0.0, got), torch.where(odd, 0.0, want), 2e-5 * want.abs().nan_to_num(0, 0, 0).clamp(min=scale), what)


def check_logp(k, top, d1, d2, inv=0.7):
    v = {n: to(t) for n, t in k.items()}
    want = R.token_logp(**k, inv_temperature=inv, top=top, d_logp=d1, d_entropy=d2)
    got = wl.token_logp(**v, inv_temperature=inv, top=top)
    check_values(got.logp, want["logp"], "logp")
    check_values(got.entropy, want["entropy"], "entropy")
    assert torch.equal(got.rank.cpu(), want["rank"])
    if top:
        assert torch.equal(got.top_index.cpu(), want["top_index"])
        check_values(got.top_logp, want["top_logp"], "top_logp")
    grad = wl.token_logp_backward(to(d1), to(d2), v["logits"], v["tokens"], got.stats, legal=v["legal"], inv_temperature=inv)
    w, dt = want["grad"], k["logits"].dtype
    within(grad, w, rounding(w, dt) + 2e-5 * max(1e-3, float(w.abs().max())), "grad")
    return got


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 8), (3, 22), (65, 7), (2, 64), (5, 63), (5, 65), (130, 97), (7, 511), (4, 513),
                                        (7, 1000), (3, 2049), (4, 4099), (300, 567), (2, 9001), (1, 20011)])
def test_token_logp_over_sizes(rows, vocab, dtype):
    for legal, top in ((False, 0), (True, 5), (False, 20)):
        say(f"case logp: {rows} x {vocab} {dtype} legal {legal} top {top}")
        k, d1, d2 = logp_inputs(rows, vocab, TYPES[dtype], rows + vocab, legal)
        if rows > 2:
            k["tokens"][1], k["tokens"][2] = -1, vocab  # left out
        check_logp(k, top, d1, d2)


@pytest.mark.parametrize("rows,vocab,dtype,top", [(2, 131072, "bf16", 20), (300, 16500, "f16", 3), (520, 9000, "f32", 1),
                                                  (1030, 8193, "f32", 2), (64, 40000, "bf16", 64)])
def test_token_logp_with_a_large_vocabulary(rows, vocab, dtype, top):
    """Against float64 torch over whole rows (the row-by-row code is for small ones)."""
    say(f"case logp: {rows} x {vocab} {dtype} top {top}")
    k, d1, d2 = logp_inputs(rows, vocab, TYPES[dtype], vocab, False)
    v = {n: to(t) for n, t in k.items()}
    x = k["logits"].double()
    logp = torch.log_softmax(x, 1)
    p = logp.exp()
    h = -(p * logp).sum(1)
    a = k["tokens"][:, None]
    got = wl.token_logp(v["logits"], v["tokens"], top=top)
    check_values(got.logp, logp.gather(1, a)[:, 0], "logp")
    check_values(got.entropy, h, "entropy")
    order = torch.sort(x, dim=1, descending=True, stable=True)
    assert torch.equal(got.top_index.cpu().long(), order.indices[:, :top])
    check_values(got.top_logp, logp.gather(1, order.indices[:, :top]), "top_logp")
    assert torch.equal(got.rank.cpu().long(), (order.indices == a).int().argmax(1))
    w = -p * (d1[:, None].double() + d2[:, None].double() * (logp + h[:, None]))
    w.scatter_add_(1, a, d1[:, None].double())
    grad = wl.token_logp_backward(to(d1), to(d2), v["logits"], v["tokens"], got.stats)
    within(grad, w, rounding(w, TYPES[dtype]) + 2e-5 * w.abs().max(), "grad")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [40, 700, 5000, 30000])
def test_token_logp_of_equal_and_ordered_logits(vocab, dtype):
    """Ties go to the lowest index: rows of one value, of few values, ascending, descending, with zeros of both signs, and
    with the largest side by side."""
    say(f"case logp: ties {vocab} {dtype}")
    n = torch.arange(vocab)
    x = torch.stack([torch.zeros(vocab), (n % 3).float(), n / vocab, -n / vocab, torch.where(n % 2 == 0, 0.0, -0.0),
                     torch.where((n >= vocab // 2) & (n < vocab // 2 + 30), 4.0, 0.0), torch.where(n % 256 == 7, 2.0, 1.0)])
    k = {"logits": x.to(TYPES[dtype]), "tokens": torch.tensor([vocab - 1, 5, 0, 7, 9, vocab // 2 + 3, 8]), "legal": None}
    check_logp(k, 20, torch.ones(7), torch.ones(7))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [30, 600, 20000])
def test_token_logp_of_masks_infinities_and_nan(vocab, dtype):
    say(f"case logp: masks {vocab} {dtype}")
    dt = TYPES[dtype]
    least = torch.finfo(dt).min
    k, d1, d2 = logp_inputs(9, vocab, dt, 3, True)
    x, on, a = k["logits"], k["legal"], k["tokens"]
    a[:] = 4
    on[:, 4] = True
    on[0] = False                       # nothing legal: left out
    on[1] = False
    on[1, 4] = True                     # one alone
    on[2, 4] = False                    # the token is not legal: -infinity
    x[3, 4] = -math.inf                 # nor has this one a probability
    x[4] = least                        # a mask's lowest value everywhere
    x[5, 1:] = least                    # and everywhere but once
    on[5, 0] = True
    x[6] = -math.inf                    # legal, but nothing above -infinity
    x[7][~on[7]] = math.nan             # what is illegal may be anything
    x[8][~on[8]] = math.inf
    got = check_logp(k, 6, d1, d2)
    assert got.logp[2] == -math.inf and got.logp[3] == -math.inf and got.rank[0] == -1 and got.rank[6] == -1
    # a legal NaN or +infinity: NaN, the other rows as they were
    on[1, 5] = on[7, 5] = True
    x[1, 5], x[7, 5] = math.nan, math.inf
    again = wl.token_logp(to(x), to(a), legal=to(on), inv_temperature=0.7, top=6)
    assert again.logp[[1, 7]].isnan().all() and again.entropy[[1, 7]].isnan().all()
    rest = [0, 2, 3, 4, 5, 6, 8]
    for one, two in zip(got, again):
        assert torch.equal(one[rest], two[rest])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [2, 7, 15, 19, 30, 135, 603, 5003, 20007])
def test_token_logp_rank_of_a_token_without_a_probability(vocab, dtype):
    """At -infinity or not legal, in every place of the last columns, which a whole load does not reach, and before them:
    each column above -infinity comes before it once, and each other of a lower index."""
    say(f"case logp: ranks of tokens at -infinity {vocab} {dtype}")
    at = [c for c in (0, 1, vocab // 2, *range(vocab - 9, vocab)) if 0 <= c < vocab]
    for legal in (False, True):
        k, d1, d2 = logp_inputs(len(at), vocab, TYPES[dtype], vocab, legal)
        k["tokens"] = torch.tensor(at)
        x = k["logits"]
        x[torch.rand(x.shape, generator=gen(22)) < 0.3] = -math.inf
        for r, a in enumerate(at):
            if legal and r % 2:
                k["legal"][r, a] = False
            else:
                x[r, a] = -math.inf
        check_logp(k, 3, d1, d2)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("vocab", [13, 60, 600, 5003, 20001])
def test_token_logp_gradient_of_illegal_columns_is_zero_whatever_the_row(vocab, dtype):
    """A legal NaN or infinity makes the row's legal columns NaN, those at -infinity aside, which have none anyway; what
    arrives infinite or as NaN has no effect on illegal columns either. The other rows are as without these."""
    say(f"case logp: gradients of spoiled rows {vocab} {dtype}")
    k, d1, d2 = logp_inputs(7, vocab, TYPES[dtype], vocab, True)
    x, on, a = k["logits"], k["legal"], k["tokens"]
    on[:, :4] = torch.tensor([False, True, True, True])
    a[:] = 2
    calm = {n: to(t.clone()) for n, t in k.items()}
    x[1, 1], x[2, 1], x[2, 0], x[5, 1], x[5, 2] = math.nan, math.inf, math.nan, math.nan, -math.inf
    for d_entropy in (None, d2):
        e1, e2 = d1.clone(), None if d_entropy is None else d_entropy.clone()
        e1[3], e1[4] = math.nan, math.inf
        got = wl.token_logp(to(x), to(a), legal=to(on))
        g = wl.token_logp_backward(to(e1), to(e2), to(x), to(a), got.stats, legal=to(on)).cpu()
        assert not g[~on].any(), g[~on].isnan().sum()
        for r in (1, 2, 5):
            assert g[r][on[r] & (x[r] != -math.inf)].isnan().all(), r
        before = wl.token_logp_backward(to(d1), to(d2) if d_entropy is not None else None, calm["logits"], calm["tokens"],
                                        wl.token_logp(**calm).stats, legal=calm["legal"]).cpu()
        assert torch.equal(g[[0, 6]], before[[0, 6]])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,loads,threads", [(300, 4, 256), (300, 8, 256), (300, 8, 512), (3, 1, 256), (3, 2, 256)])
def test_token_logp_alternatives_where_all_that_a_thread_holds_is_nan(rows, loads, threads, dtype):
    """A NaN is no alternative, and does not stand in the way of the others: here all of one thread's columns, the single one
    behind the last whole load among them."""
    each = 16 // TYPES[dtype].itemsize
    vocab = loads * threads * each + 1
    say(f"case logp: {rows} x {vocab} {dtype}, a thread's columns NaN")
    for top in (1, 2, 20):
        k, _, _ = logp_inputs(3, vocab, TYPES[dtype], vocab, False)
        for c in range(loads):
            k["logits"][1, c * threads * each: c * threads * each + each] = math.nan
        k["logits"][1, vocab - 1] = math.nan
        x = k["logits"].double().nan_to_num(nan=-math.inf)
        want = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        at = torch.arange(rows) % 3
        got = wl.token_logp(to(k["logits"][at]), to(k["tokens"][at]), top=top)
        assert torch.equal(got.top_index.cpu().long(), want[at])
        assert got.logp[1].isnan() and got.logp[0].isfinite()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_token_logp_with_strides_and_without_tokens(dtype):
    say(f"case logp: strides {dtype}")
    k, d1, d2 = logp_inputs(40, 301, TYPES[dtype], 6, True)
    v = {"logits": strided(k["logits"], 3), "legal": strided(k["legal"], 5, True), "tokens": to(k["tokens"]).int()}
    got = wl.token_logp(**v, top=4)
    base = wl.token_logp(**{n: to(t) for n, t in k.items()}, top=4)
    for one, two in zip(got, base):
        assert torch.equal(one, two)
    none = wl.token_logp(v["logits"], legal=v["legal"], top=4)
    assert none.logp is None and none.rank is None
    assert torch.equal(none.entropy, base.entropy) and torch.equal(none.top_index, base.top_index)
    grad = strided(torch.zeros(40, 301, dtype=TYPES[dtype]), 3)
    wl.token_logp_backward(to(d1), to(d2), v["logits"], v["tokens"], got.stats, legal=v["legal"], grad=grad)
    want = wl.token_logp_backward(to(d1), to(d2), to(k["logits"]), to(k["tokens"]), base.stats, legal=to(k["legal"]))
    assert torch.equal(grad, want)
    # over the logits themselves, and one row for all
    x = to(k["logits"]).clone()
    wl.token_logp_backward(to(d1), to(d2), x, to(k["tokens"]), base.stats, legal=to(k["legal"]), grad=x)
    assert torch.equal(x, want)
    one = to(k["logits"][:1]).expand(40, -1)
    many = wl.token_logp(one, v["tokens"], top=2)
    assert torch.equal(many.entropy, many.entropy[:1].expand(40)) and (many.top_index == many.top_index[:1]).all()


def test_token_logp_without_rows_and_refusals():
    x = torch.zeros(0, 7, device=DEV)
    got = wl.token_logp(x, torch.zeros(0, dtype=torch.int64, device=DEV), top=3)
    assert got.logp.shape == (0,) and got.top_index.shape == (0, 3)
    x, t = torch.zeros(4, 7, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad, word in ((lambda: wl.token_logp(x, t[:3]), "tokens"), (lambda: wl.token_logp(x, t.float()), "tokens"),
                      (lambda: wl.token_logp(x, t, top=65), "top"), (lambda: wl.token_logp(x, t, legal=x), "legal"),
                      (lambda: wl.token_logp(x, t, inv_temperature=-1.0), "inv_temperature"),
                      (lambda: wl.token_logp(x.t(), t[:1].expand(7)), "columns"),
                      (lambda: wl.token_logp_backward(None, None, x, t, None), "stats"),
                      (lambda: wl.token_logp_backward(x, None, x, t, torch.zeros(4, 4, device=DEV)), "d_logp")):
        with pytest.raises(ww.WaveError, match=word):
            bad()


def test_token_logp_objective_and_its_graph():
    """Gradients through logp and entropy; a captured forward and backward pass replays on new logits."""
    k, d1, d2 = logp_inputs(64, 567, torch.float32, 12, True)
    x = to(k["logits"]).requires_grad_(True)
    logp, entropy, rank, top_logp, top_index = wl.token_logp_objective(x, to(k["tokens"]), legal=to(k["legal"]), top=2)
    assert not top_logp.requires_grad and not rank.requires_grad
    (logp * to(d1)).sum().backward(retain_graph=True)
    want = R.token_logp(**k, d_logp=d1)["grad"]
    within(x.grad, want, 2e-5 * want.abs().max(), "logp's")
    x.grad = None
    ((logp * to(d1)).sum() + (entropy * to(d2)).sum()).backward()
    want = R.token_logp(**k, d_logp=d1, d_entropy=d2)["grad"]
    within(x.grad, want, 2e-5 * want.abs().max(), "both's")
    raw, t, on, d1, d2 = x.detach(), to(k["tokens"]), to(k["legal"]), to(d1), to(d2)

    def step():
        r = wl.token_logp(raw, t, legal=on, top=3)
        return r.logp, r.top_index, wl.token_logp_backward(d1, d2, raw, t, r.stats, legal=on)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        raw.copy_(to(logp_inputs(64, 567, torch.float32, 30 + i, True)[0]["logits"]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ far places

def far(x, stride):
    """x on the device with rows `stride` elements apart; what lies between is not written."""
    buf = torch.empty(len(x) * stride, dtype=x.dtype, device=DEV)
    v = buf.view(len(x), stride)[:, : x.shape[1]]
    v.copy_(x)
    return v


@pytest.mark.parametrize("stride", [4_000_000, 4_000_004])
def test_linear_with_rows_whose_offsets_pass_32_bits(stride):
    """2.4e9 elements from the first row to the last: read where they lie (whole 16 bytes), and copied."""
    say(f"case linear: row stride {stride}")
    k, d = layer_inputs(600, 72, 40, torch.bfloat16, 41)
    v = {n: to(t) for n, t in k.items()}
    x = far(k["x"], stride)
    got = wl.linear(x, v["weight"], v["bias"], act="gelu", residual=v["residual"], keep=True)
    check_forward(got, k, "gelu")
    check_backward(wl.linear_backward(to(d), x, v["weight"], got.pre, act="gelu", bias=True), d, k, got.pre.cpu(), "gelu")
    few = far(k["x"][:2], 2_200_000_000)
    check_forward(wl.linear(few, v["weight"], v["bias"]), {n: t[:2] if n in ("x",) else t if n != "residual" else None
                                                           for n, t in k.items()}, "none")


def test_linear_whose_result_passes_32_bits():
    """1,100,000 x 2,048: the last rows, and the gradients' against the first thousand rows alone."""
    say("case linear: 1,100,000 x 16 x 2,048")
    k, _ = layer_inputs(300, 16, 2048, torch.bfloat16, 42, residual=False)
    x = to(k["x"]).repeat(1_100_000 // 300 + 1, 1)[:1_100_000]
    w, b = to(k["weight"]), to(k["bias"])
    got = wl.linear(x, w, b, act="silu", keep=True)
    at = torch.tensor([0, 299, 1_048_576, 1_099_999])
    part = {"x": x[at.to(DEV)].cpu(), "weight": k["weight"], "bias": k["bias"], "residual": None}
    check_forward(wl.Linear(got.out[at.to(DEV)], got.pre[at.to(DEV)]), part, "silu")
    back = wl.linear_backward(got.out, x, w, got.pre, act="silu", d_weight=False)
    check_backward(wl.LinearGrads(back.x[at.to(DEV)], None, None), got.out[at.to(DEV)].cpu(), part, got.pre[at.to(DEV)].cpu(), "silu")


def test_token_logp_with_rows_whose_offsets_pass_32_bits():
    say("case logp: far rows")
    for vocab in (300, 30000):
        k, d1, d2 = logp_inputs(40, vocab, torch.float16, vocab, True)
        v = {n: to(t) for n, t in k.items()}
        base = wl.token_logp(**v, top=4)
        x, on = far(k["logits"], 60_000_000), far(k["legal"], 60_000_000)
        got = wl.token_logp(x, v["tokens"], legal=on, top=4)
        for one, two in zip(got, base):
            assert torch.equal(one, two)
        want = wl.token_logp_backward(to(d1), to(d2), v["logits"], v["tokens"], base.stats, legal=v["legal"])
        wl.token_logp_backward(to(d1), to(d2), x, v["tokens"], got.stats, legal=on, grad=x)
        assert torch.equal(x, want)


def test_orthogonalise_with_matrices_whose_offsets_pass_32_bits():
    say("case orthogonalise: far matrices")
    for shape in ((3, 40, 60), (3, 140, 200), (2, 600, 700)):
        u = torch.randn(*shape, generator=gen(7))
        buf = torch.empty(shape[0] * 1_200_000_000, dtype=torch.float32, device=DEV)
        v = torch.as_strided(buf, shape, (1_200_000_000, 1_000_001, 1))
        v.copy_(u)
        assert torch.equal(wl.orthogonalise(v), wl.orthogonalise(to(u)))
        del buf, v


# ---------------------------------------------- more than one launch's threads

def test_linear_of_more_rows_than_a_launch_has_threads_for_in_small_tiles():
    """2^30 rows in tiles of 64 would be 2^32 threads. One row again and again: every result is the first's."""
    say("case linear: 1,073,741,894 x 8 x 1")
    rows = 2 ** 30 + 70
    k, d = layer_inputs(1, 8, 1, torch.bfloat16, 43, residual=False)
    v = {n: to(t) for n, t in k.items()}
    got = wl.linear(v["x"].expand(rows, -1), v["weight"], v["bias"], act="silu").out
    check_forward(wl.Linear(got[-1:], None), k, "silu")
    assert got.min() == got.max() == got[0, 0]
    del got
    grad = wl.linear_backward(to(d).expand(rows, -1), v["x"].expand(rows, -1), v["weight"], d_weight=False).x
    within(grad[-1:], d.double() @ k["weight"].double().t(), 2.0 ** -7 * (d.double() @ k["weight"].double().t()).abs(), "d_x")
    for part in grad.split(2 ** 27):
        assert torch.equal(part[:1], part[-1:]) and bool((part.amin(0) == part.amax(0)).all())


def test_linear_in_float32_of_more_rows_than_a_launch_has_threads_for():
    """2^28 rows straight from memory are 2^23 fragments of 512 threads, 2^32. One row again and again, with a residual of
    its own each; x's gradient alone, and beside the weight's."""
    say("case linear: 268,435,526 x 64 x 1 f32")
    rows = 2 ** 28 + 70
    k, _ = layer_inputs(1, 64, 1, torch.float32, 45, residual=False)
    v = {n: to(t) for n, t in k.items()}
    residual = (torch.arange(rows, device=DEV, dtype=torch.int32) % 1024).float()[:, None]
    got = wl.linear(v["x"].expand(rows, -1), v["weight"], v["bias"], act="silu", residual=residual, keep=True)
    check_forward(wl.Linear(got.out[:1], got.pre[:1]), k, "silu")
    assert got.pre.min() == got.pre.max()
    assert float((got.out - residual - got.out[0]).abs().max()) <= 2.0 ** -13  # half an ulp of 1,025, and of the difference
    del got, residual
    say("case linear: 268,435,526 x 1 x 100 f32, x's gradient")
    k, d = layer_inputs(1, 1, 100, torch.float32, 46)
    grad = wl.linear_backward(to(d).expand(rows, -1), to(k["x"]).expand(rows, -1), to(k["weight"]), d_weight=False).x
    check_backward(wl.LinearGrads(grad[-1:], None, None), d, k, None, "none")
    assert grad.min() == grad.max()
    del grad
    say("case linear: 268,435,526 x 32 x 200 f32, both gradients")
    k, d = layer_inputs(1, 32, 200, torch.float32, 47)
    back = wl.linear_backward(to(d).expand(rows, -1), to(k["x"]).expand(rows, -1), to(k["weight"]))
    check_backward(wl.LinearGrads(back.x[-1:], None, None), d, k, None, "none")
    for part in back.x.split(2 ** 26):
        assert torch.equal(part[:1], part[-1:]) and bool((part.amin(0) == part.amax(0)).all())


@pytest.mark.parametrize("rows,vocab", [(2 ** 22 + 3, 12), (2 ** 22 // 5 + 3, 70000)])
def test_token_logp_of_more_rows_than_one_launch_takes(rows, vocab):
    """The rows behind the first launch's have their own tokens, masks and gradients."""
    say(f"case logp: {rows} x {vocab}")
    k, d1, d2 = logp_inputs(6, vocab, torch.bfloat16, vocab, False)
    on = torch.rand(6, vocab, generator=gen(1)) < 0.5
    on[torch.arange(6), k["tokens"]] = True
    x, a, legal = to(k["logits"]), to(k["tokens"]), to(on)
    want = wl.token_logp(x[:1].expand(6, -1), a, legal=legal[:1].expand(6, -1), top=3)
    last = torch.arange(rows, device=DEV) % 6
    got = wl.token_logp(x[:1].expand(rows, -1), a[last], legal=legal[:1].expand(rows, -1), top=3)
    for n in ("logp", "rank", "top_index", "entropy", "top_logp"):
        one, two = getattr(got, n), getattr(want, n)[last]
        if n in ("rank", "top_index"):
            assert torch.equal(one, two), n
        else:  # another cut of the row: the sums' own tolerance
            assert bool(((one - two).abs().nan_to_num(0.0) <= 4e-5 * two.abs().clamp(min=1)).all()), n
            assert torch.equal(one.isinf(), two.isinf())
    if vocab < 100:
        grad = wl.token_logp_backward(to(d1)[last], to(d2)[last], x[:1].expand(rows, -1), a[last], got.stats,
                                      legal=legal[:1].expand(rows, -1))
        few = wl.token_logp_backward(to(d1), to(d2), x[:1].expand(6, -1), a, want.stats, legal=legal[:1].expand(6, -1))
        assert torch.equal(grad, few[last])


@pytest.mark.parametrize("shape", [(2050, 1, 4104), (2050, 130, 132)])
def test_orthogonalise_of_more_matrices_than_one_launch_takes(shape):
    say(f"case orthogonalise: {shape}")
    at = [0, 1, 2046, 2047, 2048, 2049]
    u = torch.randn(*shape, generator=gen(44))
    check_ortho(wl.orthogonalise(to(u))[at], u[at], u.dtype)
    v = to(u)[:, :, : shape[2] - 1]
    check_ortho(wl.orthogonalise(v, dtype=torch.bfloat16)[at], u[at][:, :, : shape[2] - 1], torch.bfloat16)


@pytest.mark.parametrize("act", ["none", "gelu"])
@pytest.mark.parametrize("rows,width,out", [(64, 2600, 70), (5000, 40, 64), (1024, 512, 512), (1024, 1024, 1024), (70, 4096, 2048),
                                            (300, 300, 4100), (2500, 1, 1), (40, 9, 6000)])
def test_linear_in_float32_with_each_gradient_alone(rows, width, out, act):
    """Straight from memory or in parts, summed in one run or several, by sizes and by what is wanted."""
    say(f"case linear: {rows} x {width} x {out} f32 {act}, gradients one at a time")
    k, d = layer_inputs(rows, width, out, torch.float32, rows + width)
    v = {n: to(t) for n, t in k.items()}
    for transposed in (False, True):
        w = v["weight"].t().contiguous().t() if transposed else v["weight"]
        got = wl.linear(v["x"], w, v["bias"], residual=v["residual"], act=act, keep=True)
        check_forward(got, k, act)
        pre = None if got.pre is None else got.pre.cpu()
        for kw in ({"d_weight": False}, {"d_x": False}, {"d_x": False, "bias": True}, {"d_weight": False, "bias": True},
                   {"bias": True}, {"d_x": False, "d_weight": False, "bias": True}):
            back = wl.linear_backward(to(d), v["x"], w, got.pre, act=act, **kw)
            for value, name in ((back.x, "d_x"), (back.weight, "d_weight")):
                assert (value is not None) == kw.get(name, True)
            check_backward(back, d, k, pre, act)


@pytest.mark.parametrize("rows,width,out", [(1201, 1027, 1103), (701, 2053, 1301)])
@pytest.mark.parametrize("layout", ["as they come", "strided", "transposed", "transposed and strided", "broadcast"])
def test_linear_in_float32_parts_of_odd_sizes_strides_and_layouts(rows, width, out, layout):
    """Sizes that are taken in parts whatever is wanted, with a remainder of k in each product: zeros are laid behind it. The
    scratch tells the way: the copies in parts are six bytes an element."""
    say(f"case linear: {rows} x {width} x {out} f32 in parts, {layout}")
    k, d = layer_inputs(rows, width, out, torch.float32, 21)
    if layout == "broadcast":
        k["x"] = k["x"][:1].expand(rows, -1)
    v = {n: to(t) for n, t in k.items()}
    d_out = to(d)
    if "strided" in layout:
        v["x"], v["residual"], d_out = strided(k["x"], 7), strided(k["residual"], 3), strided(d, 1)
        v["weight"] = strided(k["weight"].t(), 5).t() if "transposed" in layout else strided(k["weight"], 5)
    elif layout == "transposed":
        v["weight"] = v["weight"].t().contiguous().t()
    elif layout == "broadcast":
        v["x"], d_out = v["x"][:1].expand(rows, -1), d_out[:1].expand(rows, -1)
        d = d[:1].expand(rows, -1)
    got = wl.linear(v["x"], v["weight"], v["bias"], act="gelu", residual=v["residual"], keep=True)
    check_forward(got, k, "gelu")
    pre = strided(got.pre.cpu(), 2) if "strided" in layout else got.pre
    for kw in ({"bias": True}, {"d_weight": False}, {"d_x": False}):
        check_backward(wl.linear_backward(d_out, v["x"], v["weight"], pre, act="gelu", **kw), d, k, got.pre.cpu(), "gelu")
    transposed = int("transposed" in layout)
    ws = v["weight"].stride(1 if transposed else 0)
    assert wl._linear_scratch(0, 0, transposed, rows, width, out, v["x"].stride(0), ws, False, False) >= 6 * (rows + out) * width
    for dx, dw in ((True, True), (True, False), (False, True)):
        assert wl._linear_back_scratch(0, 0, transposed, wl.ACTS["gelu"], rows, width, out, d_out.stride(0), v["x"].stride(0), ws, False,
                                       False, False, dx, dw, dx and dw) >= 6 * rows * out


def test_linear_in_float32_parts_of_infinities_and_of_the_largest():
    """Sizes that are taken in parts: as the small ones."""
    say("case linear: infinities f32, 1,200 x 1,024 x 1,100")
    k, _ = layer_inputs(1200, 1024, 1100, torch.float32, 8, residual=False)
    want = wl.linear(*(to(k[n]) for n in ("x", "weight", "bias"))).out
    x = k["x"].clone()
    x[3, 5], x[40, 1000] = math.inf, math.nan
    got = wl.linear(to(x), to(k["weight"]), to(k["bias"])).out
    assert not got[[3, 40]].isfinite().any()
    rest = [i for i in range(1200) if i not in (3, 40)]
    assert torch.equal(got[rest], want[rest])
    top = torch.finfo(torch.float32).max
    x = torch.zeros(1200, 1024)
    x[0, 0], x[1199, 1023] = top, -top
    w = torch.zeros(1024, 1100)
    w[0, 7] = w[1023, 1099] = 1.0
    got = wl.linear(to(x), to(w)).out.cpu()
    assert got[0, 7] == top and got[1199, 1099] == -top and int((got != 0).sum()) == 2
