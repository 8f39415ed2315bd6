"""The training operators under torch's automatic differentiation, and the training example end to end."""
import pytest
import torch

import learn_ref as R
import train_policy
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


def close(got, want, what, bound):
    off = float((got.double().cpu() - want.double().cpu()).abs().max())
    assert off <= bound * max(1.0, float(want.abs().max())), (what, off)


def test_objectives_scale_with_what_arrives_and_may_run_backward_twice():
    """Gradients of 3 times the loss, twice over one graph, against the call's own gradient (the same float32 sums: 1e-6)."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(40, 30, generator=g, device=DEV, requires_grad=True)
    a = torch.randint(0, 30, (40,), generator=g, device=DEV)
    v = torch.randn(40, generator=g, device=DEV)
    b = torch.log_softmax(x.detach(), 1).gather(1, a[:, None])[:, 0].contiguous()
    loss, *_ = wl.policy_objective(x, a, b, v, ref_logits=torch.zeros_like(x), kl_coef=0.2)
    want = wl.policy_loss(x.detach(), a, b, v, ref_logits=torch.zeros(40, 30, device=DEV), kl_coef=0.2)
    (3 * loss).backward(retain_graph=True)
    close(x.grad, 3 * want.grad, "policy", 1e-6)
    (3 * loss).backward()
    close(x.grad, 6 * want.grad, "policy twice", 2e-6)
    x.grad = None
    offsets = torch.tensor([0, 10, 20, 25, 40], device=DEV)
    loss, *_ = wl.preference_objective(x, a, offsets, b, beta=0.4)
    (2 * loss).backward()
    close(x.grad, 2 * wl.preference_loss(x.detach(), a, offsets, b, beta=0.4).grad, "preference", 1e-6)


@pytest.mark.parametrize("norm,gate_act", [("layer", "none"), ("rms", "sigmoid")])
def test_residual_norm_module_against_float64(norm, gate_act):
    """As the operator's own test: 2e-5 of the largest for float32."""
    m = wl.ResidualNorm(72, norm=norm, gate_act=gate_act, scale=0.3, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn(p.shape, generator=g, device=DEV))
    u, x, d1, d2 = (torch.randn(33, 72, generator=g, device=DEV) for _ in range(4))
    u.requires_grad_(True)
    x.requires_grad_(True)
    torch.autograd.backward(m(u, x), [d1, d2])
    v = {n: None if t is None else t.detach().cpu().double().requires_grad_(True) for n, t in (
        ("block", u), ("stream", x), ("post_gain", m.post_gain), ("post_bias", m.post_bias), ("gate", m.gate),
        ("pre_gain", m.pre_gain), ("pre_bias", m.pre_bias))}
    torch.autograd.backward(R.residual_norm(**v, **m.kw), [d1.cpu().double(), d2.cpu().double()])
    close(u.grad, v["block"].grad, "block", 2e-5)
    close(x.grad, v["stream"].grad, "stream", 2e-5)
    for n, p in m.named_parameters():
        close(p.grad, v[n].grad, n, 2e-5 * 33 ** 0.5)


def test_act_linear8_against_float64():
    """Forward from the unrounded input; the gradients from what the 8 bits stand for. bf16 outputs: 2^-8 of the value
    and of what is summed."""
    g = torch.Generator(device=DEV).manual_seed(3)
    z = torch.randn(130, 96, generator=g, device=DEV).bfloat16().requires_grad_(True)
    w = (0.1 * torch.randn(96, 40, generator=g, device=DEV)).bfloat16().requires_grad_(True)
    d = torch.randn(130, 40, generator=g, device=DEV).bfloat16()
    y = wl.act_linear8(z, w, "gelu")
    y.backward(d)
    close(y.detach(), R.act(z.detach().cpu().double(), "gelu") @ w.detach().cpu().double(), "y", 2.0 ** -7)
    kept = R.keep8(z.detach().cpu())[2].requires_grad_(True)
    da = d.cpu().double() @ w.detach().cpu().double().t()
    R.act(kept, "gelu").backward(da)
    close(z.grad, kept.grad, "z", 2.0 ** -6)
    close(w.grad, R.act(kept.detach(), "gelu").t() @ d.cpu().double(), "w", 2.0 ** -7)


def test_the_training_example_learns_the_search_policy():
    first, last, pref, pref_last = train_policy.train(trees=2, steps=40, width=128, blocks=2)
    assert last < 0.5 * first
    assert pref_last < 0.8 * pref


def objective_inputs(vocab=32):
    g = torch.Generator(device=DEV).manual_seed(4)
    rows = 12
    draw = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    k = {"actions": torch.randint(0, vocab, (rows,), generator=g, device=DEV), "behaviour_logp": draw(rows) - 3,
         "advantages": draw(rows), "weights": torch.rand(rows, generator=g, device=DEV) + 0.1,
         "legal": torch.ones(rows, vocab, dtype=torch.bool, device=DEV), "ref_logits": draw(rows, vocab)}
    p = {"tokens": k["actions"].clone(), "offsets": torch.tensor([0, 3, 6, 8, 12], device=DEV), "ref_logp": draw(rows) - 3,
         "weights": k["weights"].clone()}
    return draw(rows, vocab).requires_grad_(True), k, p


@pytest.mark.parametrize("which,name", [(0, n) for n in ("logits", "actions", "behaviour_logp", "advantages", "weights",
                                                         "legal", "ref_logits", "ref_logp")] +
                         [(1, n) for n in ("logits", "tokens", "offsets", "ref_logp", "weights")])
def test_an_objective_whose_batch_was_written_since_refuses_its_backward_pass(which, name):
    """What the backward pass would read again belongs to another batch then."""
    x, k, p = objective_inputs()
    if name == "ref_logp" and which == 0:
        k["ref_logits"] = None
        k["ref_logp"] = p["ref_logp"]
    call, kw = ((wl.policy_objective, k), (wl.preference_objective, p))[which]
    loss, *_ = call(x, **kw, **({"kl_coef": 0.1} if which == 0 else {}))
    with torch.no_grad():
        t = x if name == "logits" else kw[name]
        t.copy_(t.clone())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_objectives_of_a_batch_left_alone_after_other_calls():
    """Two losses over one batch, backward in the other order: each its own gradient (the same float32 sums: 1e-6)."""
    x, k, p = objective_inputs()
    one, *_ = wl.policy_objective(x, **k, kl_coef=0.1, entropy_coef=0.01)
    two, *_ = wl.preference_objective(x, **p, kind="squared")
    two.backward()
    close(x.grad, wl.preference_loss(x.detach(), **p, kind="squared").grad, "preference", 1e-6)
    x.grad = None
    one.backward()
    close(x.grad, wl.policy_loss(x.detach(), **k, kl_coef=0.1, entropy_coef=0.01).grad, "policy", 1e-6)


@pytest.mark.parametrize("which", ["policy", "preference", "norm", "act_linear8"])
def test_second_derivatives_are_refused(which):
    """The gradient itself is given with create_graph too; differentiating it again raises instead of giving 0."""
    x, k, p = objective_inputs()
    if which == "policy":
        y = wl.policy_objective(x, **k, kl_coef=0.1)[0]
    elif which == "preference":
        y = wl.preference_objective(x, **p)[0]
    elif which == "norm":
        y = (wl.ResidualNorm(32, device=DEV)(x, torch.zeros_like(x))[1] * k["ref_logits"]).sum()
    else:
        y = (wl.act_linear8(x, torch.ones(32, 9, device=DEV), "relu") ** 2).sum()
    [want] = torch.autograd.grad(y, x, retain_graph=True)
    [got] = torch.autograd.grad(y, x, create_graph=True)
    assert torch.equal(got.detach(), want) and want.any() and got.requires_grad
    with pytest.raises(ww.WaveError, match="second derivative"):
        torch.autograd.grad((got ** 2).sum(), x, retain_graph=True)
    with pytest.raises(ww.WaveError, match="second derivative"):
        (got ** 2).sum().backward()


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_act_linear8_of_every_type_and_activation(dtype, act):
    """Outputs in the operands' type: half an ulp of the value, as much for each operand rounded on the way (the
    activation, what arrives through the weight), and 2e-5 of the sums' magnitudes in float32."""
    g = torch.Generator(device=DEV).manual_seed(5)
    z = torch.randn(70, 64, generator=g, device=DEV).to(dtype).requires_grad_(True)
    w = (0.2 * torch.randn(64, 24, generator=g, device=DEV)).to(dtype).requires_grad_(True)
    d = torch.randn(70, 24, generator=g, device=DEV).to(dtype)
    y = wl.act_linear8(z, w, act)
    y.backward(d)
    assert y.dtype is dtype and z.grad.dtype is dtype and w.grad.dtype is dtype
    unit = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    z64, w64, d64 = (t.detach().cpu().double() for t in (z, w, d))
    kept = R.keep8(z.detach().cpu())[2].requires_grad_(True)
    a = R.act(kept, act)
    a.backward(d64 @ w64.t())

    def held(got, want, size, what):
        off = (got.detach().cpu().double() - want).abs()
        assert not (off > 3 * unit * size + 2e-5 * size + 1e-6).any(), (what, float((off / size.clamp(min=1e-9)).max()))

    forward = R.act(z64, act)
    held(y, forward @ w64, forward.abs() @ w64.abs(), "y")
    slope = torch.autograd.grad(R.act(kept, act).sum(), kept)[0]
    held(z.grad, kept.grad, (d64.abs() @ w64.abs().t()) * slope.abs().clamp(min=0.1), "z")
    held(w.grad, a.detach().t() @ d64, a.detach().abs().t() @ d64.abs(), "w")
