"""The layer, update and log-probability operators together: a network's gradients, the optimiser, the training example."""
import pytest
import torch

import layer_ref as R
import learn_ref
import train_policy
import warchest_learn as wl

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def float32_by_default():
    """Other test modules set torch's default type to float64 for the whole process."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)


DEV = "cuda:0"


def test_the_fused_network_and_its_gradients_against_float64():
    """Log-probabilities and entropies of a two-block network, and the gradients of every parameter, against the same
    network in float64 on the weights as bf16 has them. Each of a dozen results on the way forward and as many back is
    rounded to bf16, 2^-8 at most: as independent errors sqrt(24) 2^-8 / sqrt(3) = 1.1e-2 of a gradient's norm; four times
    that is taken."""
    torch.manual_seed(1)
    net = train_policy.PolicyNet(24, 64, 2, 19, DEV, fused=True)
    with torch.no_grad():
        for p in net.parameters():
            p.copy_((p + 0.05 * torch.randn_like(p)).bfloat16())
    x = torch.randn(130, 24, device=DEV).bfloat16()
    tokens = torch.randint(0, 19, (130,), device=DEV)
    d1, d2 = torch.randn(130, device=DEV), 0.3 * torch.randn(130, device=DEV)
    logp, entropy, *_ = wl.token_logp_objective(net(x), tokens)
    ((logp * d1).sum() + (entropy * d2).sum()).backward()

    v = {n: p.detach().cpu().double().requires_grad_(True) for n, p in net.named_parameters()}
    out = stream = x.cpu().double() @ v["inp"]
    for i in range(2):
        hidden = learn_ref.act(out @ v[f"up.{i}"] + v[f"up_bias.{i}"], "gelu")
        block = hidden @ v[f"down.{i}"] + v[f"down_bias.{i}"]
        names = ("post_gain", "post_bias", "gate", "pre_gain", "pre_bias")
        stream, out = learn_ref.residual_norm(block, stream, *(v[f"norms.{i}.{n}"] for n in names), **net.norms[i].kw)[:2]
    z = torch.log_softmax(out @ v["head"], 1)
    h = -(z.exp() * z).sum(1)
    lp = z.gather(1, tokens.cpu()[:, None])[:, 0]
    ((lp * d1.cpu().double()).sum() + (h * d2.cpu().double()).sum()).backward()
    lp, h = lp.detach(), h.detach()
    assert float((logp.detach().cpu() - lp).norm()) < 4.4e-2 * float(lp.norm())
    assert float((entropy.detach().cpu() - h).norm()) < 4.4e-2 * float(h.norm())
    for n, p in net.named_parameters():
        off = float((p.grad.cpu().double() - v[n].grad).norm())
        assert off < 4.4e-2 * float(v[n].grad.norm()), (n, off, float(v[n].grad.norm()))


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_against_float64(nesterov):
    """Three steps of stacked, tall, wide and alike weights. A step's update is off by what orthogonalise is (15 float32
    sums, 15 2^-23 (K / 16 + 80) of the root mean square: 2e-4), the weights' own roundings by less."""
    torch.manual_seed(2)
    ws = [torch.randn(*s, device=DEV, requires_grad=True) for s in ((40, 24), (24, 70), (24, 70), (3, 20, 33))]
    opt = wl.Muon(ws, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.01, dtype=torch.float32)
    ref = [w.detach().cpu().double() for w in ws]
    held = [torch.zeros_like(w) for w in ref]
    for step in range(3):
        for i, w in enumerate(ws):
            w.grad = torch.randn_like(w)
            g = w.grad.cpu().double()
            held[i] = 0.9 * held[i] + g
            u = g + 0.9 * held[i] if nesterov else held[i]
            o = R.orthogonalise(u, scale=max(1.0, w.shape[-1] / w.shape[-2]) ** 0.5)
            ref[i] = ref[i] * (1 - 0.1 * 0.01) - 0.1 * o
        opt.step()
        for w, r in zip(ws, ref):
            assert float((w.detach().cpu().double() - r).norm()) < (step + 1) * 2e-4 * float(r.norm())
    state = opt.state_dict()
    assert len(state["state"]) == 4


def test_muon_leaves_weights_without_a_gradient_alone():
    a, b = (torch.randn(8, 8, device=DEV, requires_grad=True) for _ in range(2))
    opt = wl.Muon([a, b])
    before = b.detach().clone()
    a.grad = torch.ones_like(a)
    opt.step()
    assert torch.equal(b, before) and a.isfinite().all()


@pytest.mark.parametrize("fused,muon", [(True, False), (False, True), (True, True)])
def test_the_training_example_with_fused_layers_and_muon(fused, muon):
    """That it runs, and that what it reports is finite."""
    lines = []
    got = train_policy.train(trees=2, steps=6, width=64, blocks=2, batch=512, say=lines.append, fused=fused, muon=muon)
    assert all(v == v and abs(v) < 1e6 for v in got)
    assert any("first choice" in line for line in lines)


def test_two_calls_on_two_streams_do_not_meet():
    """Scratch is each call's own: the same layer, update and log-probabilities on two streams at once, as alone."""
    torch.manual_seed(3)
    x, w = torch.randn(700, 1153, device=DEV), torch.randn(1153, 90, device=DEV)
    u, logits = torch.randn(300, 520, device=DEV), torch.randn(3, 70000, device=DEV)

    def work(scale):
        return (wl.linear(scale * x, w, act="gelu").out, wl.orthogonalise(u, scale=scale),
                wl.token_logp(scale * logits, top=9).top_logp)
    want = [[t.clone() for t in work(s)] for s in (1.0, 2.0)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(1.0 + i))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            for a, b in zip(one, want[i]):
                assert torch.equal(a, b)
