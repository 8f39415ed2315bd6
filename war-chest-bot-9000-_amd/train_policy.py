"""Trains a small residual policy network on what the solver finds: the training operators as they are used together.

The wave executor solves synthetic subgames; every infostate's legal actions and average strategy become one row. The
network (an input projection, residual blocks between two norms whose activations are kept in 8 bits, a head of one
logit an action) is trained in two phases:

- policy: actions drawn from the search's strategy, the clipped loss with the full KL to that strategy;
- preference: pairs of lines of decisions, the search's favourite actions against its least likely ones.

    python train_policy.py [--trees 8] [--steps 60] [--width 256] [--blocks 2]

prints the losses and the mean KL to the search's policy as they fall. Features are synthetic (one seeded vector a row),
so this is a demonstration of the calls, not a player.
"""
from __future__ import annotations

import argparse

import numpy as np
import torch

import warchest_learn as wl
import warchest_wave as ww
import workloads as W


def solved_rows(trees, device=0):
    """(strategy, legal), rows x most actions, of every infostate of `trees` solved subgames."""
    jobs = W.jobs("wave64", trees=trees, iters=32)
    ex = ww.Executor(device, ww.WC_F16)
    wave = ww.Wave(jobs)
    out = ex.solve(wave, ex.publish(W.net_for("wave64")))
    off = wave.array("legal_off").astype(np.int64)
    cells = np.concatenate([r.strategy for r in out])
    wave.close()
    ex.close()
    n = np.diff(off)
    strategy = np.zeros((len(n), int(n.max())), np.float32)
    legal = np.arange(strategy.shape[1])[None, :] < n[:, None]
    strategy[legal] = cells
    return strategy[n > 1], legal[n > 1]


class PolicyNet(torch.nn.Module):
    """float32 parameters, bf16 activations."""

    def __init__(self, inputs, width, blocks, actions, device):
        super().__init__()
        def weight(i, o, gain=1.0):
            return torch.nn.Parameter(torch.randn(i, o, device=device, dtype=torch.float32) * gain * i ** -0.5)

        self.inp = weight(inputs, width)
        self.up = torch.nn.ParameterList(weight(width, 4 * width) for _ in range(blocks))
        self.down = torch.nn.ParameterList(weight(4 * width, width) for _ in range(blocks))
        self.norms = torch.nn.ModuleList(wl.ResidualNorm(width, scale=0.5, device=device) for _ in range(blocks))
        self.head = weight(width, actions, 0.1)

    def forward(self, x):
        stream = x @ self.inp.bfloat16()
        out = stream
        for up, down, norm in zip(self.up, self.down, self.norms):
            block = wl.act_linear8(out @ up.bfloat16(), down.bfloat16())
            stream, out = norm(block, stream)
        return (out @ self.head.bfloat16()).float()


def train(trees=8, steps=60, width=256, blocks=2, batch=4096, seed=0, say=print):
    """Returns (mean KL before, mean KL after the policy phase, preference loss before, after)."""
    torch.manual_seed(seed)
    dev = torch.device("cuda", 0)
    s, l = solved_rows(trees)
    strategy, legal = torch.from_numpy(s).to(dev), torch.from_numpy(l).to(dev)
    rows, actions = strategy.shape
    search = strategy.clamp(min=1e-3).log().masked_fill(~legal, 0.0)
    x = torch.from_numpy(ww.synth_features(rows, 512, seed + 1)).to(dev).bfloat16() - 0.5
    net = PolicyNet(512, width, blocks, actions, dev)
    opt = torch.optim.AdamW(net.parameters(), lr=2e-3)
    say(f"{rows} infostates of {trees} solved subgames, up to {actions} actions")

    kls = []
    for step in range(steps):
        pick = torch.randint(0, rows, (min(batch, rows),), device=dev)
        p, on = strategy[pick], legal[pick]
        chosen = torch.multinomial(p, 1)[:, 0]
        behaviour = search[pick].gather(1, chosen[:, None])[:, 0]
        gain = p.gather(1, chosen[:, None])[:, 0] * on.sum(1) - 1.0  # how much likelier than at random
        loss, _, kl, _ = wl.policy_objective(net(x[pick]), chosen, behaviour, gain, legal=on, ref_logits=search[pick],
                                             kl_coef=1.0, entropy_coef=0.01)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        kls.append(float(kl.mean()))
        if step % 20 == 0 or step == steps - 1:
            say(f"policy step {step:4d}: loss {float(loss.detach()):8.4f}, KL to the search {kls[-1]:.4f}")

    # lines of four decisions: the search's favourites against its least likely actions
    lines, length = 256, 4
    pick = torch.randint(0, rows, (lines, length), device=dev)
    best = strategy[pick].argmax(2)
    worst = strategy[pick].masked_fill(~legal[pick], 2.0).argmin(2)
    where = torch.stack([pick, pick], 1).reshape(-1)
    tokens = torch.stack([best, worst], 1).reshape(-1)
    offsets = torch.arange(0, 2 * lines * length + 1, length, device=dev)
    barred = (~legal[where]).float() * -1e4

    def pair_logits():
        return net(x[where]) + barred

    with torch.no_grad():
        before = torch.log_softmax(pair_logits(), 1).gather(1, tokens[:, None])[:, 0].contiguous()
    prefs = []
    for step in range(steps // 2):
        loss, _, _ = wl.preference_objective(pair_logits(), tokens, offsets, before, beta=0.5)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        prefs.append(float(loss.detach()))
        if step % 10 == 0 or step == steps // 2 - 1:
            say(f"preference step {step:4d}: loss {prefs[-1]:.4f}")
    return kls[0], kls[-1], prefs[0], prefs[-1]


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("trees", 8), ("steps", 60), ("width", 256), ("blocks", 2)):
        ap.add_argument("--" + name, type=int, default=value)
    train(**vars(ap.parse_args()))
