"""Plain float64 implementations of the layer, update and log-probability operators (include/wc_learn.h), on the CPU."""
import math

import torch

from learn_ref import act

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # a rounding, relative
LEAST = {torch.float32: 0.0, torch.float16: 2.0 ** -24, torch.bfloat16: 0.0}           # and f16's step near 0


def slope(z, name):
    z = z.double().clone().requires_grad_(True)
    act(z, name).backward(torch.ones_like(z))
    return z.grad


def linear(x, weight, bias=None, act_name="none", residual=None):
    """(out, pre)"""
    z = x.double() @ weight.double()
    if bias is not None:
        z = z + bias.double()
    y = act(z, act_name)
    return (y if residual is None else y + residual.double()), z


def linear_backward(d_out, x, weight, pre, act_name):
    """(d_x, d_weight, d_bias, d_pre) at the given pre-activations."""
    d = d_out.double() if act_name == "none" else d_out.double() * slope(pre, act_name)
    return d @ weight.double().t(), x.double().t() @ d, d.sum(0), d


def orthogonalise(u, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, scale=1.0):
    u = u.double()
    if u.dim() == 3:
        return torch.stack([orthogonalise(m, steps, coefficients, eps, scale) for m in u]) if len(u) else u
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # noqa: E731  (what the structure carries)
    a, b, c = (f32(v) for v in coefficients)
    x = u / (u.square().sum().sqrt() + f32(eps))
    for _ in range(steps):
        gram = x @ x.t() if len(x) <= x.shape[1] else x.t() @ x
        p = b * gram + c * gram @ gram
        x = a * x + (p @ x if len(x) <= x.shape[1] else x @ p)
    return f32(scale) * x


def token_logp(logits, tokens=None, legal=None, inv_temperature=1.0, top=0, d_logp=None, d_entropy=None):
    """Row by row: a dict of logp, entropy, rank, top_logp, top_index, grad."""
    inv = float(torch.tensor(inv_temperature, dtype=torch.float32))
    rows, vocab = logits.shape
    out = {"logp": torch.zeros(rows, dtype=torch.float64), "entropy": torch.zeros(rows, dtype=torch.float64),
           "rank": torch.full((rows,), -1, dtype=torch.int32),
           "top_logp": torch.full((rows, top), -math.inf, dtype=torch.float64),
           "top_index": torch.full((rows, top), -1, dtype=torch.int32),
           "grad": torch.zeros(rows, vocab, dtype=torch.float64)}
    for r in range(rows):
        a = None if tokens is None else int(tokens[r])
        if a is not None and not 0 <= a < vocab:
            continue
        x = logits[r].double()
        on = torch.ones(vocab, dtype=torch.bool) if legal is None else legal[r]
        x = torch.where(on, x, torch.tensor(-math.inf, dtype=torch.float64))
        if not (x > -math.inf).any() and not x.isnan().any():
            continue
        z = (x - x.max()) * inv
        logp = z - torch.log(torch.exp(z).sum())
        p = torch.exp(logp)
        safe = torch.where(p > 0, logp, 0.0) if not p.isnan().any() else logp
        h = -(p * safe).sum()
        out["entropy"][r] = h
        if a is not None:
            out["logp"][r] = logp[a]
            out["rank"][r] = int((x > x[a]).sum() + (x[:a] == x[a]).sum())
        order = sorted((j for j in range(vocab) if x[j] > -math.inf), key=lambda j: (-float(x[j]), j)) if top else []
        for t, j in enumerate(order[:top]):
            out["top_index"][r, t] = j
            out["top_logp"][r, t] = logp[j]
        g = torch.zeros(vocab, dtype=torch.float64)
        if d_logp is not None and a is not None:
            g -= float(d_logp[r]) * p
            if on[a]:
                g[a] += float(d_logp[r])
        if d_entropy is not None:
            g -= float(d_entropy[r]) * p * (safe + h)
        out["grad"][r] = torch.where(on, inv * g, 0.0)
    return out
