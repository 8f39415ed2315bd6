"""Plain float64 implementations of the training operators (include/wc_learn.h), on the CPU, row by row.

They follow the definitions in the header and nothing else (coefficients are the float32 values that its structures carry). Gradients of the losses are written out from the formulas;
tests/test_learn_host.py holds them to differences of the losses.
"""
import math

import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half an ulp of 1, bf16 and f16 in full


def row_softmax(x, legal, inv_temp):
    """(logp, logp with 0 where p is 0, p) of one row's legal columns; None where nothing is above -infinity."""
    x = x.double() * inv_temp
    if legal is not None:
        x = torch.where(legal, x, torch.tensor(-math.inf, dtype=torch.float64))
    if not (x > -math.inf).any():
        return None
    z = x - x.max()  # first, so that a row at a type's lowest value keeps its differences
    logp = z - torch.log(torch.exp(z).sum())
    p = torch.exp(logp)
    return logp, torch.where(p > 0, logp, torch.zeros_like(logp)), p


def policy(logits, actions, behaviour_logp, advantages, weights=None, legal=None, ref_logp=None, ref_logits=None,
           inv_temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0):
    inv_temperature, clip_low, clip_high, kl_coef, entropy_coef = (
        float(torch.tensor(v, dtype=torch.float32)) for v in (inv_temperature, clip_low, clip_high, kl_coef, entropy_coef))
    rows, vocab = logits.shape
    w = torch.full((rows,), 1.0 / max(rows, 1), dtype=torch.float64) if weights is None else weights.double()
    out = {n: torch.zeros(rows, dtype=torch.float64) for n in ("logp", "kl", "entropy")}
    grad = torch.zeros(rows, vocab, dtype=torch.float64)
    loss = 0.0
    for r in range(rows):
        a = int(actions[r])
        on = None if legal is None else legal[r]
        if w[r] == 0 or not 0 <= a < vocab or (on is not None and not on[a]):
            continue
        sm = row_softmax(logits[r], on, inv_temperature)
        if sm is None:
            continue
        whole, logp, p = sm
        lp = float(whole[a])
        ratio, adv = math.exp(lp - float(behaviour_logp[r])), float(advantages[r])
        free, held = ratio * adv, min(max(ratio, 1 - clip_low), 1 + clip_high) * adv
        slope, kl = (-free if free <= held else 0.0), 0.0
        h = -float((p * logp).sum())
        g = torch.zeros(vocab, dtype=torch.float64)
        if ref_logp is not None:
            d = float(ref_logp[r]) - lp
            kl = math.expm1(d) - d
            slope -= kl_coef * math.expm1(d)
        if ref_logits is not None:
            _, logq, _ = row_softmax(ref_logits[r], on, inv_temperature)
            d = logp - logq
            kl = float((p * d).sum())
            g += kl_coef * p * (d - kl)
        g += entropy_coef * p * (logp + h) - slope * p
        g[a] += slope
        wr = float(w[r])
        loss += wr * (-min(free, held) + kl_coef * kl - entropy_coef * h)
        out["logp"][r], out["kl"][r], out["entropy"][r] = lp, kl, h
        grad[r] = wr * inv_temperature * g
    return {"loss": torch.tensor(loss, dtype=torch.float64), "grad": grad, **out}


def preference(logits, tokens, offsets, ref_logp, weights=None, beta=0.1, smoothing=0.0, kind="logistic", average=False,
               inv_temperature=1.0):
    beta, smoothing, inv_temperature = (float(torch.tensor(v, dtype=torch.float32))
                                        for v in (beta, smoothing, inv_temperature))
    rows, vocab = logits.shape
    pairs = len(offsets) // 2
    w = torch.ones(rows, dtype=torch.float64) if weights is None else weights.double()
    logp, probs, counted = torch.zeros(rows, dtype=torch.float64), {}, []
    for r in range(rows):
        t = int(tokens[r])
        sm = row_softmax(logits[r], None, inv_temperature) if w[r] != 0 and 0 <= t < vocab else None
        if sm is not None:
            logp[r], probs[r] = float(sm[0][t]), sm[2]
            counted.append(r)
    edge = [min(max(int(o), 0), rows) for o in offsets]
    share, ratio = torch.zeros(rows, dtype=torch.float64), []
    for lo, hi in zip(edge, edge[1:]):
        mine = [r for r in counted if lo <= r < hi]
        total = sum(float(w[r]) for r in mine)
        each = 1.0 if not average else (1.0 / total if total else 0.0)
        for r in mine:
            share[r] = float(w[r]) * each
        ratio.append(sum(float(share[r]) * (float(logp[r]) - float(ref_logp[r])) for r in mine))
    loss, margins = 0.0, []
    grad = torch.zeros(rows, vocab, dtype=torch.float64)
    for i in range(pairs):
        h = ratio[2 * i] - ratio[2 * i + 1]
        z = beta * h
        margins.append(z)
        if kind == "logistic":
            s = 1 / (1 + math.exp(-z)) if z > -700 else 0.0
            loss += (1 - smoothing) * math.log1p(math.exp(-z)) + smoothing * math.log1p(math.exp(z))
            d = beta * (s - (1 - smoothing))
        elif kind == "squared":
            loss += (h - 0.5 / beta) ** 2
            d = 2 * (h - 0.5 / beta)
        else:
            loss += max(0.0, 1 - z)
            d = -beta if z < 1 else 0.0
        for k, sign in ((2 * i, 1.0), (2 * i + 1, -1.0)):
            for r in counted:
                if edge[k] <= r < edge[k + 1]:
                    c = sign * d / pairs * float(share[r])
                    grad[r] = -c * probs[r] * inv_temperature
                    grad[r, int(tokens[r])] += c * inv_temperature
    return {"loss": torch.tensor(loss / max(pairs, 1), dtype=torch.float64),
            "margins": torch.tensor(margins, dtype=torch.float64), "ratios": torch.tensor(ratio, dtype=torch.float64),
            "logp": logp, "grad": grad}


def _norm(x, gain, bias, kind, eps):
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(1, keepdim=True) + eps)
    if gain is not None:
        x = x * gain
    return x if bias is None else x + bias


def residual_norm(block, stream, post_gain=None, post_bias=None, gate=None, pre_gain=None, pre_bias=None, scale=1.0,
                  eps=1e-5, norm="layer", gate_act="none"):
    """Float64 inputs; differentiable."""
    n = _norm(block, post_gain, post_bias, norm, eps)
    if gate is not None:
        n = n * {"none": lambda g: g, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[gate_act](gate)
    new = stream + scale * n
    return new, _norm(new, pre_gain, pre_bias, norm, eps)


def keep8(x):
    """(q, e, value) of the 8-bit checkpoint, one group at a time."""
    rows, width = x.shape
    groups = -(-width // 32)
    q = torch.zeros(rows, width, dtype=torch.int8)
    e = torch.zeros(rows, groups, dtype=torch.uint8)
    value = torch.zeros(rows, width, dtype=torch.float64)
    for r in range(rows):
        for g in range(groups):
            part = slice(32 * g, min(32 * g + 32, width))
            v = [float(t) for t in x[r, part]]
            if not all(math.isfinite(t) for t in v):
                q[r, part], e[r, g], value[r, part] = 1, 255, math.nan
                continue
            top, k = max(abs(t) for t in v), -126
            if top > 0:
                k = max(k, math.frexp(top)[1] - 9)
                while top > 127 * math.ldexp(1.0, k):
                    k += 1
            n = [round(math.ldexp(t, -k)) for t in v]  # Python rounds ties to even
            q[r, part], e[r, g] = torch.tensor(n, dtype=torch.int8), k + 127
            value[r, part] = torch.tensor([math.ldexp(float(t), k) for t in n], dtype=torch.float64)
    return q, e, value


def act(x, name):
    """Float64; differentiable."""
    if name == "none":
        return x * 1.0
    if name == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x))
    if name == "silu":
        return x * torch.sigmoid(x)
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
