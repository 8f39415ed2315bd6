"""The operators that train a policy or value network on what the solver finds.

Four operators, all through the public binding (warchest_learn.py):

- "policy": policy_loss, the clipped policy loss with a KL term and an entropy bonus over rows of action or token
  logits, forward and gradient in one call.
- "preference": preference_loss, the paired log-ratio loss over ragged sequences, forward and gradient.
- "norm": residual_norm (and residual_norm_backward), a block's output normed, gated, scaled and added to the residual
  stream, and the norm before the next block, in one pass.
- "recall", "layer", "weight": checkpoint8 and its readers, activations kept in 8 bits for the backward pass: written and
  read back; an activation function's forward and backward; a weight gradient from the 8-bit operand.

The plain form of each is torch's elementary operations in 32 bits, and exact() its definition in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
GROUP = 32  # channels of one row that share a power of two in an 8-bit checkpoint


def listed():
    return [
        # the actions of one small subgame's infostates: 22 heads, few rows, latency
        {"name": "policy_heads_f32", "op": "policy", "rows": 64, "vocab": 22, "dtype": "f32", "legal": True,
         "ref": "token", "masked": 0.0, "entropy": 0.01},
        # every network row of a 256-subgame wave, 567 heads, the search's own policy as the reference distribution
        {"name": "policy_wave_f32", "op": "policy", "rows": 49371, "vocab": 567, "dtype": "f32", "legal": True,
         "ref": "full", "masked": 0.1, "entropy": 0.01},
        # a batch of long token sequences with a large vocabulary, part of the rows prompts and padding
        {"name": "policy_vocab_bf16", "op": "policy", "rows": 4096, "vocab": 65536, "dtype": "bf16", "legal": False,
         "ref": "token", "masked": 0.25, "entropy": 0.0},
        # paired lines of play over 64 heads: a short update between games
        {"name": "pref_lines_f32", "op": "preference", "pairs": 16, "shortest": 1, "longest": 24, "vocab": 64,
         "dtype": "f32", "kind": "logistic", "average": False, "masked": 0.0},
        # ragged pairs, some of them empty, an odd vocabulary: rows at every alignment
        {"name": "pref_odd_f16", "op": "preference", "pairs": 33, "shortest": 0, "longest": 200, "vocab": 4099,
         "dtype": "f16", "kind": "squared", "average": True, "masked": 0.1},
        # long pairs with prompts over a large vocabulary
        {"name": "pref_vocab_bf16", "op": "preference", "pairs": 8, "shortest": 64, "longest": 512, "vocab": 65536,
         "dtype": "bf16", "kind": "logistic", "average": False, "masked": 0.3},
        # one board of the v5 network: 37 cells of 96 channels, inference
        {"name": "norm_board_f32", "op": "norm", "rows": 37, "width": 96, "dtype": "f32", "norm": "layer",
         "gate": "vector", "gate_act": "none", "backward": False},
        # odd rows and width, a gate per token through a sigmoid, a training step
        {"name": "norm_odd_f16", "op": "norm", "rows": 4099, "width": 1153, "dtype": "f16", "norm": "layer",
         "gate": "token", "gate_act": "sigmoid", "backward": True},
        # a training step of a wide residual stream with a learned gate vector
        {"name": "norm_stream_bf16", "op": "norm", "rows": 16384, "width": 4096, "dtype": "bf16", "norm": "rms",
         "gate": "vector", "gate_act": "none", "backward": True},
        # a wide layer's activation function, forward and backward, its input kept in 8 bits between the two
        {"name": "ckpt_layer_bf16", "op": "layer", "rows": 16384, "width": 8192, "dtype": "bf16", "act": "gelu"},
        # the weight gradient of the value network's first layer over a wave's rows: a small product over a long sum
        {"name": "ckpt_weight_mlp_bf16", "op": "weight", "rows": 49371, "width": 512, "out": 384, "dtype": "bf16",
         "act": "none", "result": "f32"},
        # the weight gradient of a wide layer, its operand's activation recomputed from the 8 bits
        {"name": "ckpt_weight_wide_bf16", "op": "weight", "rows": 16384, "width": 4096, "out": 4096, "dtype": "bf16",
         "act": "gelu", "result": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["policy", "preference", "norm", "recall", "layer", "weight"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "policy":
        vocab = _log_int(rng, 8, 131072)
        return {"op": op, "rows": _log_int(rng, 1, min(65536, (1 << 26) // vocab)), "vocab": vocab, "dtype": dtype,
                "legal": vocab <= 4096 and rng.random() < 0.7, "ref": rng.choice(["none", "token", "full"]),
                "masked": rng.choice([0.0, 0.1, 0.5]), "entropy": rng.choice([0.0, 0.01])}
    if op == "preference":
        vocab = _log_int(rng, 8, 131072)
        longest = _log_int(rng, 2, max(3, min(1024, (1 << 25) // vocab)))
        pairs = _log_int(rng, 1, max(2, min(256, (1 << 26) // (vocab * longest))))
        return {"op": op, "pairs": pairs, "shortest": rng.choice([0, 1, longest // 2]), "longest": longest,
                "vocab": vocab, "dtype": dtype, "kind": rng.choice(["logistic", "squared", "hinge"]),
                "average": rng.random() < 0.5, "masked": rng.choice([0.0, 0.3])}
    if op == "norm":
        width = _log_int(rng, 16, 8192)
        gate = rng.choice(["none", "vector", "token"])
        return {"op": op, "rows": _log_int(rng, 1, min(65536, (1 << 24) // width)), "width": width, "dtype": dtype,
                "norm": rng.choice(["rms", "layer"]), "gate": gate,
                "gate_act": rng.choice(["none", "sigmoid", "tanh"]) if gate != "none" else "none",
                "backward": rng.random() < 0.7}
    if op == "weight":
        width, out = _log_int(rng, 64, 4096), _log_int(rng, 32, 4096)
        dtype = rng.choice(["f16", "bf16"])
        act = rng.choice(["none", "none", "relu", "gelu", "silu"])
        return {"op": op, "rows": _log_int(rng, 1, min(65536, (1 << 38) // (width * out))), "width": width, "out": out,
                "dtype": dtype, "act": act, "result": "f32" if act in ("none", "relu") else dtype}
    width = _log_int(rng, 16, 8192)
    return {"op": op, "rows": _log_int(rng, 1, min(65536, (1 << 26) // width)), "width": width, "dtype": dtype,
            "act": "none" if op == "recall" else rng.choice(["relu", "gelu", "silu"])}


# ------------------------------------------------------------------ inputs

class _Random:
    """Seeded values on the GPU (on the CPU where there is none)."""

    def __init__(self, seed):
        self.device = torch.device("cuda" if torch.cuda.is_available() else "cpu")
        self.g = torch.Generator(device=self.device)
        self.g.manual_seed(int(seed) * 2654435761 % (1 << 62))

    def normal(self, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
        x = torch.randn(shape, generator=self.g, device=self.device, dtype=torch.float32)
        return x.mul_(scale).add_(shift).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.g, device=self.device, dtype=torch.float32)

    def some(self, n, share):
        """Truth values, round(share * n) of them true, at places of their own."""
        out = torch.zeros(n, dtype=torch.bool, device=self.device)
        out[torch.randperm(n, generator=self.g, device=self.device)[: round(share * n)]] = True
        return out


def _lengths(c):
    """The preference case's sequence lengths: the case's own, the same for every seed."""
    n, lo, hi = 2 * c["pairs"], c["shortest"], c["longest"]
    return [lo + (hi - lo) * ((7 * i + 3) % 16) // 15 for i in range(n)] if n > 2 else [lo, hi]


def prepare(case, seed):
    r, op = _Random(seed), case["op"]
    s = {"case": case}
    if op != "norm" and op not in ("recall", "layer", "weight"):
        dt = _DTYPES[case["dtype"]]
        rows = case["rows"] if op == "policy" else max(1, sum(_lengths(case)))
        vocab = case["vocab"]
        s["logits"] = r.normal(rows, vocab, scale=2.0, dtype=dt)
        left_out = r.some(rows, case["masked"])
        s["legal"] = None
        f = s["logits"].float()
        if case.get("legal"):
            legal = r.uniform(rows, vocab) < 0.5
            legal[torch.arange(rows, device=r.device), (r.uniform(rows) * vocab).long().clamp_(max=vocab - 1)] = True
            s["legal"] = legal
            f.masked_fill_(~legal, -math.inf)
        # the chosen action: a sample of the policy itself
        chosen = (f - torch.log(-torch.log(r.uniform(rows, vocab).clamp_(1e-9, 1 - 1e-7)))).argmax(1)
        logp = torch.log_softmax(f, 1).gather(1, chosen[:, None])[:, 0]
        del f
        s["chosen"] = torch.where(left_out, -1, chosen)
        counted = (~left_out).float()
    if op == "policy":
        s["behaviour_logp"] = logp + r.normal(rows, scale=0.2)
        s["advantages"] = r.normal(rows)
        s["weights"] = counted / max(1, rows - round(case["masked"] * rows))
        s["ref_logp"] = logp + r.normal(rows, scale=0.4) if case["ref"] == "token" else None
        s["ref_logits"] = (s["logits"] + r.normal(rows, vocab, scale=0.7)).to(dt) if case["ref"] == "full" else None
    elif op == "preference":
        ends = [0]
        for n in _lengths(case):
            ends.append(ends[-1] + n)
        s["offsets"] = torch.tensor(ends, dtype=torch.int64, device=r.device)
        s["weights"] = counted
        s["ref_logp"] = logp + r.normal(rows, scale=0.4)
    elif op == "norm":
        dt, rows, width = _DTYPES[case["dtype"]], case["rows"], case["width"]
        s["block"] = r.normal(rows, width, scale=1.7, shift=0.1, dtype=dt)
        s["stream"] = r.normal(rows, width, scale=3.0, dtype=dt)
        for side in ("post", "pre"):
            s[side + "_gain"] = r.normal(width, scale=0.1, shift=1.0, dtype=dt)
            s[side + "_bias"] = r.normal(width, scale=0.1, dtype=dt) if case["norm"] == "layer" else None
        s["gate"] = {"none": None, "vector": (width,), "token": (rows, width)}[case["gate"]]
        if s["gate"] is not None:
            s["gate"] = r.normal(*s["gate"], scale=0.3, shift=0.5, dtype=dt)
        s["args"] = {"norm": case["norm"], "gate_act": case["gate_act"], "scale": 0.5,
                     "eps": 1e-5 if case["norm"] == "layer" else 1e-6}
        if case["backward"]:
            s["d_out"] = r.normal(rows, width, dtype=dt)
            s["d_stream"] = r.normal(rows, width, dtype=dt)
    else:
        dt, rows, width = _DTYPES[case["dtype"]], case["rows"], case["width"]
        x = r.normal(rows, width, scale=1.5, dtype=dt)
        if op == "weight":
            # the checkpoint that the forward pass left, and the gradient that arrives
            q, k = _quantise(x)
            s["q"], s["exps"] = q, (k + 127).to(torch.uint8)
            s["grad"] = r.normal(rows, case["out"], dtype=dt)
        else:
            s["x"] = x
            if op == "layer":
                s["grad"] = r.normal(rows, width, dtype=dt)
    if own:
        _binding()
    return s


def _binding():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "war-chest-bot-9000-_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import warchest_learn

    return warchest_learn


_POLICY = {"inv_temperature": 0.8, "clip_low": 0.2, "clip_high": 0.28, "kl_coef": 0.05}
_PREFERENCE = {"beta": 0.1, "smoothing": 0.1, "hinge": 1.0}


# ------------------------------------------------------------------ plain forms

def _plain_policy(s):
    c, w, a = s["case"], s["weights"], _POLICY
    x = s["logits"].float() * a["inv_temperature"]
    if s["legal"] is not None:
        x = torch.where(s["legal"], x, -math.inf)
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    logp, p = x - top - torch.log(total), e / total
    here = s["chosen"].clamp(min=0)[:, None]
    lp = logp.gather(1, here)[:, 0]
    logp = torch.where(p > 0, logp, 0.0)
    entropy = -(p * logp).sum(1)
    ratio = torch.exp(lp - s["behaviour_logp"])
    free = ratio * s["advantages"]
    held = ratio.clamp(1 - a["clip_low"], 1 + a["clip_high"]) * s["advantages"]
    d_lp = -torch.where(free <= held, free, 0.0)
    kl, toward = torch.zeros_like(lp), None
    if s["ref_logp"] is not None:
        off = s["ref_logp"] - lp
        kl = torch.expm1(off) - off
        d_lp = d_lp - a["kl_coef"] * torch.expm1(off)
    if s["ref_logits"] is not None:
        y = s["ref_logits"].float() * a["inv_temperature"]
        if s["legal"] is not None:
            y = torch.where(s["legal"], y, -math.inf)
        y = y - y.amax(1, keepdim=True)
        toward = logp - torch.where(p > 0, y - torch.log(torch.exp(y).sum(1, keepdim=True)), 0.0)
        kl = (p * toward).sum(1)
    loss = (w * (-torch.minimum(free, held) + a["kl_coef"] * kl - c["entropy"] * entropy)).sum()
    g = -(w * d_lp)[:, None] * p
    g.scatter_add_(1, here, (w * d_lp)[:, None])
    if c["entropy"]:
        g += (w * c["entropy"])[:, None] * p * (logp + entropy[:, None])
    if toward is not None:
        g += (w * a["kl_coef"])[:, None] * p * (toward - kl[:, None])
    counted = w != 0
    return {"loss": loss, "logp": torch.where(counted, lp, 0.0), "kl": torch.where(counted, kl, 0.0),
            "entropy": torch.where(counted, entropy, 0.0), "grad": (g * a["inv_temperature"]).to(s["logits"].dtype)}


def _plain_preference(s):
    c, w, a = s["case"], s["weights"], _PREFERENCE
    x = s["logits"].float()
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    here = s["chosen"].clamp(min=0)[:, None]
    lp = (x.gather(1, here) - top - torch.log(total))[:, 0]
    at = torch.arange(len(w), device=w.device)
    inside = ((at >= s["offsets"][:-1, None]) & (at < s["offsets"][1:, None])).float() * w  # [sequences, rows]
    each = inside.sum(1)
    share = torch.where(each > 0, 1 / each.clamp(min=1e-30), 0.0) if c["average"] else torch.ones_like(each)
    ratio = (inside @ torch.where(w != 0, lp - s["ref_logp"], 0.0)) * share
    margin = ratio[0::2] - ratio[1::2]
    z = a["beta"] * margin
    if c["kind"] == "logistic":
        loss = (1 - a["smoothing"]) * torch.log1p(torch.exp(-z.abs())) + (1 - a["smoothing"]) * (-z).clamp(min=0)
        loss = loss + a["smoothing"] * (torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0))
        d = a["beta"] * (torch.sigmoid(z) - (1 - a["smoothing"]))
    elif c["kind"] == "squared":
        loss = (margin - 0.5 / a["beta"]) ** 2
        d = 2 * (margin - 0.5 / a["beta"])
    else:
        loss = (1 - z).clamp(min=0)
        d = torch.where(z < 1, -a["beta"], 0.0)
    d = d / c["pairs"]
    row = (torch.stack([d, -d], 1).reshape(-1) * share) @ inside
    g = -row[:, None] * (e / total)
    g.scatter_add_(1, here, row[:, None])
    return {"loss": loss.mean(), "margins": z, "ratios": ratio, "grad": g.to(s["logits"].dtype)}


def _plain_normed(x, kind, eps):
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    r = torch.rsqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    return (x - mean) * r, r


def _plain_norm_back(d, xhat, r, kind):
    d = d - xhat * (d * xhat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if kind == "layer" else 0)
    return d * r


def _plain_norm(s):
    c, a = s["case"], s["args"]
    dt, kind = s["block"].dtype, a["norm"]
    g1, b1, g2, b2 = (None if s[n] is None else s[n].float() for n in ("post_gain", "post_bias", "pre_gain", "pre_bias"))
    uhat, r1 = _plain_normed(s["block"].float(), kind, a["eps"])
    n = uhat * g1 + (0 if b1 is None else b1)
    raw = None if s["gate"] is None else s["gate"].float()
    gate = 1.0 if raw is None else {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[a["gate_act"]](raw)
    stream = s["stream"].float() + a["scale"] * gate * n
    xhat, r2 = _plain_normed(stream, kind, a["eps"])
    out = {"stream": stream.to(dt), "out": (xhat * g2 + (0 if b2 is None else b2)).to(dt)}
    if not c["backward"]:
        return out
    dh = s["d_out"].float()
    dx = s["d_stream"].float() + _plain_norm_back(dh * g2, xhat, r2, kind)
    out |= {"d_stream": dx.to(dt), "d_pre_gain": (dh * xhat).sum(0)}
    dn = a["scale"] * gate * dx
    out |= {"d_block": _plain_norm_back(dn * g1, uhat, r1, kind).to(dt), "d_post_gain": (dn * uhat).sum(0)}
    if b1 is not None:
        out |= {"d_pre_bias": dh.sum(0), "d_post_bias": dn.sum(0)}
    if raw is not None:
        slope = {"none": 1.0, "sigmoid": gate * (1 - gate), "tanh": 1 - gate * gate}[a["gate_act"]]
        dg = a["scale"] * n * dx * slope
        out["d_gate"] = dg.to(dt) if c["gate"] == "token" else dg.sum(0)
    return out


def _quantise(x):
    """(q, k): x's groups of 32 channels as integers of up to 127 times 2^k, k the least that fits."""
    rows, width = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -width % GROUP)).reshape(rows, -1, GROUP)
    m, e = torch.frexp(v.abs().amax(2))
    k = (e - 7 + (m > 127 / 128)).clamp(min=-126)
    k = torch.where(m == 0, -126, k)
    q = torch.round(torch.ldexp(v, -k[:, :, None])).to(torch.int8)
    return q.reshape(rows, -1)[:, :width].contiguous(), k


def _stands_for(q, k):
    rows, width = q.shape
    v = torch.nn.functional.pad(q.float(), (0, -width % GROUP)).reshape(rows, -1, GROUP)
    return torch.ldexp(v, k[:, :, None]).reshape(rows, -1)[:, :width]


def _plain_act(z, act):
    """(value, slope) of the activation function."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).float()
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g * (1 + z * (1 - g))
    u = 0.7978845608028654 * (z + 0.044715 * z * z * z)
    t = torch.tanh(u)
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * 0.7978845608028654 * (1 + 3 * 0.044715 * z * z)


def _plain_checkpoint(s):
    c = s["case"]
    if c["op"] == "weight":
        v = _stands_for(s["q"], s["exps"].int() - 127)
        if c["act"] != "none":
            v = _plain_act(v, c["act"])[0]
        g = s["grad"].float()
        return {"weight": (v.t() @ g).to(_DTYPES[c["result"]]), "bias": g.sum(0)}
    v = _stands_for(*_quantise(s["x"]))
    if c["op"] == "recall":
        return v.to(s["x"].dtype)
    return {"out": _plain_act(s["x"].float(), c["act"])[0].to(s["x"].dtype),
            "grad": (s["grad"].float() * _plain_act(v, c["act"])[1]).to(s["x"].dtype)}


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"policy": _plain_policy, "preference": _plain_preference, "norm": _plain_norm}.get(
            op, _plain_checkpoint)(s)
    wl = _binding()
    if op == "policy":
        r = wl.policy_loss(s["logits"], s["chosen"], s["behaviour_logp"], s["advantages"], s["weights"],
                           legal=s["legal"], ref_logp=s["ref_logp"], ref_logits=s["ref_logits"],
                           entropy_coef=c["entropy"], **_POLICY)
        return {"loss": r.loss, "logp": r.logp, "kl": r.kl, "entropy": r.entropy, "grad": r.grad}
    if op == "preference":
        r = wl.preference_loss(s["logits"], s["chosen"], s["offsets"], s["ref_logp"], s["weights"],
                               beta=_PREFERENCE["beta"], smoothing=_PREFERENCE["smoothing"], kind=c["kind"],
                               average=c["average"])
        return {"loss": r.loss, "margins": r.margins, "ratios": r.ratios, "grad": r.grad}
    if op == "norm":
        params = [s[n] for n in ("post_gain", "post_bias", "gate", "pre_gain", "pre_bias")]
        f = wl.residual_norm(s["block"], s["stream"], *params, **s["args"])
        out = {"stream": f.stream, "out": f.out}
        if c["backward"]:
            b = wl.residual_norm_backward(s["d_out"], s["d_stream"], s["block"], s["stream"], f.stats, *params,
                                          **s["args"])
            out |= {"d_stream": b.stream, "d_block": b.block, "d_post_gain": b.post_gain, "d_pre_gain": b.pre_gain}
            if s["pre_bias"] is not None:
                out |= {"d_post_bias": b.post_bias, "d_pre_bias": b.pre_bias}
            if s["gate"] is not None:
                out["d_gate"] = b.gate
        return out
    if op == "weight":
        weight, bias = wl.checkpoint8_weight_grad(wl.Checkpoint8(s["q"], s["exps"]), s["grad"], act=c["act"],
                                                  bias=True, dtype=_DTYPES[c["result"]])
        return {"weight": weight, "bias": bias}
    if op == "recall":
        return wl.checkpoint8_read(wl.checkpoint8(s["x"]), s["x"].dtype)
    kept, out = wl.checkpoint8_act(s["x"], c["act"])
    return {"out": out, "grad": wl.checkpoint8_act_backward(kept, s["grad"], c["act"])}


# ------------------------------------------------------------------ work

def work(c):
    op = c["op"]
    if op in ("policy", "preference"):
        rows = c["rows"] if op == "policy" else max(1, sum(_lengths(c)))
        n = (rows - round(c["masked"] * rows)) * c["vocab"]  # logits that count
        size = _BYTES[c["dtype"]]
        read = n * (size * (2 if c.get("ref") == "full" else 1) + (1 if c.get("legal") else 0))
        return {"bytes": read + rows * c["vocab"] * size + rows * 36, "flops": 10 * n}
    n, size = c["rows"] * c["width"], _BYTES[c["dtype"]]
    if op == "norm":
        # forward: two arrays in, two out; backward: four in, two out; a gate per token is read by both, and its gradient
        # written
        token = c["gate"] == "token"
        arrays = 4 + token + ((6 + 2 * token) if c["backward"] else 0)
        return {"bytes": arrays * n * size + c["rows"] * 16, "flops": n * (60 if c["backward"] else 16)}
    held = n + c["rows"] * -(-c["width"] // GROUP)
    if op == "weight":
        m = c["rows"] * c["out"]
        return {"bytes": held + m * size + c["width"] * c["out"] * _BYTES[c["result"]], "flops": 2 * n * c["out"]}
    # written and read: the 8-bit form; recall: one array in, one out; layer: input, output, gradient in, gradient out
    return {"bytes": 2 * held + (2 if op == "recall" else 4) * n * size, "flops": n * (6 if op == "recall" else 40)}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_policy(s):
    c, a = s["case"], _POLICY
    out = {"loss": None, "logp": [], "kl": [], "entropy": [], "grad": []}
    loss = 0.0
    legal = s["legal"]
    for lo in range(0, len(s["weights"]), 1024):
        part = slice(lo, lo + 1024)
        x = s["logits"][part].double() * a["inv_temperature"]
        open_ = torch.ones_like(x, dtype=torch.bool) if legal is None else legal[part]
        x = x.masked_fill(~open_, -math.inf)
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        p = torch.exp(logp)
        logp = logp.masked_fill(~open_, 0.0)
        w, adv = s["weights"][part].double(), s["advantages"][part].double()
        counted = w != 0
        pick = torch.zeros_like(p)
        pick[torch.arange(len(w)), s["chosen"][part].clamp(min=0)] = 1.0
        lp = (pick * logp).sum(1)
        h = -(p * logp).sum(1)
        ratio = torch.exp(lp - s["behaviour_logp"][part].double())
        bounded = torch.minimum(torch.maximum(ratio, torch.tensor(1 - a["clip_low"]).to(ratio)),
                                torch.tensor(1 + a["clip_high"]).to(ratio))
        first = (ratio * adv) <= (bounded * adv)
        gain = torch.where(first, ratio * adv, bounded * adv)
        slope = torch.where(first, -ratio * adv, torch.zeros_like(adv))
        kl = torch.zeros_like(lp)
        extra = torch.zeros_like(p)
        if s["ref_logp"] is not None:
            t = s["ref_logp"][part].double() - lp
            kl = torch.exp(t) - t - 1
            slope = slope + a["kl_coef"] * (1 - torch.exp(t))
        if s["ref_logits"] is not None:
            y = (s["ref_logits"][part].double() * a["inv_temperature"]).masked_fill(~open_, -math.inf)
            t = logp - (y - torch.logsumexp(y, 1, keepdim=True)).masked_fill(~open_, 0.0)
            kl = (p * t).sum(1)
            extra = a["kl_coef"] * p * (t - kl[:, None])
        extra = extra + c["entropy"] * p * (logp + h[:, None])
        loss += float((w * (a["kl_coef"] * kl - gain - c["entropy"] * h)).sum())
        out["grad"].append(a["inv_temperature"] * w[:, None] * (slope[:, None] * (pick - p) + extra))
        for name, v in (("logp", lp), ("kl", kl), ("entropy", h)):
            out[name].append(v * counted)
    return {"loss": torch.tensor(loss, dtype=torch.float64)} | {n: torch.cat(out[n]) for n in list(out)[1:]}


def _exact_preference(s):
    c, a, w = s["case"], _PREFERENCE, s["weights"].double()
    logp = torch.log_softmax(s["logits"].double(), 1)
    rows = torch.arange(len(w), device=w.device)
    here = s["chosen"].clamp(min=0)
    pick = logp[rows, here]
    ends = s["offsets"].tolist()
    ratio, share = [], torch.zeros_like(w)
    for lo, hi in zip(ends, ends[1:]):
        total = float(w[lo:hi].sum()) if c["average"] else 1.0
        part = w[lo:hi] / total if total else w[lo:hi] * 0
        share[lo:hi] = part
        ratio.append(float((part * (pick[lo:hi] - s["ref_logp"][lo:hi].double())).sum()))
    loss, margins, row = 0.0, [], torch.zeros_like(w)
    for i in range(c["pairs"]):
        h = ratio[2 * i] - ratio[2 * i + 1]
        z = a["beta"] * h
        margins.append(z)
        if c["kind"] == "logistic":
            near = 1 / (1 + math.exp(-z))
            loss -= (1 - a["smoothing"]) * math.log(near) + a["smoothing"] * math.log(1 / (1 + math.exp(z)))
            d = a["beta"] * (a["smoothing"] * near - (1 - a["smoothing"]) * (1 - near))
        elif c["kind"] == "squared":
            loss += (h - 1 / (2 * a["beta"])) ** 2
            d = 2 * (h - 1 / (2 * a["beta"]))
        else:
            loss += max(0.0, a["hinge"] - z)
            d = -a["beta"] if z < a["hinge"] else 0.0
        for k, sign in ((2 * i, 1), (2 * i + 1, -1)):
            row[ends[k]:ends[k + 1]] = sign * d / c["pairs"] * share[ends[k]:ends[k + 1]]
    g = torch.exp(logp) * -row[:, None]
    g[rows, here] += row
    f64 = {"dtype": torch.float64, "device": w.device}
    return {"loss": torch.tensor(loss / c["pairs"], **f64), "margins": torch.tensor(margins, **f64),
            "ratios": torch.tensor(ratio, **f64), "grad": g}


def _exact_norm(s):
    """By torch's automatic differentiation of the definition in float64."""
    c, a = s["case"], s["args"]
    names = ("block", "stream", "post_gain", "post_bias", "gate", "pre_gain", "pre_bias")
    v = {n: s[n].double().requires_grad_(c["backward"]) for n in names if s[n] is not None}

    def normed(x, side):
        if a["norm"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + a["eps"]) * v[side + "_gain"]
        return x + v[side + "_bias"] if side + "_bias" in v else x

    update = a["scale"] * normed(v["block"], "post")
    if "gate" in v:
        update = update * {"none": lambda t: t, "sigmoid": lambda t: 1 / (1 + torch.exp(-t)),
                           "tanh": torch.tanh}[a["gate_act"]](v["gate"])
    stream = v["stream"] + update
    h = normed(stream, "pre")
    out = {"stream": stream.detach(), "out": h.detach()}
    if c["backward"]:
        torch.autograd.backward([h, stream], [s["d_out"].double(), s["d_stream"].double()])
        out |= {"d_" + n: t.grad for n, t in v.items()}
    return out


def _exact_kept(x):
    """What the 8-bit checkpoint of x stands for."""
    rows, width = x.shape
    v = torch.zeros(rows, -(-width // GROUP) * GROUP, dtype=torch.float64, device=x.device)
    v[:, :width] = x.double()
    v = v.reshape(rows, -1, GROUP)
    top = v.abs().amax(2, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120))) - 7)
    step = torch.where(127 * step >= top, step, 2 * step)
    step = torch.where(127 * step >= top, step, 2 * step)
    return (torch.round(v / step) * step).reshape(rows, -1)[:, :width]


def _exact_act(z, act):
    z = z.clone().requires_grad_(True)
    if act == "relu":
        y = z * (z > 0)
    elif act == "silu":
        y = z / (1 + torch.exp(-z))
    else:
        y = z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    [slope] = torch.autograd.grad(y.sum(), z)
    return y.detach(), slope


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "policy":
        return _exact_policy(s)
    if op == "preference":
        return _exact_preference(s)
    if op == "norm":
        return _exact_norm(s)
    if op == "weight":
        k = s["exps"].double().repeat_interleave(GROUP, 1)[:, : case["width"]] - 127
        v = s["q"].double() * torch.exp2(k)
        if case["act"] != "none":
            v = _exact_act(v, case["act"])[0]
        g = s["grad"].double()
        return {"weight": v.t() @ g, "bias": g.sum(0)}
    kept = _exact_kept(s["x"])
    if op == "recall":
        return kept
    return {"out": _exact_act(s["x"].double(), case["act"])[0],
            "grad": s["grad"].double() * _exact_act(kept, case["act"])[1]}
