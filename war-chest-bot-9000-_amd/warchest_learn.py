"""Python binding of the training operators' C ABI (include/wc_learn.h).

What a trainer of the policy or value network runs on the solver's results, on torch tensors in device memory:

- `policy_loss`: the clipped policy loss with a KL term and an entropy bonus, and its gradient, from rows of logits;
- `preference_loss`: the paired log-ratio loss over ragged sequences, and its gradient;
- `residual_norm`, `residual_norm_backward`: a block's output normed, gated, scaled and added to the residual stream, and
  the norm before the next block;
- `checkpoint8`, `checkpoint8_act`, `checkpoint8_read`, `checkpoint8_act_backward`, `checkpoint8_weight_grad`:
  activations kept in 8 bits for the backward pass, and what the backward pass does with them;
- `linear`, `linear_backward`: a layer's product with bias, activation and residual in its epilogue, and its gradients;
- `orthogonalise`: a weight's update with its singular values brought towards 1 by Newton-Schulz products;
- `token_logp`, `token_logp_backward`: log-probabilities of given tokens with their rank, the entropy and the top
  alternatives of rows of logits, and the gradient.

Every call is queued on the current stream of its tensors' device and returns at once. Outputs and scratch are allocated
with torch on that stream; a tensor made on another stream must be ready there, and kept alive by its owner
(`Tensor.record_stream`), as for torch's own operators. Matrices need unit column stride, rows may be at any stride.
Arguments that do not fit raise `WaveError`, and then nothing was queued. The `*_objective` functions, `ResidualNorm`,
`dense` and `Dense` are the same calls with torch's automatic differentiation, `Muon` an optimiser on `orthogonalise`.

Every operator goes through the native library; what `Muon` does around its update (momentum, decay, the step) and the
casts of `dense` are torch's.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct
from collections import namedtuple

import torch

import warchest_wave as ww
from warchest_wave import WaveError

# Symbols every build must export (include/wc_learn.h), beside warchest_wave.EXPORTS.
EXPORTS = [
    "wc_policy_workspace", "wc_policy_loss", "wc_preference_workspace", "wc_preference_loss",
    "wc_residual_norm", "wc_residual_norm_workspace", "wc_residual_norm_backward",
    "wc_ckpt_write", "wc_ckpt_read", "wc_ckpt_act_backward", "wc_ckpt_weight_workspace", "wc_ckpt_weight_grad",
    "wc_linear_workspace", "wc_linear", "wc_linear_backward_workspace", "wc_linear_backward",
    "wc_orthogonalise_workspace", "wc_orthogonalise",
    "wc_token_logp_workspace", "wc_token_logp", "wc_token_logp_backward",
]

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
NORMS = {"rms": 0, "layer": 1}
GATE_ACTS = {"none": 0, "sigmoid": 1, "tanh": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
KINDS = {"logistic": 0, "squared": 1, "hinge": 2}
GROUP = 32
TOP_MAX = 64

# The structures of the header, packed in C's own layout: a call fills one in one step.
_POLICY = struct.Struct("@Qii qq PqPqPq PPPPPP fffffi PPPPPq PQ")
_PREFERENCE = struct.Struct("@Qii qqq Pq PPPPP fffiii PPPPPq PQ")
_NORM = struct.Struct("@Qiiii qq PqPq PPPqPP ffii PqPq P")
_NORM_BACK = struct.Struct("@Qiiii qq PqPq PPPqP fiii PPqPq PqPq PPPPPq PQ")
_CKPT = struct.Struct("@Qii qq ii PqPq PqPq")
_WEIGHT = struct.Struct("@Qii qqq ii PqPqPqPq P PQ")
_LINEAR = struct.Struct("@Qiiii qqq PqPq P Pq ii PqPq PQ")
_LINEAR_BACK = struct.Struct("@Qiiiiii qqq PqPqPqPq PqPq P PQ")
_ORTHO = struct.Struct("@Qiiii qqq Pqq Pqq fffffi PQ")
_LOGP = struct.Struct("@Qii qq PqPq P fiii PPPPPP PQ")
_LOGP_BACK = struct.Struct("@Qii qq PqPq P fi PPP Pq")

PolicyLoss = namedtuple("PolicyLoss", "loss logp kl entropy grad")
PreferenceLoss = namedtuple("PreferenceLoss", "loss margins ratios logp grad")
ResidualNormOut = namedtuple("ResidualNormOut", "stream out stats")
ResidualNormGrads = namedtuple("ResidualNormGrads", "block stream post_gain post_bias gate pre_gain pre_bias")
Checkpoint8 = namedtuple("Checkpoint8", "q exps")
Linear = namedtuple("Linear", "out pre")
LinearGrads = namedtuple("LinearGrads", "x weight bias")
TokenLogp = namedtuple("TokenLogp", "logp entropy rank top_logp top_index stats")

_fn = {}


def _entry(name):
    f = _fn.get(name)
    if f is None:
        f = getattr(ww.lib(), name)
        f.argtypes = [C.c_char_p, C.c_void_p] if not name.endswith("workspace") else [C.c_char_p,
                                                                                     C.POINTER(C.c_uint64)]
        f.restype = C.c_int
        _fn[name] = f
    return f


# The current stream's handle by device index, without a Stream object where torch has that (2 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name, packed, device):
    rc = (_fn.get(name) or _entry(name))(packed, _raw_stream(device.index))
    if rc:
        ww._check(rc)


def _scratch_bytes(name, packed):
    n = C.c_uint64()
    ww._check(_entry(name)(packed, C.byref(n)))
    return n.value


def _fail(text):
    raise WaveError(text)


def _device(t, name):
    if not isinstance(t, torch.Tensor):
        _fail(f"{name} is not a tensor")
    d = t.device
    if d.type != "cuda":
        _fail(f"{name} is not on a GPU")
    return d


def _dtype(t, name):
    c = DTYPES.get(t.dtype)
    if c is None:
        _fail(f"{name}: {t.dtype} is not one of float32, float16, bfloat16")
    return c


def _matrix(t, name, device, dtype, rows, width):
    """(address, row stride) of a matrix that must be rows x width."""
    if t.dtype is not dtype:
        _fail(f"{name}: {t.dtype}, expected {dtype}")
    if t.device != device:
        _fail(f"{name} is on {t.device}, not on {device}")
    if t.shape != (rows, width):
        _fail(f"{name}: shape {tuple(t.shape)}, expected ({rows}, {width})")
    s = t.stride()
    if s[1] != 1 and width > 1:
        _fail(f"{name}: columns must be contiguous")
    return t.data_ptr(), s[0]


def _vector(t, name, device, dtype, n):
    """The address of a contiguous vector of n, 0 for None."""
    if t is None:
        return 0
    if t.dtype is dtype and t.device == device and t.shape == (n,) and t.is_contiguous():
        return t.data_ptr()
    if t.dtype is not dtype:
        _fail(f"{name}: {t.dtype}, expected {dtype}")
    if t.device != device:
        _fail(f"{name} is on {t.device}, not on {device}")
    if t.shape != (n,):
        _fail(f"{name}: shape {tuple(t.shape)}, expected ({n},)")
    _fail(f"{name} must be contiguous")


def _scalar(t, name, device):
    if t is None:
        return 0
    if t.dtype != torch.float32 or t.numel() != 1 or t.device != device:
        _fail(f"{name} is one float32 on {device}")
    return t.data_ptr()


def _indices(t, name, device, n):
    if t.dtype not in (torch.int64, torch.int32):
        _fail(f"{name}: {t.dtype}, expected int64 or int32")
    return _vector(t, name, device, t.dtype, n), 64 if t.dtype == torch.int64 else 32


def _known(table, key, name):
    if key not in table:
        _fail(f"{name}: {key!r} is not one of {', '.join(table)}")
    return table[key]


def _logits(t):
    device = _device(t, "logits")
    code = _dtype(t, "logits")
    if t.dim() != 2:
        _fail(f"logits: shape {tuple(t.shape)}, expected rows x vocab")
    rows, vocab = t.shape
    return device, code, rows, vocab, _matrix(t, "logits", device, t.dtype, rows, vocab)


# Scratch sizes depend on shapes (and, for the weight gradient, on whether its rows start on 16 bytes).
@functools.lru_cache(maxsize=4096)
def _policy_scratch(device, code, rows, vocab):
    p = 256  # an address that passes for one: the size is computed from the shape, nothing is read
    return _scratch_bytes("wc_policy_workspace", _POLICY.pack(
        _POLICY.size, device, code, rows, vocab, p, vocab, 0, 0, 0, 0, p, p, p, 0, 0, 0, 1.0, 0.0, 0.0, 0.0, 0.0, 64,
        p, p, p, p, 0, 0, 0, 0))


@functools.lru_cache(maxsize=4096)
def _preference_scratch(device, code, rows, vocab, pairs):
    p = 256
    return _scratch_bytes("wc_preference_workspace", _PREFERENCE.pack(
        _PREFERENCE.size, device, code, rows, vocab, pairs, p, vocab, p, p, p, 0, 0, 1.0, 1.0, 0.0, 0, 0, 64, p, p, p,
        p, 0, 0, 0, 0))


@functools.lru_cache(maxsize=4096)
def _norm_scratch(device, code, rows, width):
    p = 256
    return _scratch_bytes("wc_residual_norm_workspace", _NORM_BACK.pack(
        _NORM_BACK.size, device, code, 0, 0, rows, width, p, width, p, width, 0, 0, 0, 0, 0, 1.0, 0, 0, 0, p, 0, 0, 0, 0,
        p, width, p, width, 0, 0, 0, 0, 0, 0, 0, 0))


@functools.lru_cache(maxsize=4096)
def _weight_scratch(device, code, rows, width, out, act, weight_code, aligned):
    p, stride = 256, out if aligned else out + 1 - out % 2
    return _scratch_bytes("wc_ckpt_weight_workspace", _WEIGHT.pack(
        _WEIGHT.size, device, code, rows, width, out, act, weight_code, p, width, p, -(-width // GROUP), p, stride, p,
        out, p, 0, 0))


def _scratch(n, device):
    """(tensor, address) of a call's workspace; nothing is allocated for none."""
    if not n:
        return None, 0
    t = torch.empty(n, dtype=torch.uint8, device=device)
    return t, t.data_ptr()


def _like(t):
    """A new contiguous tensor of t's shape, type and device."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def policy_loss(logits, actions, behaviour_logp, advantages, weights=None, *, legal=None, ref_logp=None, ref_logits=None,
                inv_temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, grad=True,
                grad_out=None):
    """The clipped policy loss of rows of logits, and its gradient (wc_policy_loss).

    logits [rows, vocab]; actions [rows] int64 or int32; behaviour_logp, advantages, weights, ref_logp [rows] float32
    (weights None: 1/rows each); legal [rows, vocab] bool; ref_logits like logits. A row of weight 0, with an action that
    is out of range or not legal, or without a legal logit above -infinity is left out. grad: True, a tensor like
    logits to write to (logits itself works), or False; grad_out: one float32, what arrives at the loss.
    Returns PolicyLoss(loss, logp, kl, entropy, grad): logp of the actions, KL and entropy per row."""
    device, code, rows, vocab, (x, xs) = _logits(logits)
    a, bits = _indices(actions, "actions", device, rows)
    f32 = torch.float32
    lg, lgs = (0, 0) if legal is None else _matrix(legal, "legal", device, torch.bool, rows, vocab)
    rl, rls = (0, 0) if ref_logits is None else _matrix(ref_logits, "ref_logits", device, logits.dtype, rows, vocab)
    if grad is True:
        grad = _like(logits)
        g, gs = grad.data_ptr(), vocab
    elif grad is False or grad is None:
        grad, g, gs = None, 0, 0
    else:
        g, gs = _matrix(grad, "grad", device, logits.dtype, rows, vocab)
    loss = torch.empty((), dtype=f32, device=device)
    logp, kl, entropy = torch.empty((3, rows), dtype=f32, device=device).unbind(0)
    need = _policy_scratch(device.index, code, rows, vocab)
    held, work = _scratch(need, device)
    at = logp.data_ptr()
    _call("wc_policy_loss", _POLICY.pack(
        _POLICY.size, device.index, code, rows, vocab, x, xs, lg, lgs, rl, rls, a,
        _vector(behaviour_logp, "behaviour_logp", device, f32, rows),
        _vector(advantages, "advantages", device, f32, rows), _vector(weights, "weights", device, f32, rows),
        _vector(ref_logp, "ref_logp", device, f32, rows), _scalar(grad_out, "grad_out", device), inv_temperature,
        clip_low, clip_high, kl_coef, entropy_coef, bits, loss.data_ptr(), at, at + 4 * rows, at + 8 * rows, g, gs, work,
        need), device)
    return PolicyLoss(loss, logp, kl, entropy, grad)


def preference_loss(logits, tokens, offsets, ref_logp, weights=None, *, beta=0.1, smoothing=0.0, kind="logistic",
                    average=False, inv_temperature=1.0, grad=True, grad_out=None):
    """The paired preference loss of ragged sequences of rows of logits, and its gradient (wc_preference_loss).

    logits [rows, vocab]; tokens [rows] and offsets [2 pairs + 1], both int64 or both int32; ref_logp, weights [rows]
    float32 (weights None: 1). Sequence s is the rows offsets[s] .. offsets[s + 1]; pair i prefers sequence 2i to
    2i + 1. kind: "logistic", "squared" or "hinge"; average: ratios per unit of weight. grad, grad_out as policy_loss.
    Returns PreferenceLoss(loss, margins, ratios, logp, grad)."""
    device, code, rows, vocab, (x, xs) = _logits(logits)
    t, bits = _indices(tokens, "tokens", device, rows)
    if offsets.dim() != 1 or offsets.shape[0] % 2 != 1:
        _fail(f"offsets: shape {tuple(offsets.shape)}, expected (2 pairs + 1,)")
    pairs = offsets.shape[0] // 2
    f32 = torch.float32
    off = _vector(offsets, "offsets", device, tokens.dtype, 2 * pairs + 1)
    if ref_logp is None:
        _fail("ref_logp is missing")
    if grad is True:
        grad = _like(logits)
        g, gs = grad.data_ptr(), vocab
    elif grad is False or grad is None:
        grad, g, gs = None, 0, 0
    else:
        g, gs = _matrix(grad, "grad", device, logits.dtype, rows, vocab)
    loss = torch.empty((), dtype=f32, device=device)
    outs = torch.empty(3 * pairs + rows, dtype=f32, device=device)
    margins, ratios, logp = outs.split((pairs, 2 * pairs, rows))
    need = _preference_scratch(device.index, code, rows, vocab, pairs)
    held, work = _scratch(need, device)
    at = outs.data_ptr()
    _call("wc_preference_loss", _PREFERENCE.pack(
        _PREFERENCE.size, device.index, code, rows, vocab, pairs, x, xs, t, off,
        _vector(ref_logp, "ref_logp", device, f32, rows), _vector(weights, "weights", device, f32, rows),
        _scalar(grad_out, "grad_out", device), inv_temperature, beta, smoothing, _known(KINDS, kind, "kind"),
        int(bool(average)), bits, loss.data_ptr(), at, at + 4 * pairs, at + 12 * pairs, g, gs, work, need), device)
    return PreferenceLoss(loss, margins, ratios, logp, grad)


def _norm_inputs(block, stream, post_gain, post_bias, gate, pre_gain, pre_bias):
    """What both directions of residual_norm check: device, codes, shape, addresses."""
    device = _device(block, "block")
    code = _dtype(block, "block")
    if block.dim() != 2:
        _fail(f"block: shape {tuple(block.shape)}, expected rows x width")
    rows, width = block.shape
    b = _matrix(block, "block", device, block.dtype, rows, width)
    s = _matrix(stream, "stream", device, block.dtype, rows, width)
    vector = gate is not None and gate.dim() == 1
    dt = next((p.dtype for p in (post_gain, post_bias, gate if vector else None, pre_gain, pre_bias)
               if p is not None), block.dtype)
    pcode = DTYPES.get(dt)
    if pcode is None:
        _fail(f"gains and biases: {dt} is not one of float32, float16, bfloat16")
    if gate is None:
        g = (0, 0)
    elif vector:
        g = (_vector(gate, "gate", device, dt, width), 0)
    else:
        g = _matrix(gate, "gate", device, block.dtype, rows, width)
        if g[1] == 0 and rows > 1:
            _fail("gate: one row for all is given as a vector")
        g = (g[0], g[1] or width)
    return (device, code, pcode, rows, width, b, s, _vector(post_gain, "post_gain", device, dt, width),
            _vector(post_bias, "post_bias", device, dt, width), g, _vector(pre_gain, "pre_gain", device, dt, width),
            _vector(pre_bias, "pre_bias", device, dt, width))


def residual_norm(block, stream, post_gain=None, post_bias=None, gate=None, pre_gain=None, pre_bias=None, *, scale=1.0,
                  eps=1e-5, norm="layer", gate_act="none", stats=True):
    """stream' = stream + scale * act(gate) * (norm(block) * post_gain + post_bias), and
    out = norm(stream') * pre_gain + pre_bias (wc_residual_norm).

    block, stream [rows, width] of one type; gains and biases [width], in that type or another of the three; gate
    [width] (learned, in the gains' type), [rows, width] (in the matrices' type) or None. norm: "layer" or "rms";
    gate_act: "none", "sigmoid" or "tanh". Returns ResidualNormOut(stream, out, stats); stats [rows, 4] is what
    residual_norm_backward needs (stats=False: not kept)."""
    device, code, pcode, rows, width, b, s, pg, pb, g, ng, nb = _norm_inputs(block, stream, post_gain, post_bias, gate,
                                                                             pre_gain, pre_bias)
    new, out = _like(block), _like(block)
    st = torch.empty((rows, 4), dtype=torch.float32, device=device) if stats else None
    _call("wc_residual_norm", _NORM.pack(
        _NORM.size, device.index, code, pcode, 0, rows, width, *b, *s, pg, pb, *g, ng, nb, scale, eps,
        _known(NORMS, norm, "norm"), _known(GATE_ACTS, gate_act, "gate_act"), new.data_ptr(), width, out.data_ptr(),
        width, st.data_ptr() if stats else 0), device)
    return ResidualNormOut(new, out, st)


def residual_norm_backward(d_out, d_stream, block, stream, stats, post_gain=None, post_bias=None, gate=None,
                           pre_gain=None, pre_bias=None, *, scale=1.0, eps=1e-5, norm="layer", gate_act="none"):
    """The gradients of residual_norm from its inputs and its stats (wc_residual_norm_backward).

    d_out arrives at out, d_stream at stream' (either may be None: 0). Returns ResidualNormGrads(block, stream,
    post_gain, post_bias, gate, pre_gain, pre_bias): matrices in the inputs' type, parameters in float32, None for a
    parameter that was None. The forward's keyword arguments fit: eps is in its stats already."""
    device, code, pcode, rows, width, b, s, pg, pb, g, ng, _ = _norm_inputs(block, stream, post_gain, post_bias, gate,
                                                                            pre_gain, pre_bias)
    dt, f32 = block.dtype, torch.float32
    do = (0, 0) if d_out is None else _matrix(d_out, "d_out", device, dt, rows, width)
    ds = (0, 0) if d_stream is None else _matrix(d_stream, "d_stream", device, dt, rows, width)
    if stats is None:
        _fail("stats is missing")
    st, _ = _matrix(stats, "stats", device, f32, rows, 4)
    if rows > 1 and stats.stride(0) != 4:
        _fail("stats must be contiguous")
    token = gate is not None and gate.dim() == 2
    mats = [_like(block) for _ in range(3 if token else 2)]
    wanted = [p is not None and not (token and p is gate) for p in (post_gain, post_bias, gate, pre_gain, pre_bias)]
    sums = iter(torch.empty((sum(wanted), width), dtype=f32, device=device).unbind(0))
    dpg, dpb, dg, dng, dnb = (next(sums) if w else None for w in wanted)
    if token:
        dg = mats[2]
    need = _norm_scratch(device.index, code, rows, width)
    held, work = _scratch(need, device)
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    _call("wc_residual_norm_backward", _NORM_BACK.pack(
        _NORM_BACK.size, device.index, code, pcode, 0, rows, width, *b, *s, pg, pb, *g, ng, scale,
        _known(NORMS, norm, "norm"), _known(GATE_ACTS, gate_act, "gate_act"), 0, st, *do, *ds, mats[0].data_ptr(), width,
        mats[1].data_ptr(), width, at(dpg), at(dpb), at(dng), at(dnb), at(dg), width, work, need), device)
    return ResidualNormGrads(mats[0], mats[1], dpg, dpb, dg, dng, dnb)


def _kept(ck):
    """A checkpoint's device, shape and addresses."""
    q, exps = ck
    device = _device(q, "q")
    if q.dim() != 2:
        _fail(f"q: shape {tuple(q.shape)}, expected rows x width")
    rows, width = q.shape
    return device, rows, width, _matrix(q, "q", device, torch.int8, rows, width), _matrix(
        exps, "exps", device, torch.uint8, rows, -(-width // GROUP))


def _write(x, act, want):
    device = _device(x, "x")
    code = _dtype(x, "x")
    if x.dim() != 2:
        _fail(f"x: shape {tuple(x.shape)}, expected rows x width")
    rows, width = x.shape
    groups = -(-width // GROUP)
    at = _matrix(x, "x", device, x.dtype, rows, width)
    q = torch.empty((rows, width), dtype=torch.int8, device=device)
    exps = torch.empty((rows, groups), dtype=torch.uint8, device=device)
    y = torch.empty((rows, width), dtype=x.dtype, device=device) if want else None
    _call("wc_ckpt_write", _CKPT.pack(_CKPT.size, device.index, code, rows, width, _known(ACTS, act, "act"), 0,
                                      q.data_ptr(), width, exps.data_ptr(), groups, *at, y.data_ptr() if want else 0,
                                      width), device)
    return Checkpoint8(q, exps), y


def checkpoint8(x):
    """x [rows, width] kept in 8 bits: Checkpoint8(q, exps), int8 [rows, width] and one exponent byte for each 32
    channels of a row (wc_ckpt_write)."""
    return _write(x, "none", False)[0]


def checkpoint8_act(x, act):
    """(Checkpoint8 of x, act(x)) in one pass. act: "relu", "gelu", "silu" or "none"."""
    return _write(x, act, True)


def _read(name, ck, act, grad, dtype):
    device, rows, width, q, e = _kept(ck)
    y = torch.empty((rows, width), dtype=dtype, device=device)
    x = (0, 0) if grad is None else _matrix(grad, "grad", device, dtype, rows, width)
    _call(name, _CKPT.pack(_CKPT.size, device.index, _dtype(y, "dtype"), rows, width, _known(ACTS, act, "act"), 0, *q, *e,
                           *x, y.data_ptr(), width), device)
    return y


def checkpoint8_read(ck, dtype=torch.bfloat16, act="none"):
    """act(what a checkpoint stands for) (wc_ckpt_read)."""
    return _read("wc_ckpt_read", ck, act, None, dtype)


def checkpoint8_act_backward(ck, grad, act):
    """grad * act'(what a checkpoint stands for) (wc_ckpt_act_backward)."""
    _device(grad, "grad")
    return _read("wc_ckpt_act_backward", ck, act, grad, grad.dtype)


def checkpoint8_weight_grad(ck, grad, *, act="none", bias=False, dtype=None):
    """(weight, bias): weight [width, out] = act(kept)^T grad, the gradient of x @ weight; bias [out] float32 = grad's
    column sums (None unless asked for) (wc_ckpt_weight_grad). dtype: float32 (the default) or grad's. gelu and silu are
    taken with a 16-bit grad, and rounded to its type; checkpoint8_read gives them in float32 for a plain product."""
    device, rows, width, q, e = _kept(ck)
    if _device(grad, "grad") != device or grad.dim() != 2:
        _fail(f"grad: shape {tuple(grad.shape)} on {grad.device}, expected rows x out on {device}")
    code, out = _dtype(grad, "grad"), grad.shape[1]
    g = _matrix(grad, "grad", device, grad.dtype, rows, out)
    weight = torch.empty((width, out), dtype=dtype or torch.float32, device=device)
    wcode = _dtype(weight, "dtype")
    b = torch.empty(out, dtype=torch.float32, device=device) if bias else None
    a = _known(ACTS, act, "act")
    # (rows 2^29 elements apart count as unaligned: the library copies them)
    aligned = (g[0] | 2 * g[1] | 2 * out) % 16 == 0 and g[1] < 1 << 29
    need = _weight_scratch(device.index, code, rows, width, out, a, wcode, aligned)
    held, work = _scratch(need, device)
    _call("wc_ckpt_weight_grad", _WEIGHT.pack(
        _WEIGHT.size, device.index, code, rows, width, out, a, wcode, *q, *e, *g, weight.data_ptr(), out,
        b.data_ptr() if bias else 0, work, need), device)
    return weight, b


# ------------------------------------------------------------------ layers

def _weight_of(t, name, device, dtype, width, out):
    """(address, row stride, layout) of a weight [width, out] that is contiguous along either index."""
    if not isinstance(t, torch.Tensor) or t.shape != (width, out):
        _fail(f"{name}: shape {tuple(getattr(t, 'shape', ()))}, expected ({width}, {out})")
    s = t.stride()
    if s[1] == 1 or out == 1 or s[0] != 1:
        return *_matrix(t, name, device, dtype, width, out), 0
    if t.dtype is not dtype:
        _fail(f"{name}: {t.dtype}, expected {dtype}")
    if t.device != device:
        _fail(f"{name} is on {t.device}, not on {device}")
    return t.data_ptr(), s[1], 1


# An address that passes for one, on 16 bytes or not: scratch depends on shapes and on where rows start, nothing is read.
def _stand_in(aligned):
    return 256 if aligned else 260


@functools.lru_cache(maxsize=4096)
def _linear_scratch(device, code, layout, rows, width, out, xs, ws, x_aligned, w_aligned):
    p = 256
    return _scratch_bytes("wc_linear_workspace", _LINEAR.pack(
        _LINEAR.size, device, code, 0, layout, rows, width, out, _stand_in(x_aligned), xs, _stand_in(w_aligned), ws, 0, 0,
        0, 0, 0, 0, 0, p, out, 0, 0))


@functools.lru_cache(maxsize=4096)
def _linear_back_scratch(device, code, layout, act, rows, width, out, ds, xs, ws, d_aligned, x_aligned, w_aligned, d_x,
                         d_weight, d_bias):
    p = 256
    return _scratch_bytes("wc_linear_backward_workspace", _LINEAR_BACK.pack(
        _LINEAR_BACK.size, device, code, layout, act, 0, 0, rows, width, out, _stand_in(d_aligned), ds, p, out,
        _stand_in(x_aligned), xs, _stand_in(w_aligned), ws, p if d_x else 0, width, p if d_weight else 0,
        width if layout else out, p if d_bias else 0, 0, 0))


def linear(x, weight, bias=None, *, act="none", residual=None, keep=False):
    """act(x @ weight + bias) + residual in one product (wc_linear).

    x [rows, width], weight [width, out] (contiguous along either index: the transposed view of an [out, width] matrix
    works as it is), bias [out] in their type or float32, residual [rows, out]. act: "none", "relu", "gelu" or "silu".
    Returns Linear(out, pre): pre [rows, out] float32, x @ weight + bias, is what linear_backward needs; None unless keep is
    true and act is not "none"."""
    device = _device(x, "x")
    code, dt = _dtype(x, "x"), x.dtype
    if x.dim() != 2:
        _fail(f"x: shape {tuple(x.shape)}, expected rows x width")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        _fail("weight: expected width x out")
    rows, width = x.shape
    out = weight.shape[1]
    xp, xs = _matrix(x, "x", device, dt, rows, width)
    wp, ws, layout = _weight_of(weight, "weight", device, dt, width, out)
    bias_code = 0
    if bias is not None:
        if bias.dtype not in (dt, torch.float32):
            _fail(f"bias: {bias.dtype}, expected {dt} or float32")
        bias_code = DTYPES[bias.dtype]
    b = _vector(bias, "bias", device, None if bias is None else bias.dtype, out)
    r = (0, 0) if residual is None else _matrix(residual, "residual", device, dt, rows, out)
    a = _known(ACTS, act, "act")
    y = torch.empty((rows, out), dtype=dt, device=device)
    pre = torch.empty((rows, out), dtype=torch.float32, device=device) if keep and a else None
    need = _linear_scratch(device.index, code, layout, rows, width, out, xs, ws, xp % 16 == 0, wp % 16 == 0)
    held, work = _scratch(need, device)
    _call("wc_linear", _LINEAR.pack(
        _LINEAR.size, device.index, code, bias_code, layout, rows, width, out, xp, xs, wp, ws, b, *r, a, 0,
        0 if pre is None else pre.data_ptr(), out, y.data_ptr(), out, work, need), device)
    return Linear(y, pre)


def linear_backward(d_out, x, weight, pre=None, *, act="none", bias=False, d_x=True, d_weight=True, dtype=None):
    """The gradients of linear from its inputs and its pre (wc_linear_backward); the residual's is d_out itself.

    d_out [rows, out]; pre may be None where act is "none". bias, d_x, d_weight: which are wanted. dtype: the weight's
    gradient's type, x's (the default) or float32. The gradient at the pre-activations is rounded to x's type for its
    products, as between two operators; float32 matrices keep it. Returns LinearGrads(x, weight, bias): weight contiguous along the
    index that the weight is, bias in float32, None for what is not wanted."""
    device = _device(x, "x")
    code, dt = _dtype(x, "x"), x.dtype
    if x.dim() != 2:
        _fail(f"x: shape {tuple(x.shape)}, expected rows x width")
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        _fail("weight: expected width x out")
    rows, width = x.shape
    out = weight.shape[1]
    a = _known(ACTS, act, "act")
    if a and pre is None:
        _fail("pre is missing")
    xp, xs = _matrix(x, "x", device, dt, rows, width)
    wp, ws, layout = _weight_of(weight, "weight", device, dt, width, out)
    dp, ds = _matrix(d_out, "d_out", device, dt, rows, out)
    z = _matrix(pre, "pre", device, torch.float32, rows, out) if a else (0, 0)
    gx = torch.empty((rows, width), dtype=dt, device=device) if d_x else None
    gw = None
    if d_weight:
        gw = torch.empty((out, width) if layout else (width, out), dtype=dtype or dt, device=device)
        if gw.dtype not in (dt, torch.float32):
            _fail(f"dtype: {gw.dtype}, expected {dt} or float32")
    gb = torch.empty(out, dtype=torch.float32, device=device) if bias else None
    need = _linear_back_scratch(device.index, code, layout, a, rows, width, out, ds, xs, ws, dp % 16 == 0, xp % 16 == 0,
                                wp % 16 == 0, bool(d_x), bool(d_weight), bool(bias))
    held, work = _scratch(need, device)
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    _call("wc_linear_backward", _LINEAR_BACK.pack(
        _LINEAR_BACK.size, device.index, code, layout, a, DTYPES[gw.dtype] if d_weight else 0, 0, rows, width, out, dp,
        ds, *z, xp, xs, wp, ws, at(gx), width, at(gw), width if layout else out, at(gb), work, need), device)
    return LinearGrads(gx, gw.t() if d_weight and layout else gw, gb)


# ------------------------------------------------------------------ updates

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


@functools.lru_cache(maxsize=4096)
def _ortho_scratch(device, code, out_code, batch, rows, width):
    p, q = 256, 512
    return _scratch_bytes("wc_orthogonalise_workspace", _ORTHO.pack(
        _ORTHO.size, device, code, out_code, 1, batch, rows, width, p, width, rows * width, q, width, rows * width, 1.0,
        0.0, 0.0, 0.0, 1.0, 0, 0, 0))


def orthogonalise(update, *, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, scale=1.0, dtype=None):
    """update [rows, width] or [batch, rows, width] with its singular values brought towards 1, times scale
    (wc_orthogonalise): X = update / (its Frobenius norm + eps), then `steps` times X = a X + (b A + c A A) X with
    A = X X^T (or the transposed form) and (a, b, c) = coefficients. dtype: the result's, float32, float16 or bfloat16
    (the default is the update's); a bfloat16 result takes a third of the others' products, in 11 bits where they have 22
    (float32 and a cast keep these). Coefficients under which a singular value s of any step has s^2 or |b s^2 + c s^4| past
    63, or the result one past 63 before scale, give infinities or NaN. Returns a contiguous tensor."""
    device = _device(update, "update")
    code = _dtype(update, "update")
    if update.dim() not in (2, 3) or 0 in update.shape[-2:]:
        _fail(f"update: shape {tuple(update.shape)}, expected rows x width or batch x rows x width")
    three = update if update.dim() == 3 else update[None]
    batch, rows, width = three.shape
    s = three.stride()
    if s[2] != 1 and width > 1:
        _fail("update: columns must be contiguous")
    if len(coefficients) != 3:
        _fail("coefficients: three are expected")
    out = torch.empty(update.shape, dtype=dtype or update.dtype, device=device)
    out_code = _dtype(out, "dtype")
    need = _ortho_scratch(device.index, code, out_code, batch, rows, width)
    held, work = _scratch(need, device)
    _call("wc_orthogonalise", _ORTHO.pack(
        _ORTHO.size, device.index, code, out_code, steps, batch, rows, width, three.data_ptr(), s[1], s[0],
        out.data_ptr(), width, rows * width, *coefficients, eps, scale, 0, work, need), device)
    return out


# -------------------------------------------------------- log-probabilities

@functools.lru_cache(maxsize=4096)
def _logp_scratch(device, code, rows, vocab, top):
    p = 256
    return _scratch_bytes("wc_token_logp_workspace", _LOGP.pack(
        _LOGP.size, device, code, rows, vocab, p, vocab, 0, 0, 0, 1.0, 64, top, 0, p, p, p, p, p, 0, 0, 0))


def token_logp(logits, tokens=None, *, legal=None, inv_temperature=1.0, top=0, stats=True):
    """Log-probabilities of the rows' tokens, their rank, the entropy and the `top` likeliest columns (wc_token_logp).

    logits [rows, vocab]; tokens [rows] int64 or int32, or None; legal [rows, vocab] bool. A row whose token is out of
    range, or without a legal logit above -infinity, is left out. Returns TokenLogp(logp, entropy, rank, top_logp,
    top_index, stats): rank int32, how many columns come before the token (0: the likeliest, -1: left out; of a token
    without a probability all of a lower index do); top_logp
    and top_index [rows, top] (int32, -1 where there are no more), None for top=0; logp and rank None without tokens;
    stats [rows, 4] is what token_logp_backward needs (stats=False: not kept)."""
    device, code, rows, vocab, (x, xs) = _logits(logits)
    f32, i32 = torch.float32, torch.int32
    t, bits = (0, 64) if tokens is None else _indices(tokens, "tokens", device, rows)
    lg, lgs = (0, 0) if legal is None else _matrix(legal, "legal", device, torch.bool, rows, vocab)
    if not isinstance(top, int) or not 0 <= top <= TOP_MAX:
        _fail(f"top: {top!r} is not 0 to {TOP_MAX}")
    entropy = torch.empty(rows, dtype=f32, device=device)
    logp = rank = top_logp = top_index = st = None
    if tokens is not None:
        logp = torch.empty(rows, dtype=f32, device=device)
        rank = torch.empty(rows, dtype=i32, device=device)
    if top:
        top_logp = torch.empty((rows, top), dtype=f32, device=device)
        top_index = torch.empty((rows, top), dtype=i32, device=device)
    if stats:
        st = torch.empty((rows, 4), dtype=f32, device=device)
    need = _logp_scratch(device.index, code, rows, vocab, top)
    held, work = _scratch(need, device)
    at = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    _call("wc_token_logp", _LOGP.pack(
        _LOGP.size, device.index, code, rows, vocab, x, xs, lg, lgs, t, inv_temperature, bits, top, 0, at(logp),
        entropy.data_ptr(), at(rank), at(top_logp), at(top_index), at(st), work, need), device)
    return TokenLogp(logp, entropy, rank, top_logp, top_index, st)


def token_logp_backward(d_logp, d_entropy, logits, tokens, stats, *, legal=None, inv_temperature=1.0, grad=None):
    """The gradient at the logits from what arrives at token_logp's logp and entropy ([rows] float32, either may be
    None: 0), from the forward's inputs and its stats (wc_token_logp_backward). grad: a tensor like logits to write to
    (logits itself works)."""
    device, code, rows, vocab, (x, xs) = _logits(logits)
    t, bits = (0, 64) if tokens is None else _indices(tokens, "tokens", device, rows)
    lg, lgs = (0, 0) if legal is None else _matrix(legal, "legal", device, torch.bool, rows, vocab)
    if stats is None:
        _fail("stats is missing")
    st, _ = _matrix(stats, "stats", device, torch.float32, rows, 4)
    if rows > 1 and stats.stride(0) != 4:
        _fail("stats must be contiguous")
    if grad is None:
        grad = _like(logits)
    g, gs = _matrix(grad, "grad", device, logits.dtype, rows, vocab)
    f32 = torch.float32
    _call("wc_token_logp_backward", _LOGP_BACK.pack(
        _LOGP_BACK.size, device.index, code, rows, vocab, x, xs, lg, lgs, t, inv_temperature, bits, st,
        _vector(d_logp, "d_logp", device, f32, rows), _vector(d_entropy, "d_entropy", device, f32, rows), g, gs), device)
    return grad


# ------------------------------------------------------- automatic differentiation

class _First(torch.autograd.Function):
    """A gradient as it is, whose own derivative raises."""

    @staticmethod
    def forward(ctx, grad, *sources):
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        _fail("a second derivative: the backward passes are native calls without derivatives of their own")


def _first_only(backward):
    """With create_graph the gradients depend on what they were computed from, by a node that raises: torch's own
    once_differentiable adds none where what arrives is a constant, and such a derivative would be 0."""
    @functools.wraps(backward)
    def first(ctx, *arrived):
        if not torch.is_grad_enabled():
            return backward(ctx, *arrived)
        with torch.no_grad():
            grads = backward(ctx, *arrived)
        sources = [t for t in (*ctx.saved_tensors, *arrived) if t is not None and t.requires_grad]
        return tuple(None if g is None else _First.apply(g, *sources) for g in grads)
    return first


def _upstream(g):
    return g if g.dtype is torch.float32 else g.float()


class _PolicyObjective(torch.autograd.Function):
    # The backward pass reads every tensor again: all of them are saved, so that torch refuses it if one was written since.
    @staticmethod
    def forward(ctx, logits, kw, *rows):
        r = _PolicyObjective.call(logits, kw, *rows, grad=False)
        ctx.save_for_backward(logits, *rows)
        ctx.kw = kw
        ctx.mark_non_differentiable(r.logp, r.kl, r.entropy)
        return r.loss, r.logp, r.kl, r.entropy

    @staticmethod
    def call(logits, kw, actions, behaviour_logp, advantages, weights, legal, ref_logp, ref_logits, **more):
        return policy_loss(logits, actions, behaviour_logp, advantages, weights, legal=legal, ref_logp=ref_logp,
                           ref_logits=ref_logits, **kw, **more)

    @staticmethod
    @_first_only
    def backward(ctx, d_loss, *_):
        logits, *rows = ctx.saved_tensors
        grad = _PolicyObjective.call(logits, ctx.kw, *rows, grad_out=_upstream(d_loss)).grad
        return grad, None, *(None for _ in rows)


def policy_objective(logits, actions, behaviour_logp, advantages, weights=None, *, legal=None, ref_logp=None,
                     ref_logits=None, **kw):
    """policy_loss as a differentiable function of the logits, and of nothing else: (loss, logp, kl, entropy). The
    backward pass reads the logits and the other tensors again instead of keeping a gradient; one that was written in
    between makes it raise, as it does with torch's own operators."""
    return _PolicyObjective.apply(logits, kw, actions, behaviour_logp, advantages, weights, legal, ref_logp, ref_logits)


class _PreferenceObjective(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, kw, *rows):
        r = preference_loss(logits, *rows, grad=False, **kw)
        ctx.save_for_backward(logits, *rows)
        ctx.kw = kw
        ctx.mark_non_differentiable(r.margins, r.ratios)
        return r.loss, r.margins, r.ratios

    @staticmethod
    @_first_only
    def backward(ctx, d_loss, *_):
        logits, *rows = ctx.saved_tensors
        grad = preference_loss(logits, *rows, grad_out=_upstream(d_loss), **ctx.kw).grad
        return grad, None, *(None for _ in rows)


def preference_objective(logits, tokens, offsets, ref_logp, weights=None, **kw):
    """preference_loss as a differentiable function of the logits, and of nothing else: (loss, margins, ratios). Its
    backward pass reads every tensor again, as policy_objective's."""
    return _PreferenceObjective.apply(logits, kw, tokens, offsets, ref_logp, weights)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, block, stream, post_gain, post_bias, gate, pre_gain, pre_bias, kw):
        r = residual_norm(block, stream, post_gain, post_bias, gate, pre_gain, pre_bias, **kw)
        ctx.save_for_backward(block, stream, r.stats, post_gain, post_bias, gate, pre_gain, pre_bias)
        ctx.kw = kw
        return r.stream, r.out

    @staticmethod
    @_first_only
    def backward(ctx, d_stream, d_out):
        saved = ctx.saved_tensors
        g = residual_norm_backward(d_out.contiguous(), d_stream.contiguous(), *saved, **ctx.kw)
        cast = [d if d is None else d.to(p.dtype) for d, p in zip(g[2:], saved[3:])]
        return (g.block, g.stream, *cast, None)


class ResidualNorm(torch.nn.Module):
    """The residual update between two norms, with its parameters: (stream', out) of (block, stream)."""

    def __init__(self, width, norm="layer", gate=True, gate_act="none", scale=1.0, eps=1e-5, device=None,
                 dtype=torch.float32):
        super().__init__()
        make = lambda v: torch.nn.Parameter(torch.full((width,), v, device=device, dtype=dtype))  # noqa: E731
        self.post_gain, self.pre_gain = make(1.0), make(1.0)
        self.post_bias, self.pre_bias = (make(0.0), make(0.0)) if norm == "layer" else (None, None)
        self.gate = make(1.0 if gate_act == "none" else 0.0) if gate else None
        self.kw = {"norm": norm, "gate_act": gate_act, "scale": scale, "eps": eps}

    def forward(self, block, stream, gate=None):
        return _ResidualNorm.apply(block, stream, self.post_gain, self.post_bias, self.gate if gate is None else gate,
                                   self.pre_gain, self.pre_bias, self.kw)


class _ActLinear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, weight, act):
        kept, a = checkpoint8_act(z, act)
        link = z.new_empty(0)  # an output: leads from the backward pass to z, which is not kept
        ctx.save_for_backward(kept.q, kept.exps, weight, link)
        ctx.set_materialize_grads(False)  # nothing arrives at link
        ctx.act = act
        return a @ weight, link

    @staticmethod
    @_first_only
    def backward(ctx, d, _):
        q, exps, weight, _ = ctx.saved_tensors
        kept, d = Checkpoint8(q, exps), d.contiguous()
        d_z = checkpoint8_act_backward(kept, d @ weight.t(), ctx.act) if ctx.needs_input_grad[0] else None
        d_w = None
        if ctx.needs_input_grad[1]:
            if d.dtype is torch.float32 and ctx.act in ("gelu", "silu"):
                # not an 8-bit operand any more, and to be kept in 32 bits: a plain product, as the forward's
                d_w = checkpoint8_read(kept, torch.float32, ctx.act).t() @ d
            else:
                d_w = checkpoint8_weight_grad(kept, d, act=ctx.act, dtype=weight.dtype)[0]
        return d_z, d_w, None


def act_linear8(z, weight, act="gelu"):
    """act(z) @ weight (z [rows, width], weight [width, out] of one type), keeping z for the backward pass in 8 bits and
    act(z) not at all: its slope and the weight's gradient are taken from the 8-bit form. In float32 with gelu or silu the
    backward pass makes act(kept) in float32 for the weight's gradient (rows x width x 4 bytes while it runs)."""
    return _ActLinear8.apply(z, weight, act)[0]


class _Dense(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, keep):
        cast = None
        if all(isinstance(t, torch.Tensor) and t.dtype in DTYPES for t in (x, weight)) and weight.dtype is not x.dtype:
            cast = weight.to(x.dtype)
        r = linear(x, weight if cast is None else cast, bias, act=act, residual=residual, keep=keep)
        ctx.save_for_backward(x, weight, bias, r.pre, cast)
        ctx.act = act
        return r.out

    @staticmethod
    @_first_only
    def backward(ctx, d):
        x, weight, bias, pre, cast = ctx.saved_tensors
        need = ctx.needs_input_grad
        d_weight = d_bias = None
        g = LinearGrads(None, None, None)
        if any(need[:3]):
            # of a weight that was cast the gradient is not rounded to the products' type
            g = linear_backward(d.contiguous(), x, weight if cast is None else cast, pre, act=ctx.act, bias=need[2],
                                d_x=need[0], d_weight=need[1], dtype=None if cast is None else torch.float32)
            d_weight = g.weight.to(weight.dtype) if need[1] else None
            d_bias = g.bias.to(bias.dtype) if need[2] else None
        return g.x, d_weight, d_bias, d if need[3] else None, None, None


def dense(x, weight, bias=None, *, act="none", residual=None):
    """linear as a differentiable function of x, the weight, the bias and the residual. The products are taken in x's type:
    a weight of another type is cast for them, and its gradient is summed and returned in its own (float32 for a float32
    weight, whatever x is). Pre-activations are kept where a gradient of the first three may be asked for: not under
    no_grad, nor for the residual alone."""
    keep = torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias))
    return _Dense.apply(x, weight, bias, residual, act, keep)


class Dense(torch.nn.Module):
    """A layer with its parameters: act(x @ weight + bias) + residual. The products are taken in x's type, for which
    parameters of another are cast; their gradients come in their own (dense)."""

    def __init__(self, width, out, bias=True, act="none", gain=1.0, device=None, dtype=torch.float32):
        super().__init__()
        w = torch.randn(width, out, device=device, dtype=torch.float32) * gain * width ** -0.5
        self.weight = torch.nn.Parameter(w.to(dtype))
        self.bias = torch.nn.Parameter(torch.zeros(out, device=device, dtype=dtype)) if bias else None
        self.act = act

    def forward(self, x, residual=None):
        b = self.bias
        if b is not None and b.dtype is not torch.float32:
            b = b.to(x.dtype)
        return dense(x, self.weight, b, act=self.act, residual=residual)


class _TokenLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, legal, kw):
        r = token_logp(logits, tokens, legal=legal, **kw)
        ctx.save_for_backward(logits, tokens, legal, r.stats)
        ctx.kw = kw
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (r.rank, r.top_logp, r.top_index) if t is not None))
        return r.logp, r.entropy, r.rank, r.top_logp, r.top_index

    @staticmethod
    @_first_only
    def backward(ctx, d_logp, d_entropy, *_):
        logits, tokens, legal, stats = ctx.saved_tensors
        one = [None if d is None else _upstream(d).contiguous() for d in (d_logp, d_entropy)]
        grad = token_logp_backward(*one, logits, tokens, stats, legal=legal, inv_temperature=ctx.kw["inv_temperature"])
        return grad, None, None, None


def token_logp_objective(logits, tokens, *, legal=None, inv_temperature=1.0, top=0):
    """token_logp whose logp and entropy are differentiable functions of the logits: (logp, entropy, rank, top_logp,
    top_index), the last three without gradients. The backward pass reads the logits again."""
    return _TokenLogp.apply(logits, tokens, legal, {"inv_temperature": inv_temperature, "top": top})


class Muon(torch.optim.Optimizer):
    """Momentum whose update's singular values are brought towards 1 (orthogonalise), for weights of two dimensions, or
    three (a stack of them). Weights of one shape and type are updated together; momentum is kept in float32. The step is lr max(1, out / in)^(1/2)
    for a weight [in, out]; weight_decay is decoupled. dtype: the type that the update is computed to."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, dtype=torch.bfloat16):
        super().__init__(params, {"lr": lr, "momentum": momentum, "nesterov": nesterov, "weight_decay": weight_decay,
                                  "steps": steps, "dtype": dtype})
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() not in (2, 3):
                    _fail(f"a weight of shape {tuple(p.shape)}: two or three dimensions are expected")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # which casts what it loads to the weight's type
        order = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(order, (p for group in self.param_groups for p in group["params"])):
            if "momentum" in self.state.get(p, ()):
                held = state_dict["state"][i]["momentum"]
                self.state[p]["momentum"] = held.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            same = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                held, g = state["momentum"], p.grad.float()
                held.mul_(group["momentum"]).add_(g)
                update = g.add(held, alpha=group["momentum"]) if group["nesterov"] else held
                same.setdefault((p.shape, p.dtype, p.device), []).append((p, update))
            for (shape, _, _), pairs in same.items():
                updates = torch.stack([u for _, u in pairs]) if len(pairs) > 1 else pairs[0][1].contiguous()
                each = orthogonalise(updates.reshape(-1, *shape[-2:]), steps=group["steps"], dtype=group["dtype"],
                                     scale=max(1.0, shape[-1] / shape[-2]) ** 0.5)
                for (p, _), o in zip(pairs, each.reshape(len(pairs), *shape).unbind(0)):
                    if group["weight_decay"]:
                        p.mul_(1 - group["lr"] * group["weight_decay"])
                    p.add_(o, alpha=-group["lr"])
        return loss
