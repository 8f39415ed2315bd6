/*
 * wc_learn.h — C ABI of the training operators beside the wave executor: what a
 * trainer of the policy or value network runs on the solver's results. The
 * reference's trainer composes these from its framework's own operators; here
 * each is one call on device-resident buffers, queued on the caller's stream.
 *
 * Every entry takes a description and a stream (a hipStream_t, NULL: the
 * device's default stream), checks the description on the host, queues its
 * kernels and returns at once: WC_OK, or a negative code with the reason in
 * wc_last_error(), and then nothing was queued. Nothing is allocated: a call
 * that needs scratch names its size in *_workspace, and the caller's workspace
 * (256-byte aligned) may be reused as soon as the queue has passed the call.
 * Results do not depend on timing: no sum is taken in an order that changes
 * from run to run.
 *
 * Matrices are row-major with unit column stride; row strides are in elements,
 * may be 0 (one row broadcast) for inputs and at least the width for outputs.
 * No alignment beyond the element's own is needed. `bytes` is the size of the
 * structure as the caller compiled it; another size is refused.
 */
#ifndef WC_LEARN_H
#define WC_LEARN_H

#include <stddef.h>
#include <stdint.h>

#include "wc_wave.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of the matrices. */
#define WC_DTYPE_F32 0
#define WC_DTYPE_F16 1
#define WC_DTYPE_BF16 2

/* ------------------------------------------------------------ policy loss
 * Clipped policy loss with a KL term and an entropy bonus, over rows of logits:
 *   x_j = inv_temperature * logits_j (legal j only), logp = x - log sum exp x, p = exp logp
 *   r = exp(logp_a - behaviour_logp), a the row's action
 *   row loss = -min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl_coef KL - entropy_coef H
 *   loss = sum of weight * row loss
 * KL is expm1(d) - d with d = ref_logp - logp_a where ref_logp is given, or the
 * whole sum of p (logp - logq), q the softmax of inv_temperature * ref_logits
 * over the same legal columns, where ref_logits is given (not both), or 0. It is
 * infinite where q leaves out a column that p does not, or the action has no
 * probability, and so is the loss then; with a kl_coef of 0 it has no part in loss
 * and gradient, whatever it is.
 *
 * A row is left out (its outputs and gradient are 0, its logits are not read
 * or have no effect) when its weight is 0, its action is outside [0, vocab) or
 * not legal, or no legal logit is above -infinity. Illegal columns may hold
 * anything, NaN included; their gradient is 0. */
typedef struct wc_policy_args {
    uint64_t bytes;
    int32_t device, dtype;      /* WC_DTYPE_* of logits, ref_logits and grad */
    int64_t rows, vocab;
    const void* logits;
    int64_t logits_stride;
    const uint8_t* legal;       /* rows x vocab, nonzero = legal; NULL: all */
    int64_t legal_stride;
    const void* ref_logits;     /* rows x vocab, or NULL */
    int64_t ref_stride;
    const void* actions;        /* rows, of index_bits */
    const float* behaviour_logp; /* rows */
    const float* advantages;    /* rows */
    const float* weights;       /* rows; NULL: 1 / rows each */
    const float* ref_logp;      /* rows, or NULL */
    const float* grad_out;      /* one float: what arrives at the loss; NULL: 1 */
    float inv_temperature, clip_low, clip_high, kl_coef, entropy_coef;
    int32_t index_bits;         /* 32 or 64 */
    float* loss;                /* 1 */
    float* logp;                /* rows each: logp_a, KL, H */
    float* kl;
    float* entropy;
    void* grad;                 /* rows x vocab, d loss / d logits * grad_out; may be logits itself; NULL: none */
    int64_t grad_stride;
    void* workspace;
    uint64_t workspace_bytes;
} wc_policy_args;
int wc_policy_workspace(const wc_policy_args* a, uint64_t* bytes);
int wc_policy_loss(const wc_policy_args* a, void* stream);

/* -------------------------------------------------------- preference loss
 * Paired log ratios over ragged sequences of rows: sequence s is the rows
 * offsets[s] .. offsets[s+1]; pair i prefers sequence 2i to sequence 2i + 1.
 *   ratio_s = sum over its rows of weight (logp_token - ref_logp), with
 *             `average` divided by the sum of its weights (0 where that is 0)
 *   h = ratio_2i - ratio_2i+1, z = beta h
 *   logistic: -(1 - smoothing) log sigma(z) - smoothing log sigma(-z)
 *   squared:  (h - 1 / (2 beta))^2
 *   hinge:    max(0, 1 - z)
 *   loss = mean over pairs
 * A row is left out (no effect, gradient 0) when its weight is 0, its token is
 * outside [0, vocab), or no logit is above -infinity; a row in no sequence has
 * no effect and gradient 0 either.
 * Offsets are clamped to 0 .. rows; a sequence whose end is not after its
 * start is empty. Sequences must not overlap. */
#define WC_PREFERENCE_LOGISTIC 0
#define WC_PREFERENCE_SQUARED 1
#define WC_PREFERENCE_HINGE 2
typedef struct wc_preference_args {
    uint64_t bytes;
    int32_t device, dtype;
    int64_t rows, vocab, pairs;
    const void* logits;
    int64_t logits_stride;
    const void* tokens;         /* rows, of index_bits */
    const void* offsets;        /* 2 pairs + 1, of index_bits */
    const float* ref_logp;      /* rows */
    const float* weights;       /* rows; NULL: 1 */
    const float* grad_out;      /* one float; NULL: 1 */
    float inv_temperature, beta, smoothing;
    int32_t kind, average, index_bits;
    float* loss;                /* 1 */
    float* margins;             /* pairs: z */
    float* ratios;              /* 2 pairs */
    float* logp;                /* rows: logp_token, 0 for a row left out */
    void* grad;                 /* rows x vocab; may be logits itself; NULL: none */
    int64_t grad_stride;
    void* workspace;
    uint64_t workspace_bytes;
} wc_preference_args;
int wc_preference_workspace(const wc_preference_args* a, uint64_t* bytes);
int wc_preference_loss(const wc_preference_args* a, void* stream);

/* ----------------------------------------------------------- residual norm
 * A block's output normed, gated, scaled and added to the residual stream, and
 * the norm before the next block:
 *   n = norm(block) * post_gain + post_bias
 *   stream' = stream + scale * act(gate) * n
 *   out = norm(stream') * pre_gain + pre_bias
 * norm: WC_NORM_LAYER subtracts the row's mean and divides by the square root
 * of its variance + eps; WC_NORM_RMS divides by the root of the mean square +
 * eps. Statistics, sums and everything between the inputs and the outputs are
 * float32. The second norm sees stream' before it is rounded to its type.
 * gate: one row (gate_stride 0: a learned vector) or a row each; NULL: 1.
 * width at most WC_NORM_MAX_WIDTH. */
#define WC_NORM_RMS 0
#define WC_NORM_LAYER 1
#define WC_GATE_NONE 0
#define WC_GATE_SIGMOID 1
#define WC_GATE_TANH 2
#define WC_NORM_MAX_WIDTH 16384
typedef struct wc_norm_args {
    uint64_t bytes;
    int32_t device, dtype;      /* of every matrix (a gate with a row each among them) */
    int32_t param_dtype, pad;   /* of the gains, the biases and a gate vector */
    int64_t rows, width;
    const void* block;
    int64_t block_stride;
    const void* stream;
    int64_t stream_stride;
    const void* post_gain;      /* width; NULL: 1 */
    const void* post_bias;      /* width; NULL: 0 */
    const void* gate;
    int64_t gate_stride;
    const void* pre_gain;
    const void* pre_bias;
    float scale, eps;
    int32_t norm, gate_act;
    void* new_stream;           /* rows x width; may be stream itself */
    int64_t new_stream_stride;
    void* out;                  /* rows x width */
    int64_t out_stride;
    float* stats;               /* rows x 4: mean and 1/root of the block, then of stream'; NULL: not kept */
} wc_norm_args;
int wc_residual_norm(const wc_norm_args* a, void* stream);

/* Its gradients, from the forward's inputs and stats. d_stream (what arrives
 * at stream'; NULL: 0) and d_out (at out; NULL: 0). Gradients of parameters
 * are float32, summed over the rows; each may be NULL (not wanted). A gate
 * with a row each gets its gradient in its own type, rows x width. */
typedef struct wc_norm_back_args {
    uint64_t bytes;
    int32_t device, dtype;
    int32_t param_dtype, pad0;
    int64_t rows, width;
    const void* block;
    int64_t block_stride;
    const void* stream;
    int64_t stream_stride;
    const void* post_gain;
    const void* post_bias;
    const void* gate;
    int64_t gate_stride;
    const void* pre_gain;
    float scale;
    int32_t norm, gate_act, pad;
    const float* stats;
    const void* d_out;
    int64_t d_out_stride;
    const void* d_new_stream;
    int64_t d_new_stream_stride;
    void* d_block;              /* rows x width */
    int64_t d_block_stride;
    void* d_stream;             /* rows x width; may be d_new_stream itself */
    int64_t d_stream_stride;
    float* d_post_gain;         /* width each */
    float* d_post_bias;
    float* d_pre_gain;
    float* d_pre_bias;
    void* d_gate;               /* gate_stride 0: width floats; else rows x width of dtype */
    int64_t d_gate_stride;
    void* workspace;
    uint64_t workspace_bytes;
} wc_norm_back_args;
int wc_residual_norm_workspace(const wc_norm_back_args* a, uint64_t* bytes);
int wc_residual_norm_backward(const wc_norm_back_args* a, void* stream);

/* ---------------------------------------------- activations kept in 8 bits
 * A row's channels in groups of WC_CKPT_GROUP; each group holds integers
 * q in -127 .. 127 and one exponent byte e: the values q * 2^(e - 127). The
 * power is the least that holds the group's largest magnitude, and q is
 * x / 2^(e - 127) rounded to nearest, ties to even; so writing and reading are
 * exact steps, and a value is off by at most 1/127 of its group's largest. The least
 * power is 2^-126 (e = 1). A group with an infinity or a NaN is held as e =
 * 255 and reads back as NaN throughout. A value that rounded past the largest
 * of the type it is read in (f16's from 65024, the others' from 3.376e38) is
 * read as that largest. */
#define WC_CKPT_GROUP 32
#define WC_ACT_NONE 0
#define WC_ACT_RELU 1
#define WC_ACT_GELU 2 /* x/2 (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))), the v5 network's */
#define WC_ACT_SILU 3
typedef struct wc_ckpt_args {
    uint64_t bytes;
    int32_t device, dtype;      /* of x, y and grad */
    int64_t rows, width;
    int32_t act, pad;
    int8_t* q;                  /* rows x width */
    int64_t q_stride;
    uint8_t* exps;              /* rows x ceil(width / 32) */
    int64_t exps_stride;
    const void* x;              /* write: the values to keep; act backward: the gradient at act's output */
    int64_t x_stride;
    void* y;                    /* write: act(x), NULL: not wanted; read: the kept values; act backward: the gradient at act's input */
    int64_t y_stride;
} wc_ckpt_args;
/* q, exps from x, and y = act(x) of the unrounded x. */
int wc_ckpt_write(const wc_ckpt_args* a, void* stream);
/* y = act(what q, exps stand for). */
int wc_ckpt_read(const wc_ckpt_args* a, void* stream);
/* y = x * act'(what q, exps stand for). y may be x itself. */
int wc_ckpt_act_backward(const wc_ckpt_args* a, void* stream);

/* Weight gradient from the 8-bit operand: weight[i][j] = sum over rows of
 * act(kept[r][i]) * grad[r][j] (width x out, the layout of wc_net_desc's W_1),
 * bias[j] = sum over rows of grad[r][j]. Products on the matrix cores in grad's
 * 16-bit type with float32 sums: kept values are exact in bf16, and in f16
 * within f16's range (larger ones are taken as its largest, steps under 2^-24
 * are rounded); a GELU or SiLU recomputed from them is rounded to that type, for a
 * float32 weight too: less than what the 8 bits left out. float32 grad is taken with
 * WC_ACT_NONE and WC_ACT_RELU, as three bf16 parts whose products are exact (what of
 * a part is under 2^-133 is lost: grad's last bits below 2^-110). */
typedef struct wc_ckpt_weight_args {
    uint64_t bytes;
    int32_t device, dtype;      /* of grad */
    int64_t rows, width, out;
    int32_t act, weight_dtype;  /* weight: WC_DTYPE_F32 or grad's */
    const int8_t* q;
    int64_t q_stride;
    const uint8_t* exps;
    int64_t exps_stride;
    const void* grad;           /* rows x out */
    int64_t grad_stride;
    void* weight;               /* width x out */
    int64_t weight_stride;
    float* bias;                /* out; NULL: not wanted */
    void* workspace;
    uint64_t workspace_bytes;
} wc_ckpt_weight_args;
int wc_ckpt_weight_workspace(const wc_ckpt_weight_args* a, uint64_t* bytes);
int wc_ckpt_weight_grad(const wc_ckpt_weight_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* WC_LEARN_H */
