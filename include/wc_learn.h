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
 * An output that may be one of the inputs itself starts where that starts and has
 * its row stride; no other output may overlap an input.
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

/* ------------------------------------------------------------- linear layer
 * y = act(x W + bias) + residual, one product with its epilogue: sums, bias,
 * activation and residual in float32, rounded once to y's type. W is width x
 * out (WC_WEIGHT_IN_OUT) or out x width (WC_WEIGHT_OUT_IN, a row an output).
 * pre, where given, gets x W + bias in float32, for the backward pass.
 * 16-bit matrices: products on the matrix cores with float32 sums. float32:
 * small ones as they are, larger ones as three bf16 parts an element and six
 * products of parts (what is left out is below 2^-25 of a product, and of a part
 * what is under 2^-133: an element's last bits below 2^-110); there an
 * infinite element's row or column of the result is not finite, and may be NaN
 * where its product alone would be infinite.
 * rows below 2^31, width and out at most 2^20. */
#define WC_WEIGHT_IN_OUT 0
#define WC_WEIGHT_OUT_IN 1
typedef struct wc_linear_args {
    uint64_t bytes;
    int32_t device, dtype;      /* of every matrix */
    int32_t bias_dtype, weight_layout; /* bias: float32 or the matrices' */
    int64_t rows, width, out;
    const void* x;              /* rows x width */
    int64_t x_stride;
    const void* weight;
    int64_t weight_stride;
    const void* bias;           /* out; NULL: 0 */
    const void* residual;       /* rows x out; NULL: 0 */
    int64_t residual_stride;
    int32_t act, pad;           /* WC_ACT_* */
    float* pre;                 /* rows x out; NULL: not kept */
    int64_t pre_stride;
    void* y;                    /* rows x out; may be residual itself */
    int64_t y_stride;
    void* workspace;
    uint64_t workspace_bytes;
} wc_linear_args;
int wc_linear_workspace(const wc_linear_args* a, uint64_t* bytes);
int wc_linear(const wc_linear_args* a, void* stream);

/* Its gradients: d_pre = d_out act'(pre), d_x = d_pre W^T, d_weight = x^T d_pre
 * in the weight's layout, d_bias = the column sums of d_pre, each NULL where not
 * wanted (the residual's gradient is d_out). d_pre is rounded to the matrices'
 * type for its products, as it would be between two operators, which is as much
 * again as d_x and d_weight's own rounding (in bf16 2.3e-3 of their norm in all,
 * 1.7e-3 without; float32 matrices have none); d_bias is summed before that, in
 * float32. A d_pre that float32 holds is no reason for an
 * infinity, where it passes f16's largest (a slope is up to 1.13) either. */
typedef struct wc_linear_back_args {
    uint64_t bytes;
    int32_t device, dtype;
    int32_t weight_layout, act;
    int32_t grad_dtype, pad;    /* of d_weight: float32 or the matrices' */
    int64_t rows, width, out;
    const void* d_out;          /* rows x out */
    int64_t d_out_stride;
    const float* pre;           /* rows x out; with WC_ACT_NONE not read */
    int64_t pre_stride;
    const void* x;              /* read for d_weight */
    int64_t x_stride;
    const void* weight;         /* read for d_x */
    int64_t weight_stride;
    void* d_x;                  /* rows x width */
    int64_t d_x_stride;
    void* d_weight;
    int64_t d_weight_stride;
    float* d_bias;              /* out */
    void* workspace;
    uint64_t workspace_bytes;
} wc_linear_back_args;
int wc_linear_backward_workspace(const wc_linear_back_args* a, uint64_t* bytes);
int wc_linear_backward(const wc_linear_back_args* a, void* stream);

/* ------------------------------------------------------------ orthogonalise
 * A matrix's singular values brought towards 1 (a weight's update, before it is
 * applied): X = update / (Frobenius norm + eps), then `steps` times
 *   A = X X^T, X = a X + (b A + c A A) X
 * (the transposed form where rows > width), and out = scale X. `batch` matrices
 * of one shape. X is held in 22 bits an element (in steps of 2^-34, so that one
 * below 2^-13 has fewer), A and its polynomial too, but for a bf16 result of more
 * than 128 rows and columns in 11 (off by about as much as that result's
 * rounding); sums are float32, the norm's float64.
 * X, A and B = b A + c A A are held times 2^10 in f16: an element of any of them
 * that passes 63 may make the result infinite or NaN. None does while every
 * singular value s of the matrix that a step starts from has s^2 and |b s^2 + c s^4|
 * below 63 (s below 7.9), and the result's, before scale, are below 63: with
 * the usual coefficients (3.4445, -4.775, 2.0315) s stays below 1.3, B below 2.9. */
typedef struct wc_orthogonalise_args {
    uint64_t bytes;
    int32_t device, dtype;      /* of update */
    int32_t out_dtype, steps;   /* steps: 1 .. 64 */
    int64_t batch, rows, width; /* batch at most 65535, rows and width 2^20 */
    const void* update;
    int64_t update_stride, update_batch; /* elements from row to row, from matrix to matrix */
    void* out;                  /* may be update itself: one matrix, or of its type and strides */
    int64_t out_stride, out_batch;
    float a, b, c, eps, scale;
    int32_t pad;
    void* workspace;
    uint64_t workspace_bytes;
} wc_orthogonalise_args;
int wc_orthogonalise_workspace(const wc_orthogonalise_args* a, uint64_t* bytes);
int wc_orthogonalise(const wc_orthogonalise_args* a, void* stream);

/* ------------------------------------------------- token log-probabilities
 * Of rows of logits, over their legal columns:
 *   z = inv_temperature * logits, logp = z - log sum exp z, p = exp logp
 *   logp of the row's token, its rank (how many columns have a larger logit, or
 *   an equal one and a lower index; 0: the likeliest), the entropy -sum p logp,
 *   and the `top` likeliest columns in that order with their log-probabilities.
 * A row is left out (logp and entropy 0, rank -1, its logits not read) when its
 * token is outside [0, vocab) or no legal logit is above -infinity. A token that
 * is not legal, or whose logit is -infinity, has logp -infinity, and its rank
 * counts all columns of a lower index beside those above -infinity. Alternatives
 * are columns above -infinity: where there are fewer than `top`, and in a row
 * that is left out, the others are column -1 with -infinity. Illegal columns may
 * hold anything. A legal NaN or +infinity makes a row's values NaN (a NaN is no
 * alternative). tokens NULL: every row counts; logp and rank are not written. */
#define WC_TOP_MAX 64
typedef struct wc_logp_args {
    uint64_t bytes;
    int32_t device, dtype;
    int64_t rows, vocab;
    const void* logits;
    int64_t logits_stride;
    const uint8_t* legal;       /* rows x vocab, nonzero = legal; NULL: all */
    int64_t legal_stride;
    const void* tokens;         /* rows, of index_bits; NULL: none */
    float inv_temperature;
    int32_t index_bits, top, pad; /* top: 0 .. WC_TOP_MAX */
    float* logp;                /* rows each */
    float* entropy;
    int32_t* rank;
    float* top_logp;            /* rows x top */
    int32_t* top_index;
    float* stats;               /* rows x 4, for the backward pass; NULL: not kept */
    void* workspace;
    uint64_t workspace_bytes;
} wc_logp_args;
int wc_token_logp_workspace(const wc_logp_args* a, uint64_t* bytes);
int wc_token_logp(const wc_logp_args* a, void* stream);

/* The gradient at the logits from what arrives at logp and at the entropy (each
 * may be NULL: 0): inv_temperature (d_logp ([j = token] - p_j) - d_entropy p_j
 * (logp_j + H)), 0 in illegal columns and in rows that were left out. */
typedef struct wc_logp_back_args {
    uint64_t bytes;
    int32_t device, dtype;
    int64_t rows, vocab;
    const void* logits;
    int64_t logits_stride;
    const uint8_t* legal;
    int64_t legal_stride;
    const void* tokens;
    float inv_temperature;
    int32_t index_bits;
    const float* stats;
    const float* d_logp;        /* rows */
    const float* d_entropy;     /* rows */
    void* grad;                 /* rows x vocab; may be logits itself */
    int64_t grad_stride;
} wc_logp_back_args;
int wc_token_logp_backward(const wc_logp_back_args* a, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* WC_LEARN_H */
