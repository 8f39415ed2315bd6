// Policy and preference losses over rows of logits (include/wc_learn.h).
#include <algorithm>

#include "learn.h"
#include "learn_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

constexpr int BLOCK = 256;

// A softmax's running statistics over part of a row: the maximum, the sum of
// e^(x - m), the sum of e^(x - m) (x - m) (for the entropy) and of
// e^(x - m) (x - y) (for the KL sum), and y's maximum and sum.
struct Part {
    float m, s, t, d, my, sy;
};

__device__ __forceinline__ Part none() { return {-INFINITY, 0.f, 0.f, 0.f, -INFINITY, 0.f}; }

// The statistics of two parts together. A part without a finite logit has
// m = -infinity and adds nothing (its differences would be NaN).
__device__ __forceinline__ Part join(const Part& a, const Part& b) {
    Part r;
    r.m = fmaxf(a.m, b.m);
    r.my = fmaxf(a.my, b.my);
    const float da = a.m - r.m, db = b.m - r.m;
    const bool ha = a.m != -INFINITY, hb = b.m != -INFINITY;
    const float fa = ha ? fast_exp(da) : 0.f, fb = hb ? fast_exp(db) : 0.f;
    r.s = a.s * fa + b.s * fb;
    r.t = (ha ? fa * (a.t + a.s * da) : 0.f) + (hb ? fb * (b.t + b.s * db) : 0.f);
    r.d = a.d * fa + b.d * fb;
    r.sy = (a.my != -INFINITY ? a.sy * fast_exp(a.my - r.my) : 0.f) +
           (b.my != -INFINITY ? b.sy * fast_exp(b.my - r.my) : 0.f);
    return r;
}

__device__ __forceinline__ Part shuffle(const Part& a, int mask) {
    return {__shfl_xor(a.m, mask), __shfl_xor(a.s, mask), __shfl_xor(a.t, mask),
            __shfl_xor(a.d, mask), __shfl_xor(a.my, mask), __shfl_xor(a.sy, mask)};
}

// A logit times the inverse temperature, rounded once and the same everywhere:
// contracted into a later difference, the product of a row's maximum would
// differ from itself by its rounding, which for a mask of the type's lowest
// value is 1e30.
__device__ __forceinline__ float scaled(float x, float inv_temp) {
#pragma clang fp contract(off)
    return x * inv_temp;
}

// What one row needs of its logits, and where they are.
template <class T>
struct Rows {
    const T* x;
    int64_t x_stride;
    const uint8_t* legal;
    int64_t legal_stride;
    const T* y;
    int64_t y_stride;
    const void* actions;
    const float* weights;
    int64_t vocab;
    float inv_temp;
    int bits;

    // The row's action, or -1 for a row that is left out before its logits are read.
    __device__ __forceinline__ int64_t action(int64_t r) const {
        if (weights && weights[r] == 0.f) return -1;
        const int64_t a = index_at(actions, bits, r);
        if (a < 0 || a >= vocab) return -1;
        if (legal && !legal[r * legal_stride + a]) return -1;
        return a;
    }

    // Up to eight logits from column c: illegal and missing ones are -infinity.
    __device__ __forceinline__ void get(int64_t r, int64_t c, int n, float (&v)[8], float (&u)[8]) const {
        load_n(x + r * x_stride + c, n, -INFINITY, v);
        if (y) load_n(y + r * y_stride + c, n, -INFINITY, u);
        bool on[8];
#pragma unroll
        for (int i = 0; i < 8; i++) on[i] = i < n && (!legal || legal[r * legal_stride + c + i]);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = on[i] ? scaled(v[i], inv_temp) : -INFINITY;
            u[i] = y ? (on[i] ? scaled(u[i], inv_temp) : -INFINITY) : 0.f;
        }
    }
};

__device__ __forceinline__ void add8(Part& p, const float (&v)[8], const float (&u)[8], bool has_y) {
    Part q = none();
#pragma unroll
    for (int i = 0; i < 8; i++) q.m = fmaxf(q.m, v[i]);
    if (q.m == -INFINITY && !has_y) {
        // nothing here, unless a NaN, which the maximum passes over
        for (int i = 0; i < 8; i++) q.s += v[i] == -INFINITY ? 0.f : v[i];
        p.s += q.s;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const bool in = v[i] != -INFINITY;
        const float z = v[i] - q.m, e = in ? fast_exp(z) : 0.f;
        q.s += e;
        q.t += in ? e * z : 0.f;
        q.d += in ? e * (v[i] - u[i]) : 0.f;
    }
    if (has_y) {
#pragma unroll
        for (int i = 0; i < 8; i++) q.my = fmaxf(q.my, u[i]);
#pragma unroll
        for (int i = 0; i < 8; i++) q.sy += u[i] != -INFINITY ? fast_exp(u[i] - q.my) : 0.f;
    }
    p = join(p, q);
}

// One row's part [chunk * blockIdx.y ..) of its statistics.
template <class T>
__global__ __launch_bounds__(BLOCK) void k_row_parts(Rows<T> in, int64_t rows, int64_t chunk, int splits, Part* parts) {
    __shared__ Part lds[BLOCK / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        if (in.action(r) < 0) continue;
        const int64_t lo = blockIdx.y * chunk, hi = min(lo + chunk, in.vocab);
        Part p = none();
        for (int64_t c = lo + 8 * threadIdx.x; c < hi; c += 8 * BLOCK) {
            float v[8], u[8];
            in.get(r, c, (int)min<int64_t>(8, hi - c), v, u);
            add8(p, v, u, in.y != nullptr);
        }
        for (int mask = 32; mask; mask >>= 1) p = join(p, shuffle(p, mask));
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = p;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < BLOCK / 64; w++) p = join(p, lds[w]);
            parts[r * splits + blockIdx.y] = p;
        }
        __syncthreads();
    }
}

// What a row's gradient needs: inv_temp * (coef ([j = a] - p) + ent p (logp + h) + klc p (logp - logq - kl)).
// The maximum and the sum's logarithm stay apart: together, a row at a mask's
// value would lose the second.
struct RowGrad {
    float m, log_s, my, log_sy, coef, ent, h, klc, kl;
    int32_t on;
};

// A counted row's loss, outputs and gradient coefficients from its statistics.
// The loss's own terms are 64-bit: rows' losses cancel in their sum, and the
// clip's bounds rounded to 32 bits would shift all clipped rows alike.
struct PolicyRow {
    const float *behaviour_logp, *advantages, *weights, *ref_logp;
    float clip_low, clip_high, kl_coef, entropy_coef, even;
    bool full;
    float *logp, *kl, *entropy;

    __device__ __forceinline__ double finish(int64_t r, const Part& p, float xa, RowGrad* g) const {
        const float log_s = logf(p.s), lp = (xa - p.m) - log_s, h = log_s - p.t / p.s;
        const float w = weights ? weights[r] : even;
        // e^(x_a - m - behaviour) / s: without the logarithm's rounding and the difference's
        const double adv = advantages[r], ratio = expf((xa - p.m) - behaviour_logp[r]) / p.s;
        const double open = ratio * adv, held = fmin(fmax(ratio, 1.0 - clip_low), 1.0 + clip_high) * adv;
        const bool first = !(open > held);  // a NaN takes this side, and shows
        float slope = first ? -(float)open : 0.f, k = 0.f;
        if (ref_logp) {
            const float off = ref_logp[r] - lp, e = expm1f(off);
            k = e - off;
            slope -= kl_coef * e;
        }
        if (full) k = p.d / p.s - (p.m - p.my) - (log_s - logf(p.sy));
        logp[r] = lp;
        kl[r] = k;
        entropy[r] = h;
        *g = {p.m, log_s, p.my, logf(p.sy), w * slope, w * entropy_coef, h, full ? w * kl_coef : 0.f, k, 1};
        return w * ((double)kl_coef * k - (first ? open : held) - (double)entropy_coef * h);
    }
};

template <class T>
__global__ void k_policy_rows(Rows<T> in, PolicyRow row, int64_t rows, int splits, const Part* parts, RowGrad* grads,
                              double* losses) {
    const int64_t r = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    const int64_t a = in.action(r);
    Part p = none();
    if (a >= 0)
        for (int k = 0; k < splits; k++) p = join(p, parts[r * splits + k]);
    RowGrad g = {};
    double loss = 0.0;
    if (p.m != -INFINITY || p.s != 0.f) {
        loss = row.finish(r, p, scaled((float)in.x[r * in.x_stride + a], in.inv_temp), &g);
    } else {
        row.logp[r] = row.kl[r] = row.entropy[r] = 0.f;
    }
    grads[r] = g;
    losses[r] = loss;
}

// The sum of n row losses in a fixed order, in 64 bits.
__global__ __launch_bounds__(1024) void k_sum(const double* v, int64_t n, double scale, float* out) {
    __shared__ double lds[16];
    double s = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += v[i];
    for (int mask = 32; mask; mask >>= 1) s += __shfl_xor(s, mask);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; w++) s += lds[w];
        *out = (float)(s * scale);
    }
}

template <class T>
__global__ __launch_bounds__(BLOCK) void k_row_grads(Rows<T> in, int64_t rows, int64_t chunk, const RowGrad* grads,
                                                     const float* grad_out, T* out, int64_t out_stride) {
    const float go = (grad_out ? *grad_out : 1.f) * in.inv_temp;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const RowGrad g = grads[r];
        // without a coefficient (clipped, left out, in no sequence) the gradient is 0 whatever the logits
        const bool on = g.on && (g.coef != 0.f || g.ent != 0.f || g.klc != 0.f);
        const int64_t a = on ? index_at(in.actions, in.bits, r) : -1;
        const int64_t lo = blockIdx.y * chunk, hi = min(lo + chunk, in.vocab);
        for (int64_t c = lo + 8 * threadIdx.x; c < hi; c += 8 * BLOCK) {
            const int n = (int)min<int64_t>(8, hi - c);
            float o[8] = {};
            if (on) {
                float v[8], u[8];
                in.get(r, c, n, v, u);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (v[i] == -INFINITY) continue;
                    const float lp = (v[i] - g.m) - g.log_s, p = fast_exp(lp);
                    float d = -g.coef;
                    if (g.ent != 0.f) d += g.ent * (lp + g.h);
                    if (g.klc != 0.f) d += g.klc * (lp - ((u[i] - g.my) - g.log_sy) - g.kl);
                    o[i] = go * (p * d + (c + i == a ? g.coef : 0.f));
                }
            }
            store_n(out + r * out_stride + c, n, o);
        }
    }
}

// Columns of one row go to workgroups in chunks of at least 4096, so that few
// rows still fill the device.
void split(int64_t rows, int64_t vocab, int cus, int64_t* chunk, int* splits) {
    const int64_t most = (vocab + 4095) / 4096, want = std::max<int64_t>(1, 8 * cus / std::max<int64_t>(rows, 1));
    const int64_t n = std::max<int64_t>(1, std::min(most, want));
    *chunk = ((vocab + n - 1) / n + 7) / 8 * 8;
    *splits = (int)((vocab + *chunk - 1) / *chunk);
}

template <class T>
Rows<T> rows_of(const wc_policy_args& a) {
    return {(const T*)a.logits, a.logits_stride, a.legal, a.legal_stride, (const T*)a.ref_logits, a.ref_stride,
            a.actions, a.weights, a.vocab, a.inv_temperature, a.index_bits};
}

template <class T>
Rows<T> rows_of(const wc_preference_args& a) {
    return {(const T*)a.logits, a.logits_stride, nullptr, 0, nullptr, 0, a.tokens, a.weights, a.vocab,
            a.inv_temperature, a.index_bits};
}

uint32_t grid_rows(int64_t rows) { return (uint32_t)std::min<int64_t>(rows, 1 << 20); }

template <class T>
void policy(const wc_policy_args& a, int cus, hipStream_t s) {
    int64_t chunk;
    int splits;
    split(a.rows, a.vocab, cus, &chunk, &splits);
    uint8_t* w = (uint8_t*)a.workspace;
    Part* parts = (Part*)w;
    RowGrad* grads = (RowGrad*)(w += pad256(size_t(a.rows) * splits * sizeof(Part)));
    double* losses = (double*)(w += pad256(size_t(a.rows) * sizeof(RowGrad)));
    const Rows<T> in = rows_of<T>(a);
    const PolicyRow row = {a.behaviour_logp, a.advantages, a.weights, a.ref_logp, a.clip_low, a.clip_high, a.kl_coef,
                           a.entropy_coef, 1.f / (float)std::max<int64_t>(a.rows, 1), a.ref_logits != nullptr, a.logp, a.kl, a.entropy};
    if (a.rows) {
        const dim3 grid(grid_rows(a.rows), splits);
        k_row_parts<T><<<grid, BLOCK, 0, s>>>(in, a.rows, chunk, splits, parts);
        k_policy_rows<T><<<dim3((a.rows + 63) / 64), 64, 0, s>>>(in, row, a.rows, splits, parts, grads, losses);
    }
    k_sum<<<1, 1024, 0, s>>>(losses, a.rows, 1.0, a.loss);
    if (a.grad && a.rows) {
        const dim3 grid(grid_rows(a.rows), splits);
        k_row_grads<T><<<grid, BLOCK, 0, s>>>(in, a.rows, chunk, grads, a.grad_out, (T*)a.grad, a.grad_stride);
    }
}

// -------------------------------------------------------------- preference

template <class T>
__global__ void k_token_rows(Rows<T> in, int64_t rows, int splits, const Part* parts, float* logp, RowGrad* grads) {
    const int64_t r = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    const int64_t a = in.action(r);
    Part p = none();
    if (a >= 0)
        for (int k = 0; k < splits; k++) p = join(p, parts[r * splits + k]);
    RowGrad g = {};
    float lp = 0.f;
    if (p.m != -INFINITY || p.s != 0.f) {
        const float log_s = logf(p.s);
        lp = (scaled((float)in.x[r * in.x_stride + a], in.inv_temp) - p.m) - log_s;
        g.m = p.m;
        g.log_s = log_s;
        g.on = 1;
    }
    logp[r] = lp;
    grads[r] = g;
}

struct Pairs {
    const void* offsets;
    const float *ref_logp, *weights;
    int64_t rows, pairs;
    float beta, smoothing;
    int kind, average, bits;
};

__device__ __forceinline__ int64_t clamp_row(int64_t x, int64_t rows) { return x < 0 ? 0 : x > rows ? rows : x; }

// One pair per workgroup: both sequences' ratios in 64-bit sums (long sums of
// differences that nearly cancel), the pair's loss, and the coefficient of
// every row of both.
__global__ __launch_bounds__(BLOCK) void k_pairs(Pairs p, const float* logp, RowGrad* grads, double* losses,
                                                 float* margins, float* ratios) {
    __shared__ double lds[4][BLOCK / 64];
    const int64_t i = blockIdx.x;
    int64_t lo[2], hi[2];
    double sum[4] = {};
    for (int k = 0; k < 2; k++) {
        lo[k] = clamp_row(index_at(p.offsets, p.bits, 2 * i + k), p.rows);
        hi[k] = clamp_row(index_at(p.offsets, p.bits, 2 * i + k + 1), p.rows);
        for (int64_t r = lo[k] + threadIdx.x; r < hi[k]; r += BLOCK) {
            if (!grads[r].on) continue;
            const float w = p.weights ? p.weights[r] : 1.f;
            sum[2 * k] += (double)w * ((double)logp[r] - p.ref_logp[r]);
            sum[2 * k + 1] += w;
        }
    }
    for (int q = 0; q < 4; q++) {
        for (int mask = 32; mask; mask >>= 1) sum[q] += __shfl_xor(sum[q], mask);
        if ((threadIdx.x & 63) == 0) lds[q][threadIdx.x >> 6] = sum[q];
    }
    __syncthreads();
    for (int q = 0; q < 4; q++) sum[q] = (lds[q][0] + lds[q][1]) + (lds[q][2] + lds[q][3]);
    double share[2], ratio[2];
    for (int k = 0; k < 2; k++) {
        share[k] = !p.average ? 1.0 : sum[2 * k + 1] != 0.0 ? 1.0 / sum[2 * k + 1] : 0.0;
        ratio[k] = sum[2 * k] * share[k];
    }
    const double h = ratio[0] - ratio[1], z = p.beta * h;
    double loss, d;
    if (p.kind == WC_PREFERENCE_LOGISTIC) {
        const double tail = log1p(exp(-fabs(z))), e = exp(-fabs(z));
        loss = tail + (1.0 - p.smoothing) * fmax(-z, 0.0) + p.smoothing * fmax(z, 0.0);
        d = p.beta * ((z >= 0 ? 1.0 / (1.0 + e) : e / (1.0 + e)) - (1.0 - p.smoothing));
        if (z != z) loss = z;
    } else if (p.kind == WC_PREFERENCE_SQUARED) {
        const double t = h - 0.5 / p.beta;
        loss = t * t;
        d = 2.0 * t;
    } else {
        loss = z < 1.0 ? 1.0 - z : 0.0;
        d = z < 1.0 ? -(double)p.beta : 0.0;
        if (z != z) loss = d = z;
    }
    d /= (double)p.pairs;
    for (int k = 0; k < 2; k++) {
        const float c = (float)((k ? -d : d) * share[k]);
        for (int64_t r = lo[k] + threadIdx.x; r < hi[k]; r += BLOCK)
            if (grads[r].on) grads[r].coef = c * (p.weights ? p.weights[r] : 1.f);
    }
    if (threadIdx.x == 0) {
        losses[i] = loss;
        margins[i] = (float)z;
        ratios[2 * i] = (float)ratio[0];
        ratios[2 * i + 1] = (float)ratio[1];
    }
}

template <class T>
void preference(const wc_preference_args& a, int cus, hipStream_t s) {
    int64_t chunk;
    int splits;
    split(a.rows, a.vocab, cus, &chunk, &splits);
    uint8_t* w = (uint8_t*)a.workspace;
    Part* parts = (Part*)w;
    RowGrad* grads = (RowGrad*)(w += pad256(size_t(a.rows) * splits * sizeof(Part)));
    double* losses = (double*)(w += pad256(size_t(a.rows) * sizeof(RowGrad)));
    const Rows<T> in = rows_of<T>(a);
    const Pairs p = {a.offsets, a.ref_logp, a.weights, a.rows, a.pairs, a.beta, a.smoothing, a.kind, a.average,
                     a.index_bits};
    if (a.rows) {
        k_row_parts<T><<<dim3(grid_rows(a.rows), splits), BLOCK, 0, s>>>(in, a.rows, chunk, splits, parts);
        k_token_rows<T><<<dim3((a.rows + 63) / 64), 64, 0, s>>>(in, a.rows, splits, parts, a.logp, grads);
    }
    if (a.pairs) k_pairs<<<dim3(a.pairs), BLOCK, 0, s>>>(p, a.logp, grads, losses, a.margins, a.ratios);
    k_sum<<<1, 1024, 0, s>>>(losses, a.pairs, a.pairs ? 1.0 / (double)a.pairs : 0.0, a.loss);
    if (a.grad && a.rows)
        k_row_grads<T><<<dim3(grid_rows(a.rows), splits), BLOCK, 0, s>>>(in, a.rows, chunk, grads, a.grad_out,
                                                                         (T*)a.grad, a.grad_stride);
}

}  // namespace

size_t policy_scratch(const wc_policy_args& a, int cus) {
    int64_t chunk;
    int splits;
    split(a.rows, a.vocab, cus, &chunk, &splits);
    return pad256(size_t(a.rows) * splits * sizeof(Part)) + pad256(size_t(a.rows) * sizeof(RowGrad)) +
           pad256(size_t(a.rows) * sizeof(double));
}

size_t preference_scratch(const wc_preference_args& a, int cus) {
    int64_t chunk;
    int splits;
    split(a.rows, a.vocab, cus, &chunk, &splits);
    return pad256(size_t(a.rows) * splits * sizeof(Part)) + pad256(size_t(a.rows) * sizeof(RowGrad)) +
           pad256(size_t(a.pairs) * sizeof(double));
}

void launch_policy(const wc_policy_args& a, int cus, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) policy<float>(a, cus, s);
    else if (a.dtype == WC_DTYPE_F16) policy<f16>(a, cus, s);
    else policy<bf16>(a, cus, s);
}

void launch_preference(const wc_preference_args& a, int cus, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) preference<float>(a, cus, s);
    else if (a.dtype == WC_DTYPE_F16) preference<f16>(a, cus, s);
    else preference<bf16>(a, cus, s);
}

}  // namespace learn
}  // namespace wc
