// Policy and preference losses over rows of logits (include/wc_learn.h), for one
// element type: policy_f32.hip, policy_f16.hip and policy_bf16.hip build one each.
//
// A row's softmax needs its maximum, then sums over all of it, then, for the
// gradient, every logit again. Memory bounds it: 4 bytes moved per 16-bit
// logit against some 20 operations. So a row is read once and held in
// registers, as it came, from its load to its gradient's store (k_rows), by as
// few threads as hold it: part of a wavefront for a few heads, one wavefront up
// to 8 KB, a workgroup up to 256 KB. Longer rows are read twice (k_row_parts,
// k_row_grads), and so are the preference loss's, whose gradient waits for
// whole sequences.
//
// On one MI355X, where a large copy moves 5.09 TB/s (read and write):
// - 4,096 x 65,536 bf16, a quarter of the rows left out: 203 us, 4.6 TB/s (two
//   passes, 366 us; 512 threads a row with half the registers each, which
//   spilled, 260);
// - 49,371 x 567 float32 with a reference distribution and legal columns: 97 us,
//   3.5 TB/s. Vector arithmetic issues in half of the cycles, and the wavefronts
//   wait for memory two thirds of their time, at 3.2 wavefronts a SIMD; five would
//   spill (159 us), and workgroups that stay and take row after row were slower (114 us);
// - 800,000 x 12 float32 with a reference and legal columns: 78 us, 2.0 TB/s: of the
//   8 lanes that a row has three load, and all of them add and take logarithms;
// - 64 x 22: 4 us, one launch.
#pragma once

#include <algorithm>

#include "learn.h"
#include "learn_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

// ------------------------------------------------------------------- softmax

// Powers are of 2: z = (x - m) rate, rate = inv_temp log2(e). The difference to
// the maximum comes first, so that a row at a mask's lowest value keeps its
// differences, and the products are never contracted into another's sum.
// The float32 rate is off by `off` of itself, a temperature that differs by
// 3e-8; log-probabilities are given for the caller's by the first-order term.
struct Rate {
    float rate, off, inv_temp;
};

// A softmax's statistics over part of a row: the maximum logit, the sums of
// e = 2^z, of e z (for the entropy) and of e ((x - m) - (y - my)) (for the KL
// sum: each row's differences to its own maximum, so that a constant added to
// either row, or a row at a mask's lowest value, changes nothing), and y's
// maximum and sum.
struct Part {
    float m, s, t, d, my, sy;
};

// The statistics of two parts together. A part without a finite logit has
// m = -infinity and adds nothing but the NaN that it may have found.
__device__ __forceinline__ Part join(const Part& a, const Part& b, float rate) {
    Part r;
    r.m = fmaxf(a.m, b.m);
    r.my = fmaxf(a.my, b.my);
    const bool ha = a.m != -INFINITY, hb = b.m != -INFINITY;
    const float da = ha ? (a.m - r.m) * rate : 0.f, db = hb ? (b.m - r.m) * rate : 0.f;
    const float fa = power(da), fb = power(db);
    r.s = a.s * fa + b.s * fb;
    r.t = fa * (a.t + a.s * fmaxf(da, -300.f)) + fb * (b.t + b.s * fmaxf(db, -300.f));
    // the KL sums' differences are to other maxima now; a part that weighs nothing adds
    // nothing, whatever the distance
    r.d = (fa > 0.f && a.s > 0.f ? fa * (a.d + a.s * ((a.m - r.m) - (a.my - r.my))) : 0.f) +
          (fb > 0.f && b.s > 0.f ? fb * (b.d + b.s * ((b.m - r.m) - (b.my - r.my))) : 0.f);
    r.sy = (a.my != -INFINITY ? a.sy * power((a.my - r.my) * rate) : a.sy) +
           (b.my != -INFINITY ? b.sy * power((b.my - r.my) * rate) : b.sy);
    return r;
}

// Logits per 16-byte load.
template <class T>
constexpr int EACH = 16 / sizeof(T);

template <class T>
using Raw = typename VecN<T, EACH<T>>::type;

// What the rows are.
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
    Rate rate;
    int bits;
    float even;  // the weight of a row where none are given
};

// What a row starts with. Its logits are read if `read`, and count if `on`:
// the legal byte of the action is another load away, so the logits' go first.
struct Head {
    int64_t a;
    float w;
    bool read, on;

    template <class T>
    __device__ __forceinline__ Head(const Rows<T>& in, int64_t r, bool there) {
        a = -1;
        w = 0.f;
        if (there) {
            w = in.weights ? in.weights[r] : in.even;
            a = index_at(in.actions, in.bits, r);
        }
        read = w != 0.f && a >= 0 && a < in.vocab;
        on = read && (!in.legal || in.legal[r * in.legal_stride + a]);
    }
};

// Part of a row as G threads hold it: NV whole 16-byte loads each (-infinity
// where the row has none), and the columns past the last whole load, one a
// thread. Wide accesses at one place and single ones at another keep both
// short: a check per column in each of the NV would cost more registers than
// the logits.
template <class T, int G, int NV>
struct Held {
    static constexpr int E = EACH<T>;
    Raw<T> v[NV];
    T one;

    // Columns 0 .. n of `row`; legal (may be null) alike.
    __device__ __forceinline__ void load(const T* row, const uint8_t* legal, int n, int lane) {
        typedef uint8_t Bytes __attribute__((ext_vector_type(E), aligned(1)));
        const int whole = n / E;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = lane + k * G;
            if (c < whole) {
                v[k] = *(const Raw<T>*)(row + c * E);
            } else {
#pragma unroll
                for (int i = 0; i < E; i++) v[k][i] = (T)-INFINITY;
            }
        }
        const int last = whole * E + lane;
        one = last < n && (!legal || legal[last]) ? row[last] : (T)-INFINITY;
        if (legal) {
#pragma unroll
            for (int k = 0; k < NV; k++) {
                const int c = lane + k * G;
                if (c < whole) {
                    const Bytes on = *(const Bytes*)(legal + c * E);
#pragma unroll
                    for (int i = 0; i < E; i++) v[k][i] = on[i] ? v[k][i] : (T)-INFINITY;
                }
            }
        }
    }
    __device__ __forceinline__ void none() {
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < E; i++) v[k][i] = (T)-INFINITY;
        one = (T)-INFINITY;
    }
    // Takes away what the compiler knows of the logits, so that each pass over
    // them converts them anew: kept as floats from one pass to the next they
    // would not fit the registers.
    __device__ __forceinline__ void forget() {
        typedef uint32_t Words __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < NV; k++) {
            Words w = __builtin_bit_cast(Words, v[k]);
            asm volatile("" : "+v"(w));
            v[k] = __builtin_bit_cast(Raw<T>, w);
        }
    }
};

// Sums and maxima over the G threads that hold a row, the same bits in each: a
// butterfly in a wavefront, then the wavefronts' values in order through LDS.
// The slots alternate, so one barrier each is enough: a slot is written again
// only after a barrier that every reader of its last use has passed.
template <int G>
struct Group {
    static constexpr int WAVES = G > 64 ? G / 64 : 1;
    typedef float4 Slots[2][WAVES];
    Slots& lds;
    int slot = 0;

    template <int N, bool MAX>
    __device__ __forceinline__ void all(float (&v)[N]) {
#pragma unroll
        for (int mask = (G < 64 ? G : 64) / 2; mask; mask >>= 1)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float o = __shfl_xor(v[i], mask);
                v[i] = MAX ? fmaxf(v[i], o) : v[i] + o;
            }
        if constexpr (G > 64) {
            static_assert(N <= 4, "a slot holds four");
            float* mine = (float*)&lds[slot][threadIdx.x >> 6];
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < N; i++) mine[i] = v[i];
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = MAX ? -INFINITY : 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float* o = (const float*)&lds[slot][w];
#pragma unroll
                for (int i = 0; i < N; i++) v[i] = MAX ? fmaxf(v[i], o[i]) : v[i] + o[i];
            }
            slot ^= 1;
        }
    }
};

// Adds one logit to the sums; m and my are the maxima.
template <bool FULL>
__device__ __forceinline__ void count(Part& p, float x, float y, float m, float my, float rate) {
    const float z = (x - m) * rate, e = power(z);
    p.s += e;
    p.t += e * fmaxf(z, -300.f);  // e is 0 there, and 0 * -infinity would be NaN
    if (FULL) {
        const float v = y - my;
        p.d += e > 0.f ? e * ((x - m) - v) : 0.f;
        p.sy += power(v * rate);
    }
}

// The statistics of the logits that G threads hold. Everything is relative to
// the common maximum, so one exponential per logit is enough.
template <class T, int G, int NV, bool FULL>
__device__ __forceinline__ Part held_stats(Held<T, G, NV>& x, Held<T, G, FULL ? NV : 1>& y, float rate,
                                           Group<G>& group) {
    constexpr int E = EACH<T>;
    Part p = {(float)x.one, 0.f, 0.f, 0.f, FULL ? (float)y.one : -INFINITY, 0.f};
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            p.m = fmaxf(p.m, (float)x.v[k][i]);
            if (FULL) p.my = fmaxf(p.my, (float)y.v[k][i]);
        }
        __builtin_amdgcn_sched_barrier(0);  // one load's values converted at a time
    }
    if constexpr (FULL) {
        float top[2] = {p.m, p.my};
        group.template all<2, true>(top);
        p.m = top[0], p.my = top[1];
    } else {
        float top[1] = {p.m};
        group.template all<1, true>(top);
        p.m = top[0];
    }
    x.forget();
    if (FULL) y.forget();
    // a row of nothing but -infinity: 0 keeps its differences -infinity
    const float m = p.m == -INFINITY ? 0.f : p.m, my = p.my == -INFINITY ? 0.f : p.my;
    count<FULL>(p, (float)x.one, (float)y.one, m, my, rate);
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int i = 0; i < E; i++)
            count<FULL>(p, (float)x.v[k][i], FULL ? (float)y.v[FULL ? k : 0][i] : 0.f, m, my, rate);
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (FULL) {
        float sum[4] = {p.s, p.t, p.d, p.sy};
        group.template all<4, false>(sum);
        p.s = sum[0], p.t = sum[1], p.d = sum[2], p.sy = sum[3];
    } else {
        float sum[2] = {p.s, p.t};
        group.template all<2, false>(sum);
        p.s = sum[0], p.t = sum[1];
    }
    x.forget();
    if (FULL) y.forget();
    return p;
}

// Whether a row has anything to count: a logit above -infinity, or a NaN.
__device__ __forceinline__ bool counts(const Part& p) { return p.m != -INFINITY || p.s != 0.f; }

// What a row's gradient needs: coef ([j = a] - p) + ent p (logp + h) + klc p (logp - logq - kl),
// m and my the maxima, log_s and log_sy the sums' logarithms to base 2.
struct RowGrad {
    float m, log_s, my, log_sy, coef, ent, h, klc, kl;
    int32_t on;

    // Without a coefficient (clipped, left out, in no sequence) the gradient is 0 whatever the logits.
    __device__ __forceinline__ bool any() const { return on && (coef != 0.f || ent != 0.f || klc != 0.f); }
};

constexpr float LN2 = 0.6931471805599453f;

// A row's gradient as a function of a logit: p (base + slope logp - toward logq),
// logarithms to base 2; PLAIN without the two. Where p is 0 the gradient is (0
// times infinity would be NaN).
struct Slope {
    float m, log_s, my, log_sy, base, slope, toward, hit;

    __device__ __forceinline__ Slope(const RowGrad& g, float go)
        : m(g.m), log_s(g.log_s), my(g.klc != 0.f ? g.my : 0.f), log_sy(g.klc != 0.f ? g.log_sy : 0.f),
          base(go * (g.ent * g.h - (g.klc != 0.f ? g.klc * g.kl : 0.f) - g.coef)),
          slope(go * (g.ent + g.klc) * LN2), toward(go * g.klc * LN2), hit(go * g.coef) {}

    template <bool FULL, bool PLAIN>
    __device__ __forceinline__ float at(float x, float y, float rate) const {
        const float lp = (x - m) * rate - log_s, p = power(lp);
        if (PLAIN) return p * base;
        float d = base + slope * lp;
        // finite: a reference of no probability has no effect where the KL has no coefficient
        if (FULL) d -= toward * fmaxf((y - my) * rate - log_sy, -3.4028234663852886e38f);
        return p == 0.f ? 0.f : p * d;
    }
};

// The gradient of the n columns that G threads hold; `a` the action's column
// or -1, whose gradient has the coefficient more: the thread that holds it
// writes it once again.
template <class T, int G, int NV, bool FULL, bool PLAIN>
__device__ __forceinline__ void put_grad(T* row, int n, int lane, const Held<T, G, NV>& x,
                                         const Held<T, G, FULL ? NV : 1>& y, const Slope& g, float rate, int a) {
    constexpr int E = EACH<T>;
    const int whole = n / E, last = whole * E + lane;
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = lane + k * G;
        if (c < whole) {
            Raw<T> o;
#pragma unroll
            for (int i = 0; i < E; i++)
                o[i] = (T)g.at<FULL, PLAIN>((float)x.v[k][i], FULL ? (float)y.v[FULL ? k : 0][i] : 0.f, rate);
            *(Raw<T>*)(row + c * E) = o;
            if (a >= c * E && a < c * E + E) {
                float xa = 0.f, ya = 0.f;
#pragma unroll
                for (int i = 0; i < E; i++) {
                    if (c * E + i != a) continue;
                    xa = (float)x.v[k][i];
                    if (FULL) ya = (float)y.v[FULL ? k : 0][i];
                }
                row[a] = (T)(g.at<FULL, PLAIN>(xa, ya, rate) + g.hit);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (last < n) {
        const float d = g.at<FULL, PLAIN>((float)x.one, (float)y.one, rate);
        row[last] = (T)(last == a ? d + g.hit : d);
    }
}

template <class T, int G, int NV>
__device__ __forceinline__ void put_zero(T* row, int n, int lane) {
    constexpr int E = EACH<T>;
    const int whole = n / E, last = whole * E + lane;
#pragma unroll
    for (int k = 0; k < NV; k++)
        if (lane + k * G < whole) *(Raw<T>*)(row + (lane + k * G) * E) = Raw<T>{};
    if (last < n) row[last] = (T)0.f;
}

// A counted row's loss, outputs and gradient coefficients from its statistics.
// The loss's own terms are 64-bit: rows' losses cancel in their sum, and the
// clip's bounds rounded to 32 bits would shift all clipped rows alike.
struct PolicyRow {
    const float *behaviour_logp, *advantages, *ref_logp;
    float clip_low, clip_high, kl_coef, entropy_coef;
    bool full;
    float *logp, *kl, *entropy;
    double* losses;
    float* loss;

    // What a row adds to its logits, loaded before they are waited for.
    struct Terms {
        float behaviour, advantage, ref, xa;
    };
    template <class T>
    __device__ __forceinline__ Terms terms(const Rows<T>& in, int64_t r, const Head& h) const {
        return {behaviour_logp[r], advantages[r], ref_logp ? ref_logp[r] : 0.f, (float)in.x[r * in.x_stride + h.a]};
    }

    __device__ __forceinline__ double finish(const Rate& k, const Part& p, const Terms& in, float w, RowGrad* g,
                                             float3* out) const {
        const float log2_s = __log2f(p.s), log_s = logf(p.s), over = 1.f / p.s;
        const float mean = p.t * LN2 * over, fix = k.off * mean;  // mean of z, and what the rate's error adds to log s
        const float za = (in.xa - p.m) * k.inv_temp + fix, lp = za - log_s, h = (log_s - fix) - mean;
        // e^(z_a - behaviour) / s: without the logarithm's rounding and the difference's
        const double adv = in.advantage, ratio = expf(za - in.behaviour) * over;
        const double open = ratio * adv, held = fmin(fmax(ratio, 1.0 - clip_low), 1.0 + clip_high) * adv;
        const bool first = !(open > held);  // a NaN takes this side, and shows
        float slope = first ? -(float)open : 0.f, kl = 0.f, log2_sy = 0.f;
        if (ref_logp) {
            const float d = in.ref - lp, e = expm1f(d);
            kl = e == INFINITY ? e : e - d;  // an action of no probability: infinite
            if (kl_coef != 0.f) slope -= kl_coef * e;
        }
        if (full) {
            log2_sy = __log2f(p.sy);
            kl = p.d * over * k.rate * LN2 - (log_s - logf(p.sy));
        }
        *out = make_float3(lp, kl, h);
        *g = {p.m, log2_s, p.my, log2_sy, w * slope, w * entropy_coef, h, full ? w * kl_coef : 0.f, kl, 1};
        // an infinite KL has no effect where its coefficient is 0 (here and in Slope: a choice for each
        // term; one that several terms hang on cost 10 registers, and 10% of 800,000 x 12 float32)
        return w * ((double)kl_coef * (kl_coef != 0.f ? kl : 0.f) - (first ? open : held) - (double)entropy_coef * h);
    }
};

// A token's log-probability, and the statistics for its gradient.
__device__ __forceinline__ float token(const Rate& k, const Part& p, float xa, RowGrad* g) {
    const float log_s = logf(p.s);
    g->m = p.m;
    g->log_s = __log2f(p.s);
    g->on = 1;
    return (xa - p.m) * k.inv_temp + k.off * (p.t * LN2 / p.s) - log_s;
}

// ------------------------------------------------- rows that registers hold

// Rows of up to a wavefront are launched with 256 threads, or all in one
// workgroup. Four wavefronts a SIMD, three where a thread holds 64 registers of
// logits, two where it holds 128: few threads with much of a row each leave
// more of the registers to logits than many with little.
template <int G>
constexpr int group_block() {
    return G > 64 ? G : 1024;
}
template <int LOADS>
constexpr int group_waves() {
    return LOADS > 16 ? 2 : LOADS == 16 ? 3 : 4;
}

// A row on G threads, NV 16-byte loads of logits (FULL: and of the reference's)
// each. TOKEN: log-probabilities and statistics only, for the preference loss.
template <class T, int G, int NV, bool FULL, bool TOKEN>
__global__ __launch_bounds__(group_block<G>(), (group_waves<NV * (FULL ? 2 : 1)>())) void k_rows(Rows<T> in, PolicyRow row, int64_t rows, RowGrad* grads,
                                                              const float* grad_out, T* grad, int64_t grad_stride) {
    __shared__ typename Group<G>::Slots slots;
    __shared__ double total[1024 / (G > 64 ? 1024 : G)];
    Group<G> group{slots};
    const int lane = threadIdx.x % G, per = G > 64 ? 1 : blockDim.x / G, n = (int)in.vocab;
    const float go = (grad_out ? *grad_out : 1.f) * in.rate.inv_temp;
    double sum = 0.0;
    for (int64_t r0 = int64_t(blockIdx.x) * per; r0 < rows; r0 += int64_t(gridDim.x) * per) {
        const int64_t r = r0 + (G > 64 ? 0 : threadIdx.x / G);
        const Head head(in, r, r < rows);
        Held<T, G, NV> x;
        Held<T, G, FULL ? NV : 1> y;
        y.one = (T)0.f;
        PolicyRow::Terms terms = {};
        if (head.read) {
            const uint8_t* legal = in.legal ? in.legal + r * in.legal_stride : nullptr;
            if constexpr (TOKEN) terms.xa = (float)in.x[r * in.x_stride + head.a];
            else terms = row.terms(in, r, head);
            x.load(in.x + r * in.x_stride, legal, n, lane);
            if constexpr (FULL) y.load(in.y + r * in.y_stride, legal, n, lane);
            // every wavefront reads the action's logit, and one writes its gradient, perhaps there
            if (G > 64) settle(terms.xa);
        } else {
            x.none();
            if constexpr (FULL) y.none();
        }
        RowGrad g;
        g.m = g.log_s = g.my = g.log_sy = g.coef = g.ent = g.h = g.klc = g.kl = 0.f;
        g.on = 0;
        float3 out = make_float3(0.f, 0.f, 0.f);
        double loss = 0.0;
        if (G <= 64 || head.read) {  // a workgroup's row is left out as one
            const Part p = held_stats<T, G, NV, FULL>(x, y, in.rate.rate, group);
            if (head.on && counts(p)) {
                if constexpr (TOKEN) out.x = token(in.rate, p, terms.xa, &g);
                else loss = row.finish(in.rate, p, terms, head.w, &g, &out);
            }
        }
        if (r < rows) {
            if (lane == 0) {
                row.logp[r] = out.x;
                if constexpr (TOKEN) {
                    grads[r] = g;
                } else {
                    row.kl[r] = out.y;
                    row.entropy[r] = out.z;
                    sum += loss;
                }
            }
            if (!TOKEN && grad) {
                T* to = grad + r * grad_stride;
                if (!g.any())
                    put_zero<T, G, NV>(to, n, lane);
                else if (!FULL && g.ent == 0.f)
                    put_grad<T, G, NV, FULL, true>(to, n, lane, x, y, Slope(g, go), in.rate.rate, (int)head.a);
                else
                    put_grad<T, G, NV, FULL, false>(to, n, lane, x, y, Slope(g, go), in.rate.rate, (int)head.a);
            }
        }
    }
    if constexpr (!TOKEN) {  // the workgroup's losses, in an order that does not change
        if constexpr (G <= 64) {
            if (lane == 0) total[threadIdx.x / G] = sum;
            __syncthreads();
            if (threadIdx.x >= 64) return;
            sum = 0.0;
            for (int k = threadIdx.x; k < per; k += 64) sum += total[k];
            for (int mask = 32; mask; mask >>= 1) sum += __shfl_xor(sum, mask);
        }
        if (threadIdx.x == 0) {
            if (gridDim.x == 1) *row.loss = (float)sum;
            else row.losses[blockIdx.x] = sum;
        }
    }
}

// -------------------------------------------------------------- longer rows

constexpr int BLOCK = 256;
constexpr int64_t CHUNK = 8192;  // columns per workgroup
template <class T>
constexpr int CHUNK_LOADS = CHUNK / (BLOCK * EACH<T>);

// The statistics of one chunk of one row: workgroup r * splits + chunk. 2,048 x
// 131,072 float32: 200 us, 5.4 TB/s; the gradient then reads and writes for 364 (5.9
// TB/s), and 10 go to the rows' ends between.
template <class T, bool FULL>
__global__ __launch_bounds__(BLOCK) void k_row_parts(Rows<T> in, int64_t tiles, int splits, Part* parts) {
    constexpr int NV = CHUNK_LOADS<T>;
    __shared__ typename Group<BLOCK>::Slots slots;
    Group<BLOCK> group{slots};
    for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
        const int64_t r = t / splits, c0 = (t - r * splits) * CHUNK;
        if (!Head(in, r, true).read) continue;
        const uint8_t* legal = in.legal ? in.legal + r * in.legal_stride + c0 : nullptr;
        const int n = (int)min(CHUNK, in.vocab - c0);
        Held<T, BLOCK, NV> x;
        Held<T, BLOCK, FULL ? NV : 1> y;
        y.one = (T)0.f;
        x.load(in.x + r * in.x_stride + c0, legal, n, threadIdx.x);
        if constexpr (FULL) y.load(in.y + r * in.y_stride + c0, legal, n, threadIdx.x);
        const Part p = held_stats<T, BLOCK, NV, FULL>(x, y, in.rate.rate, group);
        if (threadIdx.x == 0) parts[t] = p;
    }
}

// A row's parts joined, its outputs and coefficients: one thread per row.
template <class T, bool TOKEN>
__global__ void k_row_ends(Rows<T> in, PolicyRow row, int64_t rows, int splits, const Part* parts, RowGrad* grads) {
    const int64_t r = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    if (r >= rows) return;
    const Head head(in, r, true);
    Part p = {-INFINITY, 0.f, 0.f, 0.f, -INFINITY, 0.f};
    if (head.on)
        for (int k = 0; k < splits; k++) p = join(p, parts[r * splits + k], in.rate.rate);
    RowGrad g = {};
    float3 out = make_float3(0.f, 0.f, 0.f);
    double loss = 0.0;
    if (counts(p)) {
        if (TOKEN) out.x = token(in.rate, p, (float)in.x[r * in.x_stride + head.a], &g);
        else loss = row.finish(in.rate, p, row.terms(in, r, head), head.w, &g, &out);
    }
    row.logp[r] = out.x;
    grads[r] = g;
    if (!TOKEN) {
        row.kl[r] = out.y;
        row.entropy[r] = out.z;
        row.losses[r] = loss;
    }
}

// The sum of n losses in a fixed order, by one workgroup.
struct LossSum {
    const double* losses;
    int64_t n;
    double scale;
    float* out;
};
template <int THREADS>
__device__ __forceinline__ void sum_losses(const LossSum& l) {
    __shared__ double lds[THREADS / 64];
    const double* v = l.losses;
    double s = 0;
    int64_t i = threadIdx.x;
    for (; i + 3 * THREADS < l.n; i += 4 * THREADS)
        s += (v[i] + v[i + THREADS]) + (v[i + 2 * THREADS] + v[i + 3 * THREADS]);
    for (; i < l.n; i += THREADS) s += v[i];
    for (int mask = 32; mask; mask >>= 1) s += __shfl_xor(s, mask);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 64; w++) s += lds[w];
        *l.out = (float)(s * l.scale);
    }
}
__global__ __launch_bounds__(1024) void k_sum(LossSum l) { sum_losses<1024>(l); }

// The gradient from the rows' coefficients, a second read of the logits. The
// last rows go first: they are what the pass before left in the caches. The
// last workgroup adds the losses beside the others. 4,608 x 65,536 bf16, 30% of
// the rows left out: 151 us for 1.03 GB, 6.8 TB/s, more than memory gives; the
// preference loss there 277 us in all, of which the first read takes 112. A
// workgroup takes one row's chunk whatever its length: 97,754 rows of 12 or of 64
// float32 take 190 us, all of it launching and latency (their bytes 2.5 and 10.5).
template <class T, bool FULL>
__global__ __launch_bounds__(BLOCK) void k_row_grads(Rows<T> in, int64_t tiles, int splits, const RowGrad* grads,
                                                     const float* grad_out, T* out, int64_t out_stride,
                                                     LossSum losses) {
    constexpr int NV = CHUNK_LOADS<T>;
    if (blockIdx.x == gridDim.x - 1) return sum_losses<BLOCK>(losses);
    const float go = (grad_out ? *grad_out : 1.f) * in.rate.inv_temp;
    for (int64_t i = blockIdx.x; i < tiles; i += gridDim.x - 1) {
        const int64_t t = tiles - 1 - i, r = t / splits, c0 = (t - r * splits) * CHUNK;
        const RowGrad g = grads[r];
        T* to = out + r * out_stride + c0;
        const int n = (int)min(CHUNK, in.vocab - c0);
        if (!g.any()) {
            put_zero<T, BLOCK, NV>(to, n, threadIdx.x);
            continue;
        }
        const int64_t a = index_at(in.actions, in.bits, r) - c0;
        const uint8_t* legal = in.legal ? in.legal + r * in.legal_stride + c0 : nullptr;
        Held<T, BLOCK, NV> x;
        Held<T, BLOCK, FULL ? NV : 1> y;
        y.one = (T)0.f;
        x.load(in.x + r * in.x_stride + c0, legal, n, threadIdx.x);
        if constexpr (FULL) y.load(in.y + r * in.y_stride + c0, legal, n, threadIdx.x);
        const int at = a >= 0 && a < n ? (int)a : -1;
        if (!FULL && g.ent == 0.f)
            put_grad<T, BLOCK, NV, FULL, true>(to, n, threadIdx.x, x, y, Slope(g, go), in.rate.rate, at);
        else
            put_grad<T, BLOCK, NV, FULL, false>(to, n, threadIdx.x, x, y, Slope(g, go), in.rate.rate, at);
    }
}

// ------------------------------------------------------------------ launches

inline Rate rate_of(float inv_temp) {
    const double exact = (double)inv_temp * 1.4426950408889634074;
    const float rate = (float)exact;
    // log s of the caller's rate = log s of this one - (rate / exact - 1) * the mean of z
    return {rate, (float)((double)rate / exact - 1.0), inv_temp};
}

template <class T>
Rows<T> rows_of(const wc_policy_args& a) {
    return {(const T*)a.logits, a.logits_stride, a.legal, a.legal_stride, (const T*)a.ref_logits, a.ref_stride,
            a.actions, a.weights, a.vocab, rate_of(a.inv_temperature), a.index_bits,
            1.f / (float)std::max<int64_t>(a.rows, 1)};
}

template <class T>
Rows<T> rows_of(const wc_preference_args& a) {
    return {(const T*)a.logits, a.logits_stride, nullptr, 0, nullptr, 0, a.tokens, a.weights, a.vocab,
            rate_of(a.inv_temperature), a.index_bits, 1.f};
}

inline int splits_of(int64_t vocab) { return (int)((vocab + CHUNK - 1) / CHUNK); }

inline uint32_t tile_grid(int64_t tiles) { return (uint32_t)std::min<int64_t>(tiles, 1 << 22); }

// Whether k_rows holds a row: up to 128 registers per thread of 512.
inline bool holds(int dtype, int64_t vocab, bool full) {
    return vocab * (dtype == WC_DTYPE_F32 ? 4 : 2) * (full ? 2 : 1) <= 256 << 10;
}

// Rows that one workgroup of up to 1,024 holds at once go to one, which then
// sums their losses itself: 64 x 22 float32 in one launch and without scratch
// 18 us a call; in workgroups of 256, with scratch and a second launch, 21.
inline bool one_group(int64_t rows, int lanes) { return rows == 1 || (lanes <= 64 && rows * lanes <= 1024); }

// Lanes that hold a row of n 16-byte loads, while one wavefront does.
inline int lanes_of(int64_t n) { return n <= 64 ? 8 : n <= 128 ? 16 : n <= 256 ? 32 : n <= 512 ? 64 : 256; }

// Returns the workgroups: as many losses.
template <class T, int G, int NV, bool FULL, bool TOKEN>
int64_t rows_at(const Rows<T>& in, const PolicyRow& row, int64_t rows, RowGrad* grads, const float* grad_out, T* grad,
                int64_t grad_stride, hipStream_t s) {
    const int block = G > 64 ? G : one_group(rows, G) ? (int)((rows * G + 63) / 64 * 64) : 256;
    const int64_t per = block / (G > 64 ? block : G), grid = std::min<int64_t>((rows + per - 1) / per, 1 << 22);
    k_rows<T, G, NV, FULL, TOKEN><<<dim3((uint32_t)grid), block, 0, s>>>(in, row, rows, grads, grad_out, grad,
                                                                         grad_stride);
    return grid;
}

// The fewest threads that hold a row in at most eight loads each, and with the
// least left empty: what a wavefront does once a row (the sums' butterflies,
// the logarithms) it then does for several rows at once. 567 float32 columns
// with a reference: 110 us on 32 lanes of five loads, 147 on 64 lanes of three.
template <class T, bool FULL, bool TOKEN>
int64_t rows_held(const Rows<T>& in, const PolicyRow& row, int64_t rows, RowGrad* grads, const float* go, T* grad,
                  int64_t gs, hipStream_t s) {
    const int64_t n = in.vocab / EACH<T>;
    if (n <= 8) return rows_at<T, 8, 1, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 16) return rows_at<T, 8, 2, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 24) return rows_at<T, 8, 3, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 32) return rows_at<T, 8, 4, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 48) return rows_at<T, 8, 6, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 64) return rows_at<T, 8, 8, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 80) return rows_at<T, 16, 5, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 96) return rows_at<T, 16, 6, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 128) return rows_at<T, 16, 8, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 160) return rows_at<T, 32, 5, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 192) return rows_at<T, 32, 6, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 256) return rows_at<T, 32, 8, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 320) return rows_at<T, 64, 5, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 384) return rows_at<T, 64, 6, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 512) return rows_at<T, 64, 8, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 1024) return rows_at<T, 256, 4, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if (n <= 2048) return rows_at<T, 256, 8, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    if constexpr (TOKEN) {  // no gradient to write: more threads, with less each, load faster (65,536 bf16: 112 us, 134)
        if (n <= 4096) return rows_at<T, 512, 8, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
        if (n <= 8192) return rows_at<T, 512, 16, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
        return rows_at<T, 512, 32, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    } else if constexpr (FULL) {
        if (n <= 4096) return rows_at<T, 256, 16, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
        return rows_at<T, 512, 16, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    } else {
        if (n <= 4096) return rows_at<T, 256, 16, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
        if (n <= 8192) return rows_at<T, 256, 32, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
        return rows_at<T, 512, 32, FULL, TOKEN>(in, row, rows, grads, go, grad, gs, s);
    }
}

template <class T, bool FULL>
void policy(const wc_policy_args& a, hipStream_t s) {
    const Rows<T> in = rows_of<T>(a);
    uint8_t* w = (uint8_t*)a.workspace;
    const PolicyRow row = {a.behaviour_logp, a.advantages, a.ref_logp, a.clip_low, a.clip_high, a.kl_coef,
                           a.entropy_coef, FULL, a.logp, a.kl, a.entropy, (double*)w, a.loss};
    int64_t losses = a.rows;
    if (a.rows && holds(a.dtype, a.vocab, FULL)) {
        losses = rows_held<T, FULL, false>(in, row, a.rows, nullptr, a.grad_out, (T*)a.grad, a.grad_stride, s);
        if (losses == 1) return;
    } else if (a.rows) {
        const int splits = splits_of(a.vocab);
        const int64_t tiles = a.rows * splits;
        RowGrad* grads = (RowGrad*)(w += pad256(size_t(a.rows) * sizeof(double)));
        Part* parts = (Part*)(w += pad256(size_t(a.rows) * sizeof(RowGrad)));
        k_row_parts<T, FULL><<<tile_grid(tiles), BLOCK, 0, s>>>(in, tiles, splits, parts);
        k_row_ends<T, false><<<dim3((uint32_t)((a.rows + 63) / 64)), 64, 0, s>>>(in, row, a.rows, splits, parts, grads);
        if (a.grad) {
            k_row_grads<T, FULL><<<tile_grid(tiles) + 1, BLOCK, 0, s>>>(in, tiles, splits, grads, a.grad_out, (T*)a.grad,
                                                                        a.grad_stride, {row.losses, losses, 1.0, a.loss});
            return;
        }
    }
    k_sum<<<1, 1024, 0, s>>>({row.losses, losses, 1.0, a.loss});
}

// ---------------------------------------------------------------- preference

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
// every row of both. 6 to 9 us of dependent loads; the pairs side by side, in
// launches whose threads 32 bits can count.
constexpr int64_t MOST_PAIR_BLOCKS = 1 << 22;
__global__ __launch_bounds__(BLOCK) void k_pairs(Pairs p, int64_t first, const float* logp, RowGrad* grads,
                                                 double* losses, float* margins, float* ratios) {
    __shared__ double lds[4][BLOCK / 64];
    const int64_t i = first + blockIdx.x;
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
        const double e = exp(-fabs(z)), tail = log1p(e);
        // an infinite margin, and a share of 0 of its infinite term
        const double far = z > 0.0 ? p.smoothing : 1.0 - p.smoothing;
        loss = tail + (far > 0.0 ? far * fabs(z) : 0.0);
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
void preference(const wc_preference_args& a, hipStream_t s) {
    const Rows<T> in = rows_of<T>(a);
    const int splits = splits_of(a.vocab);
    const int64_t tiles = a.rows * splits;
    uint8_t* w = (uint8_t*)a.workspace;
    RowGrad* grads = (RowGrad*)w;
    double* losses = (double*)(w += pad256(size_t(a.rows) * sizeof(RowGrad)));
    PolicyRow row = {};
    row.logp = a.logp;
    if (a.rows && holds(a.dtype, a.vocab, false)) {
        rows_held<T, false, true>(in, row, a.rows, grads, nullptr, nullptr, 0, s);
    } else if (a.rows) {
        Part* parts = (Part*)(w += pad256(size_t(a.pairs) * sizeof(double)));
        k_row_parts<T, false><<<tile_grid(tiles), BLOCK, 0, s>>>(in, tiles, splits, parts);
        k_row_ends<T, true><<<dim3((uint32_t)((a.rows + 63) / 64)), 64, 0, s>>>(in, row, a.rows, splits, parts, grads);
    }
    const Pairs p = {a.offsets, a.ref_logp, a.weights, a.rows, a.pairs, a.beta, a.smoothing, a.kind, a.average,
                     a.index_bits};
    for (int64_t i = 0; i < a.pairs; i += MOST_PAIR_BLOCKS)
        k_pairs<<<dim3((uint32_t)std::min(a.pairs - i, MOST_PAIR_BLOCKS)), BLOCK, 0, s>>>(p, i, a.logp, grads, losses,
                                                                                          a.margins, a.ratios);
    const LossSum sum = {losses, a.pairs, a.pairs ? 1.0 / (double)a.pairs : 0.0, a.loss};
    if (a.grad && a.rows)
        k_row_grads<T, false><<<tile_grid(tiles) + 1, BLOCK, 0, s>>>(in, tiles, splits, grads, a.grad_out, (T*)a.grad,
                                                                     a.grad_stride, sum);
    else
        k_sum<<<1, 1024, 0, s>>>(sum);
}

template <class T>
void policy_of(const wc_policy_args& a, hipStream_t s) {
    if (a.ref_logits) policy<T, true>(a, s);
    else policy<T, false>(a, s);
}

}  // namespace
}  // namespace learn
}  // namespace wc
