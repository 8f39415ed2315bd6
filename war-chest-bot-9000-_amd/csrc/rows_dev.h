// Rows of logits held in registers: loads, softmax statistics over the threads that hold a row, and gradients from
// them. What the policy and preference losses (policy_dev.h) and the token log-probabilities (logp_dev.h) share.
#pragma once

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
// times infinity would be NaN). A row whose sum is NaN (a NaN or +infinity among
// its logits) is NaN, but 0 where its logits' own powers are, as in illegal
// columns, which are -infinity here.
struct Slope {
    float m, log_s, my, log_sy, base, slope, toward, hit;

    __device__ __forceinline__ Slope(const RowGrad& g, float go)
        : m(g.m), log_s(g.log_s), my(g.klc != 0.f ? g.my : 0.f), log_sy(g.klc != 0.f ? g.log_sy : 0.f),
          base(go * (g.ent * g.h - (g.klc != 0.f ? g.klc * g.kl : 0.f) - g.coef)),
          slope(go * (g.ent + g.klc) * LN2), toward(go * g.klc * LN2), hit(go * g.coef) {
        const bool spoiled = log_s != log_s;
        base = spoiled ? log_s : base;
        m = spoiled ? 0.f : m;
        log_s = spoiled ? 0.f : log_s;
    }
    // Whether PLAIN is right where p is 0, too.
    __device__ __forceinline__ bool finite() const { return base - base == 0.f; }

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

inline Rate rate_of(float inv_temp) {
    const double exact = (double)inv_temp * 1.4426950408889634074;
    const float rate = (float)exact;
    // log s of the caller's rate = log s of this one - (rate / exact - 1) * the mean of z
    return {rate, (float)((double)rate / exact - 1.0), inv_temp};
}

}  // namespace
}  // namespace learn
}  // namespace wc
