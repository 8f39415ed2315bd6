// Log-probabilities of given tokens, their rank, the entropy and the top alternatives of rows of logits, and the gradient
// (include/wc_learn.h), for one element type: logp_f32.hip, logp_f16.hip and logp_bf16.hip build one each.
//
//   z_j = inv_temperature x_j, logp_j = z_j - log sum exp z, H = -sum p logp
//   grad_j = inv_temperature (d_logp ([j = a] - p_j) - d_H p_j (logp_j + H))
//
// Rows are read once and held in registers (rows_dev.h): as few threads as hold a row, or a workgroup for each chunk of
// a long one, whose statistics and lists are joined by a second launch.
//
// 4,096 x 65,536 bf16 with the gradient: forward 138 us for the 403 MB of the rows that count (conversions, exponentials and
// comparisons bound it, not the 78 us of the memory). Backward, which reads these and writes 537 MB: 154 us after the forward
// pass, of which the last-level cache still holds a part, 185 after itself, 201 after a gigabyte of other memory, 4.7 TB/s; a
// copy of all the logits takes 220 there. 49,371 x 567 float32 with masks and five alternatives: 44 us, of which the memory's
// are 25; 410 vector instructions a row, and what a row's reductions wait for.
#pragma once

#include <algorithm>

#include "rows_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

constexpr int LOGP_BLOCK = 256;

// A logit and its column; of equal ones the lower column is the better.
struct Pick {
    float v;
    int i;
};
constexpr Pick NO_PICK = {-INFINITY, 0x7FFFFFFF};

__device__ __forceinline__ bool better(const Pick& a, const Pick& b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

// Reductions over G lanes of a wavefront, the same bits in each: in a row of 16 lanes by the cross-lane operand of the
// instruction itself (halves are alike when a mirror exchanges them), then rows and halves exchanged.
template <int CTRL>
__device__ __forceinline__ float lane_moved(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
template <int G, class F>
__device__ __forceinline__ float over_lanes(float v, F&& f) {
    static_assert(G >= 8 && G <= 64, "part of a wavefront");
    v = f(v, lane_moved<0xB1>(v));   // lanes 1 0 3 2 of four
    v = f(v, lane_moved<0x4E>(v));   // lanes 2 3 0 1
    v = f(v, lane_moved<0x141>(v));  // eight mirrored
    if constexpr (G >= 16) v = f(v, lane_moved<0x140>(v));  // sixteen mirrored
    if constexpr (G >= 32) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    if constexpr (G >= 64) {
        const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    return v;
}
struct Larger {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Added {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// The same over a row's G threads. Slots alternate: one is written again only after a barrier that every reader of its
// last use has passed.
template <int G>
struct Team {
    static constexpr int WAVES = G > 64 ? G / 64 : 1, LANES = G > 64 ? 64 : G;
    typedef float4 Slots[2][WAVES];
    Slots& lds;
    int slot = 0;

    template <int N, class F>
    __device__ __forceinline__ void all(float (&v)[N], F&& f) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = over_lanes<LANES>(v[i], f);
        if constexpr (G > 64) {
            static_assert(N <= 4, "a slot holds four");
            float* mine = (float*)&lds[slot][threadIdx.x >> 6];
            if ((threadIdx.x & 63) == 0) {
#pragma unroll
                for (int i = 0; i < N; i++) mine[i] = v[i];
            }
            __syncthreads();
            const float* first = (const float*)&lds[slot][0];
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = first[i];
#pragma unroll
            for (int w = 1; w < WAVES; w++) {
                const float* o = (const float*)&lds[slot][w];
#pragma unroll
                for (int i = 0; i < N; i++) v[i] = f(v[i], o[i]);
            }
            slot ^= 1;
        }
    }
    // The best of the threads' picks.
    __device__ __forceinline__ Pick best(Pick p) {
#pragma unroll
        for (int mask = LANES / 2; mask; mask >>= 1) {
            const Pick o = {__shfl_xor(p.v, mask), __shfl_xor(p.i, mask)};
            if (better(o, p)) p = o;
        }
        if constexpr (G > 64) {
            Pick* mine = (Pick*)&lds[slot][threadIdx.x >> 6];
            if ((threadIdx.x & 63) == 0) *mine = p;
            __syncthreads();
            p = *(const Pick*)&lds[slot][0];
#pragma unroll
            for (int w = 1; w < WAVES; w++) {
                const Pick o = *(const Pick*)&lds[slot][w];
                if (better(o, p)) p = o;
            }
            slot ^= 1;
        }
        return p;
    }
};

// The best of a thread's logits that come after `last`. A NaN is none, nor is -infinity.
template <class T, int G, int NV>
__device__ __forceinline__ Pick best_after(const Held<T, G, NV>& x, int n, int lane, const Pick& last) {
    constexpr int E = EACH<T>;
    Pick p = NO_PICK;
    auto take = [&](float v, int i) {
        if (better(last, {v, i}) && v > p.v) p = {v, i};  // columns come in order
    };
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int i = 0; i < E; i++) take((float)x.v[k][i], (lane + k * G) * E + i);
        __builtin_amdgcn_sched_barrier(0);
    }
    take((float)x.one, n / E * E + lane);
    return p;
}

// The top picks of what a team holds, or of lists. A bound that at least `top` of them reach: the top-th largest of the
// threads' own maxima. What reaches it goes to LDS, a few more than `top` (21 of 2,048 normal logits on 256 threads for
// 20), and each finds its rank there by comparing with the others. A thread that holds more than its share of the
// largest, or very many equal logits, may fill the places: then the picks are taken one by one.
constexpr int MOST_CANDIDATES = 512;

template <int G>
struct Candidates {
    static constexpr int TEAMS = G > 64 ? 1 : LOGP_BLOCK / G;
    static constexpr int PLACES = G > 64 ? MOST_CANDIDATES : 64;
    Pick picks[TEAMS][PLACES];
    int count[TEAMS];
    float maxima[G > 64 ? G : 1];
    float bound;
};

// Floats in the order of unsigned integers, with zeros of both signs alike.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);
    return u ^ ((int32_t)u < 0 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t k) {
    return __uint_as_float(k ^ ((int32_t)k < 0 ? 0x80000000u : 0xFFFFFFFFu));
}

constexpr float LEAST = -3.4028234663852886e38f;  // the least logit that is an alternative

// The top-th largest of the threads' maxima, or less; at least LEAST.
template <int G>
__device__ __forceinline__ float bound_of(float own, float largest, int top, Team<G>& team, Candidates<G>& c) {
    if (top == 1) return fmaxf(largest, LEAST);
    if (top > G) return LEAST;
    if constexpr (G <= 64) {
        float b = largest;
        for (int t = 1; t < top; t++) {
            if (own == b) own = -INFINITY;  // equal ones at once: the bound is lower then, and holds
            b = over_lanes<G>(own, Larger());
        }
        return fmaxf(b, LEAST);
    } else {
        // bit by bit from the highest, by the first wavefront
        c.maxima[threadIdx.x] = own;
        __syncthreads();
        if (threadIdx.x < 64) {
            uint32_t key[G / 64], b = 0;
#pragma unroll
            for (int k = 0; k < G / 64; k++) key[k] = order_of(c.maxima[threadIdx.x + 64 * k]);
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                int reach = 0;
#pragma unroll
                for (int k = 0; k < G / 64; k++) reach += __popcll(__ballot(key[k] >= (b | bit)));
                if (reach >= top) b |= bit;
                if (reach == top) break;
            }
            if (threadIdx.x == 0) c.bound = b <= order_of(-INFINITY) ? LEAST : of_order(b);
        }
        __syncthreads();
        return c.bound;
    }
}

// Writes the picks: out(t, pick) for t < top, NO_PICK where there are fewer. scan(bound, add) adds the thread's logits
// from the bound on; after(last) is the thread's best after a pick.
template <int G, class Scan, class After, class Out>
__device__ __forceinline__ void top_of(float own, float largest, int top, int lane, Team<G>& team, Candidates<G>& c,
                                       Scan&& scan, After&& after, Out&& out) {
    typedef Candidates<G> C;
    const int mine = G > 64 ? 0 : threadIdx.x / G;
    auto sync = [] {
        if constexpr (G > 64) __syncthreads();
        else {  // a team is in one wavefront, whose LDS accesses stay in order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };
    if (lane == 0) c.count[mine] = 0;
    const float bound = bound_of<G>(own, largest, top, team, c);
    sync();
    if (own >= bound)
        scan(bound, [&](float v, int i) {
            const int at = atomicAdd(&c.count[mine], 1);
            if (at < C::PLACES) c.picks[mine][at] = {v, i};
        });
    sync();
    const int have = *(volatile int*)&c.count[mine];
    if (have <= C::PLACES) {
        for (int k = lane; k < have; k += G) {
            const Pick p = c.picks[mine][k];
            int rank = 0;
            for (int o = 0; o < have; o++) rank += better(c.picks[mine][o], p);
            if (rank < top) out(rank, p);
        }
        for (int t = have + lane; t < top; t += G) out(t, NO_PICK);
    }
    if (G > 64 ? have > C::PLACES : __any(have > C::PLACES)) {
        // all of a wavefront's teams, since they take part in each other's exchanges
        Pick last = {INFINITY, -1}, best = after(last);
        for (int t = 0; t < top; t++) {
            if (best.i == last.i) best = after(last);
            last = team.best(best);
            if (lane == 0) out(t, last);
        }
    }
    sync();
}

struct LogpRows {
    int64_t rows;
    const void* tokens;  // may be null
    int32_t top, splits, chunk;
    float *logp, *entropy;
    int32_t* rank;
    float* top_logp;
    int32_t* top_index;
    float4* stats;  // the maximum, the sum's logarithm to base 2, the entropy, 1 if counted
};

// A chunk's share, for the rows that have several.
struct ChunkPart {
    Part p;
    int32_t before, pad;
};

// A row's outputs from its statistics: what the alternatives need in every thread, and written by one.
__device__ __forceinline__ void row_out(const LogpRows& o, const Rate& k, int64_t r, const Part& p, float mine, int rank,
                                        bool on, bool write, float* fix, float* log_s) {
    float lp = 0.f, h = 0.f;
    *log_s = *fix = 0.f;
    if (on) {
        const float mean = p.t * LN2 / p.s;
        *log_s = logf(p.s);
        *fix = k.off * mean;
        h = (*log_s - *fix) - mean;
        lp = (mine - p.m) * k.inv_temp + *fix - *log_s;
    }
    if (!write) return;
    if (o.logp) o.logp[r] = lp;
    if (o.rank) o.rank[r] = on ? rank : -1;
    o.entropy[r] = h;
    if (o.stats) o.stats[r] = make_float4(on ? p.m : 0.f, on ? __log2f(p.s) : 0.f, h, on ? 1.f : 0.f);
}

__device__ __forceinline__ void top_out(const LogpRows& o, const Rate& k, int64_t r, int t, const Pick& p, float m,
                                        float fix, float log_s) {
    const bool is = p.i != NO_PICK.i;
    o.top_logp[r * o.top + t] = is ? (p.v - m) * k.inv_temp + fix - log_s : -INFINITY;
    o.top_index[r * o.top + t] = is ? p.i : -1;
}

// A row, or one chunk of it, on G threads.
template <class T, int G, int NV, bool CHUNKS>
__global__ __launch_bounds__(G > 64 ? G : LOGP_BLOCK, G > 256 ? 4 : 1) void k_logp(Rows<T> in, LogpRows o, ChunkPart* parts,
                                                                                  Pick* picks) {
    constexpr int E = EACH<T>, TEAMS = G > 64 ? 1 : LOGP_BLOCK / G;
    __shared__ typename Team<G>::Slots slots;
    __shared__ Candidates<G> candidates;
    Team<G> team{slots};
    const int lane = threadIdx.x % G;
    const int64_t unit = int64_t(blockIdx.x) * TEAMS + (G > 64 ? 0 : threadIdx.x / G);
    const int64_t r = CHUNKS ? unit / o.splits : unit;
    const int64_t c0 = CHUNKS ? (unit - r * o.splits) * o.chunk : 0;
    const int n = (int)(CHUNKS ? min<int64_t>(o.chunk, in.vocab - c0) : in.vocab);
    const bool there = r < o.rows;
    int64_t a = -1;
    if (there && o.tokens) a = index_at(o.tokens, in.bits, r);
    const bool read = there && (!o.tokens || (a >= 0 && a < in.vocab));
    if (G > 64 && !read && CHUNKS) return;
    Held<T, G, NV> x;
    const float rate = in.rate.rate;
    const T* row = in.x + r * in.x_stride;
    const uint8_t* legal = in.legal ? in.legal + r * in.legal_stride : nullptr;
    // the token's logit, and those before it in its load (of E, counted from the chunk's start)
    const int at = (int)(a - c0), near = at >= 0 && at < n ? at % E : 0;
    float mine = -INFINITY, beside = -INFINITY;
    if (read) {
        if (o.tokens) {
            if (!legal || legal[a]) mine = (float)row[a];
            if (lane < near && (!legal || legal[a - near + lane])) beside = (float)row[a - near + lane];
        }
        x.load(row + c0, legal ? legal + c0 : nullptr, n, lane);
    } else {
        x.none();
    }

    float own = fmaxf((float)x.one, -INFINITY);  // of nothing but NaN: -infinity, which no bound counts
#pragma unroll
    for (int k = 0; k < NV; k++) {
#pragma unroll
        for (int i = 0; i < E; i++) own = fmaxf(own, (float)x.v[k][i]);
        __builtin_amdgcn_sched_barrier(0);  // one load's values converted at a time
    }
    float largest[1] = {own};
    team.all(largest, Larger());
    x.forget();
    const float m = largest[0] == -INFINITY ? 0.f : largest[0];  // a row of nothing but -infinity keeps its differences
    // Larger logits come before the token, and equal ones of a lower index: all at or above it in the loads before its
    // own, all above it from there on, and what is equal beside it. (Below -infinity there is no float: then all
    // are counted once more.)
    const bool lowest = o.tokens && mine == -INFINITY;
    const float below = of_order(order_of(mine) - (mine == 0.f ? 2 : 1));  // not -0, which is no less than 0
    float s = 0.f, t = 0.f;
    int before = lane < near && beside == mine;
    auto count = [&](float v, float from) {
        const float z = (v - m) * rate, e = power(z);
        s += e;
        t += e * fmaxf(z, -300.f);  // e is 0 there, and 0 * -infinity would be NaN
        before += v > from;
    };
    const int whole = n / E;
    const float over_one = whole * E + lane < at ? below : mine;  // the columns past the last whole load are loads of one
    count((float)x.one, at / E == whole ? mine : over_one);
#pragma unroll
    for (int k = 0; k < NV; k++) {
        const float from = (lane + k * G + 1) * E <= at ? below : mine;
#pragma unroll
        for (int i = 0; i < E; i++) count((float)x.v[k][i], from);
        __builtin_amdgcn_sched_barrier(0);
    }
    x.forget();
    float sums[3] = {s, t, (float)before};
    team.all(sums, Added());
    const Part p = {largest[0], sums[0], sums[1], 0.f, -INFINITY, 0.f};
    const bool on = read && counts(p);
    if (lowest) {  // a token of no probability: what is above -infinity comes before it, and every column of a lower index
        float more[1] = {0.f};
        auto late = [&](float v, int i) { more[0] += v > -INFINITY || i < at; };
#pragma unroll
        for (int k = 0; k < NV; k++) {
            // past the last whole load the columns are loads of one
#pragma unroll
            for (int i = 0; i < E; i++)
                if (lane + k * G < whole) late((float)x.v[k][i], (lane + k * G) * E + i);
            __builtin_amdgcn_sched_barrier(0);
        }
        x.forget();
        if (whole * E + lane < n) late((float)x.one, whole * E + lane);
        sums[2] = more[0];
    }
    if (G > 64 ? lowest : __any(lowest)) {
        float more[1] = {sums[2]};
        team.all(more, Added());
        if (lowest) sums[2] = more[0];
    }
    float fix = 0.f, log_s = 0.f;
    if constexpr (CHUNKS) {
        if (lane == 0) parts[unit] = {p, (int32_t)sums[2], 0};
    } else if (there) {
        row_out(o, in.rate, r, p, mine, (int)sums[2], on, lane == 0, &fix, &log_s);
    }
    if (!o.top) return;
    top_of<G>(
        on ? own : -INFINITY, on ? largest[0] : -INFINITY, o.top, lane, team, candidates,
        [&](float bound, auto&& add) {
            x.forget();
#pragma unroll
            for (int k = 0; k < NV; k++) {
                float most = (float)x.v[k][0];
#pragma unroll
                for (int i = 1; i < E; i++) most = fmaxf(most, (float)x.v[k][i]);
                if (most >= bound) {
#pragma unroll
                    for (int i = 0; i < E; i++)
                        if ((float)x.v[k][i] >= bound) add((float)x.v[k][i], (lane + k * G) * E + i);
                }
            }
            if ((float)x.one >= bound) add((float)x.one, whole * E + lane);
        },
        [&](const Pick& last) {
            x.forget();
            return on ? best_after(x, n, lane, last) : NO_PICK;
        },
        [&](int k, const Pick& q) {
            if constexpr (CHUNKS) picks[unit * o.top + k] = {q.v, q.i == NO_PICK.i ? q.i : (int)(q.i + c0)};
            else if (there) top_out(o, in.rate, r, k, q, p.m, fix, log_s);
        });
}

// A row's chunks joined: a workgroup a row.
template <class T>
__global__ __launch_bounds__(LOGP_BLOCK) void k_logp_join(Rows<T> in, LogpRows o, const ChunkPart* parts,
                                                          const Pick* picks) {
    __shared__ ChunkPart wave_part[LOGP_BLOCK / 64];
    __shared__ Team<LOGP_BLOCK>::Slots slots;
    __shared__ Candidates<LOGP_BLOCK> candidates;
    Team<LOGP_BLOCK> team{slots};
    const int t = threadIdx.x;
    const int64_t r = blockIdx.x;
    int64_t a = -1;
    if (o.tokens) a = index_at(o.tokens, in.bits, r);
    const bool read = !o.tokens || (a >= 0 && a < in.vocab);
    const float rate = in.rate.rate;
    float v = -INFINITY;
    if (read && o.tokens && (!in.legal || in.legal[r * in.legal_stride + a])) v = (float)in.x[r * in.x_stride + a];
    // a chunk's list is in order: its head is its largest
    const Pick* lists = picks + r * o.splits * o.top;
    ChunkPart mine = {{-INFINITY, 0.f, 0.f, 0.f, -INFINITY, 0.f}, 0, 0};
    float own = -INFINITY;
    if (read)
        for (int k = t; k < o.splits; k += LOGP_BLOCK) {
            const ChunkPart c = parts[r * o.splits + k];
            if (o.top) own = fmaxf(own, lists[k * o.top].v);
            mine.p = join(mine.p, c.p, rate);
            mine.before += c.before;
        }
    for (int mask = 32; mask; mask >>= 1) {
        Part q;
        q.m = __shfl_xor(mine.p.m, mask), q.s = __shfl_xor(mine.p.s, mask), q.t = __shfl_xor(mine.p.t, mask);
        q.d = q.sy = 0.f, q.my = -INFINITY;
        // the lower lane's first, in both: the same bits
        mine.p = t & mask ? join(q, mine.p, rate) : join(mine.p, q, rate);
        mine.before += __shfl_xor(mine.before, mask);
    }
    if ((t & 63) == 0) wave_part[t >> 6] = mine;
    __syncthreads();
    mine = wave_part[0];
    for (int w = 1; w < LOGP_BLOCK / 64; w++) {
        mine.p = join(mine.p, wave_part[w].p, rate);
        mine.before += wave_part[w].before;
    }
    const bool on = read && counts(mine.p);
    float fix = 0.f, log_s = 0.f;
    row_out(o, in.rate, r, mine.p, v, mine.before, on, t == 0, &fix, &log_s);
    if (!o.top) return;
    top_of<LOGP_BLOCK>(
        on ? own : -INFINITY, on ? mine.p.m : -INFINITY, o.top, t, team, candidates,
        [&](float bound, auto&& add) {
            for (int k = t; k < o.splits; k += LOGP_BLOCK)
                for (int u = 0; u < o.top; u++) {
                    const Pick q = lists[k * o.top + u];
                    if (!(q.v >= bound)) break;
                    add(q.v, q.i);
                }
        },
        [&](const Pick& last) {
            Pick p = NO_PICK;
            if (on)
                for (int k = t; k < o.splits; k += LOGP_BLOCK)
                    for (int u = 0; u < o.top; u++) {
                        const Pick q = lists[k * o.top + u];
                        if (!better(last, q)) continue;
                        if (better(q, p)) p = q;
                        break;
                    }
            return p;
        },
        [&](int k, const Pick& q) { top_out(o, in.rate, r, k, q, mine.p.m, fix, log_s); });
}

// The gradient of a row, or of one chunk of it.
template <class T, int G, int NV>
__global__ __launch_bounds__(LOGP_BLOCK) void k_logp_back(Rows<T> in, LogpRows o, const float* d_logp,
                                                          const float* d_entropy, T* grad, int64_t grad_stride) {
    const int lane = threadIdx.x % G;
    const int64_t unit = int64_t(blockIdx.x) * (LOGP_BLOCK / G) + threadIdx.x / G;
    const int64_t r = unit / o.splits, c0 = (unit - r * o.splits) * o.chunk;
    if (r >= o.rows) return;
    const int n = (int)min<int64_t>(o.chunk, in.vocab - c0);
    const float4 st = o.stats[r];
    int64_t a = -1;
    if (o.tokens) a = index_at(o.tokens, in.bits, r);
    RowGrad g = {};
    g.m = st.x;
    g.log_s = st.y;
    g.h = st.z;
    g.on = st.w != 0.f && (!o.tokens || (a >= 0 && a < in.vocab));
    g.coef = o.tokens && d_logp ? d_logp[r] : 0.f;
    g.ent = d_entropy ? -d_entropy[r] : 0.f;
    T* to = grad + r * grad_stride + c0;
    if (!g.any()) {
        put_zero<T, G, NV>(to, n, lane);
        return;
    }
    const uint8_t* legal = in.legal ? in.legal + r * in.legal_stride + c0 : nullptr;
    Held<T, G, NV> x;
    Held<T, G, 1> none;
    none.one = (T)0.f;
    x.load(in.x + r * in.x_stride + c0, legal, n, lane);
    int at = a >= c0 && a < c0 + n ? (int)(a - c0) : -1;
    if (at >= 0 && legal && !legal[at]) at = -1;
    const Slope slope(g, in.rate.inv_temp);
    if (g.ent == 0.f && slope.finite()) put_grad<T, G, NV, false, true>(to, n, lane, x, none, slope, in.rate.rate, at);
    else put_grad<T, G, NV, false, false>(to, n, lane, x, none, slope, in.rate.rate, at);
}

// ------------------------------------------------------------------ launches

// Rows beyond what a workgroup holds are cut into chunks, and so are long ones that are too few to fill the device
// otherwise: into chunks of eight loads a thread, or of as many as leave two workgroups a CU.
struct LogpPlan {
    int splits, loads;  // loads a thread, for chunks
    size_t picks, bytes;
};

template <class T>
LogpPlan logp_plan(int64_t rows, int64_t vocab, int top, int cus) {
    constexpr int64_t E = EACH<T>;
    const int64_t n = vocab / E;
    LogpPlan p = {};
    if (n <= LOGP_BLOCK || (n <= 8192 && rows >= cus)) {
        p.splits = 1;
        return p;
    }
    auto cut = [&](int loads) { return (vocab + E * LOGP_BLOCK * loads - 1) / (E * LOGP_BLOCK * loads); };
    p.loads = 8;
    while (p.loads > 1 && rows * cut(p.loads) < 2 * cus) p.loads /= 2;
    p.splits = (int)cut(p.loads);
    p.picks = pad256(size_t(rows) * p.splits * sizeof(ChunkPart));
    p.bytes = p.picks + pad256(size_t(rows) * p.splits * top * sizeof(Pick));
    return p;
}

// The fewest threads that hold a row of n loads in at most eight loads each (as rows_held in policy_dev.h), and at least
// `lanes` of them: a row's top alternatives are bounded by as many threads' maxima.
template <class T, class F>
void held_by(int64_t n, int lanes, F&& launch) {
    using std::integral_constant;
#define HELD_BY(most, g, nv) \
    if (n <= most && (g >= 64 || g >= lanes)) return launch(integral_constant<int, g>(), integral_constant<int, nv>());
    HELD_BY(8, 8, 1)
    HELD_BY(16, 8, 2)
    HELD_BY(32, 8, 4)
    HELD_BY(64, 8, 8)
    HELD_BY(80, 16, 5)
    HELD_BY(128, 16, 8)
    HELD_BY(160, 32, 5)
    HELD_BY(256, 32, 8)
    HELD_BY(320, 64, 5)
    HELD_BY(512, 64, 8)
    HELD_BY(1024, 256, 4)
    HELD_BY(2048, 256, 8)
#undef HELD_BY
}

template <class T>
Rows<T> logp_rows(const void* logits, int64_t stride, const uint8_t* legal, int64_t legal_stride, int64_t vocab,
                  float inv_temperature, int bits) {
    return {(const T*)logits, stride, legal, legal_stride, nullptr, 0, nullptr, nullptr, vocab, rate_of(inv_temperature),
            bits, 1.f};
}

// Rows of a launch, which holds fewer than 2^32 threads: at most 512 a row or chunk.
inline int64_t rows_at_once(int64_t splits) { return std::max<int64_t>(1, (int64_t(1) << 22) / splits); }

template <class T>
void logp_of(const wc_logp_args& a, const LogpPlan& p, hipStream_t s) {
    const Rows<T> in = logp_rows<T>(a.logits, a.logits_stride, a.legal, a.legal_stride, a.vocab, a.inv_temperature,
                                    a.index_bits);
    LogpRows o = {a.rows, a.tokens, a.top, p.splits, 0, a.logp, a.entropy, a.rank, a.top_logp, a.top_index,
                  (float4*)a.stats};
    auto grid = [&](int g) {
        const int64_t per = g > 64 ? 1 : LOGP_BLOCK / g;
        return dim3((uint32_t)((a.rows * p.splits + per - 1) / per));
    };
    if (p.splits == 1) {
        const int64_t n = a.vocab / EACH<T>;
        if (n > 4096) {
            k_logp<T, 512, 16, false><<<grid(512), 512, 0, s>>>(in, o, nullptr, nullptr);
        } else if (n > 2048) {
            k_logp<T, 512, 8, false><<<grid(512), 512, 0, s>>>(in, o, nullptr, nullptr);
        } else {
            held_by<T>(n, a.top, [&](auto g, auto nv) {
                k_logp<T, g(), nv(), false><<<grid(g()), LOGP_BLOCK, 0, s>>>(in, o, nullptr, nullptr);
            });
        }
        return;
    }
    ChunkPart* parts = (ChunkPart*)a.workspace;
    Pick* picks = (Pick*)((char*)a.workspace + p.picks);
    o.chunk = LOGP_BLOCK * EACH<T> * p.loads;
    if (p.loads == 8) k_logp<T, LOGP_BLOCK, 8, true><<<grid(LOGP_BLOCK), LOGP_BLOCK, 0, s>>>(in, o, parts, picks);
    else if (p.loads == 4) k_logp<T, LOGP_BLOCK, 4, true><<<grid(LOGP_BLOCK), LOGP_BLOCK, 0, s>>>(in, o, parts, picks);
    else if (p.loads == 2) k_logp<T, LOGP_BLOCK, 2, true><<<grid(LOGP_BLOCK), LOGP_BLOCK, 0, s>>>(in, o, parts, picks);
    else k_logp<T, LOGP_BLOCK, 1, true><<<grid(LOGP_BLOCK), LOGP_BLOCK, 0, s>>>(in, o, parts, picks);
    k_logp_join<T><<<dim3((uint32_t)a.rows), LOGP_BLOCK, 0, s>>>(in, o, parts, picks);
}

template <class T>
void logp(const wc_logp_args& a, int cus, hipStream_t s) {
    const LogpPlan p = logp_plan<T>(a.rows, a.vocab, a.top, cus);
    wc_logp_args o = a;
    for (int64_t lo = 0; lo < a.rows; lo += o.rows) {
        o.rows = std::min(a.rows - lo, rows_at_once(p.splits));
        o.logits = (const T*)a.logits + lo * a.logits_stride;
        if (a.legal) o.legal = a.legal + lo * a.legal_stride;
        if (a.tokens) o.tokens = (const char*)a.tokens + lo * (a.index_bits / 8);
        if (a.logp) o.logp = a.logp + lo;
        if (a.rank) o.rank = a.rank + lo;
        o.entropy = a.entropy + lo;
        if (a.top) o.top_logp = a.top_logp + lo * a.top, o.top_index = a.top_index + lo * a.top;
        if (a.stats) o.stats = a.stats + 4 * lo;
        logp_of<T>(o, p, s);
    }
}

template <class T>
void logp_back_of(const wc_logp_back_args& a, hipStream_t s) {
    const Rows<T> in = logp_rows<T>(a.logits, a.logits_stride, a.legal, a.legal_stride, a.vocab, a.inv_temperature,
                                    a.index_bits);
    constexpr int64_t E = EACH<T>, CHUNK_COLUMNS = LOGP_BLOCK * E * 8;
    const int64_t n = std::min<int64_t>(a.vocab / E, 8 * LOGP_BLOCK);
    const int splits = a.vocab / E <= n ? 1 : (int)((a.vocab + CHUNK_COLUMNS - 1) / CHUNK_COLUMNS);
    LogpRows o = {};
    o.rows = a.rows;
    o.tokens = a.tokens;
    o.splits = splits;
    o.chunk = splits == 1 ? (int)a.vocab : (int)CHUNK_COLUMNS;
    o.stats = (float4*)a.stats;
    held_by<T>(n, 8, [&](auto g, auto nv) {
        const int64_t per = LOGP_BLOCK / g();
        k_logp_back<T, g(), nv()><<<dim3((uint32_t)((a.rows * splits + per - 1) / per)), LOGP_BLOCK, 0, s>>>(
            in, o, a.d_logp, a.d_entropy, (T*)a.grad, a.grad_stride);
    });
}

template <class T>
void logp_back(const wc_logp_back_args& a, hipStream_t s) {
    const int64_t most = rows_at_once((a.vocab + LOGP_BLOCK * EACH<T> * 8 - 1) / (LOGP_BLOCK * EACH<T> * 8));
    wc_logp_back_args o = a;
    for (int64_t lo = 0; lo < a.rows; lo += o.rows) {
        o.rows = std::min(a.rows - lo, most);
        o.logits = (const T*)a.logits + lo * a.logits_stride;
        if (a.legal) o.legal = a.legal + lo * a.legal_stride;
        if (a.tokens) o.tokens = (const char*)a.tokens + lo * (a.index_bits / 8);
        o.stats = a.stats + 4 * lo;
        if (a.d_logp) o.d_logp = a.d_logp + lo;
        if (a.d_entropy) o.d_entropy = a.d_entropy + lo;
        o.grad = (T*)a.grad + lo * a.grad_stride;
        logp_back_of<T>(o, s);
    }
}

}  // namespace
}  // namespace learn
}  // namespace wc
