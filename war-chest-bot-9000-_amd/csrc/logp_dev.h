// Log-probabilities of given tokens, their rank, the entropy and the top alternatives of rows of logits, and the gradient
// (include/wc_learn.h), for one element type: logp_f32.hip, logp_f16.hip and logp_bf16.hip build one each.
//
//   z_j = inv_temperature x_j, logp_j = z_j - log sum exp z, H = -sum p logp
//   grad_j = inv_temperature (d_logp ([j = a] - p_j) - d_H p_j (logp_j + H))
//
// Rows are read once and held in registers (rows_dev.h): as few threads as hold a row, or a workgroup for each chunk of
// a long one, whose statistics and lists are joined by a second launch.
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

// The best of G threads' picks, the same in each.
template <int G>
struct PickGroup {
    static constexpr int WAVES = G > 64 ? G / 64 : 1;
    typedef Pick Slots[2][WAVES];
    Slots& lds;
    int slot = 0;

    __device__ __forceinline__ Pick best(Pick p) {
#pragma unroll
        for (int mask = (G < 64 ? G : 64) / 2; mask; mask >>= 1) {
            const Pick o = {__shfl_xor(p.v, mask), __shfl_xor(p.i, mask)};
            if (better(o, p)) p = o;
        }
        if constexpr (G > 64) {
            if ((threadIdx.x & 63) == 0) lds[slot][threadIdx.x >> 6] = p;
            __syncthreads();
            p = lds[slot][0];
#pragma unroll
            for (int w = 1; w < WAVES; w++)
                if (better(lds[slot][w], p)) p = lds[slot][w];
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
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < E; i++) take((float)x.v[k][i], (lane + k * G) * E + i);
    take((float)x.one, n / E * E + lane);
    return p;
}

// How many of a thread's logits are ranked before `mine`.
template <class T, int G, int NV>
__device__ __forceinline__ int before(const Held<T, G, NV>& x, int n, int lane, const Pick& mine) {
    constexpr int E = EACH<T>;
    int count = 0;
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < E; i++) count += better({(float)x.v[k][i], (lane + k * G) * E + i}, mine);
    return count + better({(float)x.one, n / E * E + lane}, mine);
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
    float before;
    float pad;
};

// A row's outputs from its statistics: by lane 0.
__device__ __forceinline__ void row_out(const LogpRows& o, const Rate& k, int64_t r, const Part& p, float mine, int rank,
                                        bool on, float* fix, float* log_s) {
    float lp = 0.f, h = 0.f;
    *log_s = *fix = 0.f;
    if (on) {
        const float mean = p.t * LN2 / p.s;
        *log_s = logf(p.s);
        *fix = k.off * mean;
        h = (*log_s - *fix) - mean;
        lp = (mine - p.m) * k.inv_temp + *fix - *log_s;
    }
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
__global__ __launch_bounds__(LOGP_BLOCK) void k_logp(Rows<T> in, LogpRows o, ChunkPart* parts, Pick* picks) {
    __shared__ typename Group<G>::Slots slots;
    __shared__ typename PickGroup<G>::Slots pick_slots;
    Group<G> group{slots};
    PickGroup<G> pick{pick_slots};
    const int lane = threadIdx.x % G;
    const int64_t unit = int64_t(blockIdx.x) * (LOGP_BLOCK / G) + threadIdx.x / G;
    const int64_t r = CHUNKS ? unit / o.splits : unit;
    const int64_t c0 = CHUNKS ? (unit - r * o.splits) * o.chunk : 0;
    const int n = (int)(CHUNKS ? min<int64_t>(o.chunk, in.vocab - c0) : in.vocab);
    const bool there = r < o.rows;
    int64_t a = -1;
    if (there && o.tokens) a = index_at(o.tokens, in.bits, r);
    const bool read = there && (!o.tokens || (a >= 0 && a < in.vocab));
    if (G > 64 && !read && CHUNKS) return;
    Held<T, G, NV> x;
    Held<T, G, 1> none;
    none.one = (T)0.f;
    Pick mine = {-INFINITY, (int)(a - c0)};
    if (read) {
        const uint8_t* legal = in.legal ? in.legal + r * in.legal_stride + c0 : nullptr;
        if (o.tokens && (!in.legal || in.legal[r * in.legal_stride + a])) mine.v = (float)in.x[r * in.x_stride + a];
        x.load(in.x + r * in.x_stride + c0, legal, n, lane);
    } else {
        x.none();
    }
    const Part p = held_stats<T, G, NV, false>(x, none, in.rate.rate, group);
    float rank[1] = {0.f};
    if (o.tokens) {
        rank[0] = (float)before(x, n, lane, mine);
        group.template all<1, false>(rank);
    }
    const bool on = read && counts(p);
    float fix = 0.f, log_s = 0.f;
    if constexpr (CHUNKS) {
        if (lane == 0) parts[unit] = {p, rank[0], 0.f};
    } else if (lane == 0 && there) {
        row_out(o, in.rate, r, p, mine.v, (int)rank[0], on, &fix, &log_s);
    }
    if (!o.top) return;
    Pick last = {INFINITY, -1}, own = best_after(x, n, lane, last);
    for (int t = 0; t < o.top; t++) {
        if (own.i == last.i) own = best_after(x, n, lane, last);
        last = pick.best(own);
        if (lane == 0) {
            if constexpr (CHUNKS) picks[unit * o.top + t] = {last.v, last.i == NO_PICK.i ? last.i : (int)(last.i + c0)};
            else if (there) top_out(o, in.rate, r, t, on ? last : NO_PICK, p.m, fix, log_s);
        }
    }
}

// A row's chunks joined: a workgroup a row.
template <class T>
__global__ __launch_bounds__(LOGP_BLOCK) void k_logp_join(Rows<T> in, LogpRows o, const ChunkPart* parts,
                                                          const Pick* picks) {
    __shared__ ChunkPart wave_part[LOGP_BLOCK / 64];
    __shared__ PickGroup<LOGP_BLOCK>::Slots pick_slots;
    PickGroup<LOGP_BLOCK> pick{pick_slots};
    const int t = threadIdx.x;
    const int64_t r = blockIdx.x;
    int64_t a = -1;
    if (o.tokens) a = index_at(o.tokens, in.bits, r);
    const bool read = !o.tokens || (a >= 0 && a < in.vocab);
    const float rate = in.rate.rate;
    ChunkPart mine = {{-INFINITY, 0.f, 0.f, 0.f, -INFINITY, 0.f}, 0.f, 0.f};
    if (read)
        for (int k = t; k < o.splits; k += LOGP_BLOCK) {
            const ChunkPart c = parts[r * o.splits + k];
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
    if (t == 0) {
        float v = -INFINITY;
        if (read && o.tokens && (!in.legal || in.legal[r * in.legal_stride + a])) v = (float)in.x[r * in.x_stride + a];
        row_out(o, in.rate, r, mine.p, v, (int)mine.before, on, &fix, &log_s);
    }
    // a chunk's list is in order: a thread's best is at its lists' heads
    const int64_t lists = r * o.splits;
    auto best_of = [&](const Pick& last) {
        Pick p = NO_PICK;
        if (on)
            for (int k = t; k < o.splits; k += LOGP_BLOCK)
                for (int u = 0; u < o.top; u++) {
                    const Pick q = picks[(lists + k) * o.top + u];
                    if (!better(last, q)) continue;
                    if (better(q, p)) p = q;
                    break;
                }
        return p;
    };
    Pick last = {INFINITY, -1}, own = NO_PICK;
    for (int u = 0; u < o.top; u++) {
        if (u == 0 || own.i == last.i) own = best_of(last);
        last = pick.best(own);
        if (t == 0) top_out(o, in.rate, r, u, last, mine.p.m, fix, log_s);
    }
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
    if (g.ent == 0.f) put_grad<T, G, NV, false, true>(to, n, lane, x, none, Slope(g, in.rate.inv_temp), in.rate.rate, at);
    else put_grad<T, G, NV, false, false>(to, n, lane, x, none, Slope(g, in.rate.inv_temp), in.rate.rate, at);
}

// ------------------------------------------------------------------ launches

// Rows beyond what a workgroup holds in eight loads a thread are cut into chunks; into smaller ones where the rows are
// too few to fill the device otherwise.
struct LogpPlan {
    int splits, loads;  // loads a thread, for chunks
    size_t picks, bytes;
};

template <class T>
LogpPlan logp_plan(int64_t rows, int64_t vocab, int top, int cus) {
    constexpr int64_t E = EACH<T>;
    LogpPlan p = {};
    if (vocab / E <= 8 * LOGP_BLOCK && (vocab / E <= LOGP_BLOCK || rows >= cus)) {
        p.splits = 1;
        return p;
    }
    p.loads = 8;
    while (p.loads > 1 && rows * ((vocab + E * LOGP_BLOCK * p.loads - 1) / (E * LOGP_BLOCK * p.loads)) < 2 * cus) p.loads /= 2;
    p.splits = (int)((vocab + E * LOGP_BLOCK * p.loads - 1) / (E * LOGP_BLOCK * p.loads));
    p.picks = pad256(size_t(rows) * p.splits * sizeof(ChunkPart));
    p.bytes = p.picks + pad256(size_t(rows) * p.splits * top * sizeof(Pick));
    return p;
}

// The fewest threads that hold a row in at most eight loads each (as rows_held in policy_dev.h).
template <class T, class F>
void held_by(int64_t n, F&& launch) {
    using std::integral_constant;
#define HELD_BY(most, g, nv) \
    if (n <= most) return launch(integral_constant<int, g>(), integral_constant<int, nv>());
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

template <class T>
void logp(const wc_logp_args& a, int cus, hipStream_t s) {
    if (!a.rows) return;
    const LogpPlan p = logp_plan<T>(a.rows, a.vocab, a.top, cus);
    const Rows<T> in = logp_rows<T>(a.logits, a.logits_stride, a.legal, a.legal_stride, a.vocab, a.inv_temperature,
                                    a.index_bits);
    LogpRows o = {a.rows, a.tokens, a.top, p.splits, 0, a.logp, a.entropy, a.rank, a.top_logp, a.top_index,
                  (float4*)a.stats};
    auto grid = [&](int g) {
        const int64_t per = LOGP_BLOCK / g;
        return dim3((uint32_t)((a.rows * p.splits + per - 1) / per));
    };
    if (p.splits == 1) {
        held_by<T>(a.vocab / EACH<T>, [&](auto g, auto nv) {
            k_logp<T, g(), nv(), false><<<grid(g()), LOGP_BLOCK, 0, s>>>(in, o, nullptr, nullptr);
        });
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
void logp_back(const wc_logp_back_args& a, hipStream_t s) {
    if (!a.rows) return;
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
    held_by<T>(n, [&](auto g, auto nv) {
        const int64_t per = LOGP_BLOCK / g();
        k_logp_back<T, g(), nv()><<<dim3((uint32_t)((a.rows * splits + per - 1) / per)), LOGP_BLOCK, 0, s>>>(
            in, o, a.d_logp, a.d_entropy, (T*)a.grad, a.grad_stride);
    });
}

}  // namespace
}  // namespace learn
}  // namespace wc
