// Matrix products on the matrix cores, C[m x n] = sum over k of A[i][k] B[k][j], with an epilogue that the caller gives:
// the layers' products (linear_dev.h) and the Newton-Schulz steps (newton.hip).
//
// An operand's index of summation is its contiguous one (INNER: A as rows of k, B as rows of k for each column) or its
// outer one. Tiles of 64 values of k go from memory to LDS without passing registers: A in three buffers and B in two,
// so that a step's loads have at least a step to arrive and one barrier a step is enough; whole lines of 128 bytes of an
// INNER operand. INNER tiles come back as 16 bytes a lane, the others through the transposing LDS read. A workgroup of
// four wavefronts owns a square tile of 64 F, each wavefront a quarter in F x F fragments of 32 x 32. Everything else
// goes between the matrix instructions: F of them, then the loads and the reads of one part.
//
// An operand may have several planes that add up to it; the product is then a sum of segments, pairs of planes, one
// after the other along k.
//
// 16,384 x 4,096 x 4,096 bf16: 410 to 447 us, 1.23 to 1.34 PFLOP/s, with matrix instructions in 75% of the cycles at the
// 1.63 GHz that the device's power allows; without the epilogue's bias, activation and residual.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "learn_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

constexpr int PRODUCT_BLOCK = 256, STEP = 64, A_BUFFERS = 3, B_BUFFERS = 2;
constexpr int MOST_SEGMENTS = 6, MOST_PLANES = 3;

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char* LdsAt;

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// One operand: rows of `pitch` bytes on 16-byte bounds, the contiguous index in whole chunks of eight
// (zeros past its end where it is k). `outer` rows of A or columns of B.
struct Operand16 {
    const char* plane[MOST_PLANES];
    int64_t pitch, batch;  // bytes from row to row, from one matrix to the next
    int64_t outer;
};

struct Product {
    Operand16 a, b;
    int64_t k;                 // of each segment
    int32_t segments;
    uint8_t pa[MOST_SEGMENTS], pb[MOST_SEGMENTS];  // a segment's planes
    int32_t tiles_m, tiles_n, runs, batches;
    int32_t triangle;          // the tiles' size where the result is symmetric and only those on and above the diagonal are made
    int32_t steps, run_steps;  // steps of all segments together, and of one run
    float* part;               // runs > 1: runs x batches x m x n partial products
};

static __device__ __align__(16) uint4 g_zeros;  // what lies past the end is read from here

template <int F>
struct TileShape {
    static constexpr int TILE = 64 * F, SIDE = TILE * 2 * STEP;
    static constexpr int LDS = (A_BUFFERS + B_BUFFERS) * SIDE;
    static constexpr int PARTS = 2 * F;  // a wavefront's loads of one operand's tile
    // Sixteen lanes' reads of 16 bytes are taken together, 256 bytes: an INNER row's 16-byte units are exchanged by its pair
    // of rows modulo 8. Where rows are on k: 64-byte units a row, exchanged so that the four rows of a transposing read lie in different
    // banks. A pitch of an odd number of 128 bytes puts rows 0 and 1 there by itself.
    static __device__ __forceinline__ int turn(int row) { return F & 1 ? (row >> 1) & 1 : row & 3; }
};

// One operand's way from memory to LDS, as one wavefront has it: PARTS loads a step of 64 lanes x 16 bytes each, to
// places in LDS that follow each other.
template <int F, bool INNER>
struct Fetch {
    typedef TileShape<F> S;
    uint32_t at[S::PARTS];  // the lane's place, from the tile's first row
    int first;              // the wavefront's first load and the lane, of the tile's 16-byte chunks
    const char* p;          // the tile of the step to load, the same for all lanes
    int64_t step, start;    // bytes from step to step, and from a plane's start to the tile's
    int segment, left;      // of the segment: steps left

    __device__ __forceinline__ void set(const Product& q, const Operand16& o, const uint8_t* planes, int batch, int64_t at0,
                                        int wave, int lane, int s, int steps_in) {
        first = wave * S::PARTS * 64 + lane;
        const uint32_t pitch = (uint32_t)o.pitch;
        const int beyond = (int)min<int64_t>(o.outer - at0, S::TILE);  // rows or columns of the tile that are there
#pragma unroll
        for (int k = 0; k < S::PARTS; k++) {
            const int g = first + 64 * k;
            if (INNER) {
                // past the last row any row will do: its products are not stored
                at[k] = (uint32_t)min(g / 8, beyond - 1) * pitch + 16 * ((g % 8) ^ (g / 16 & 7));
            } else {
                const int row = g / (8 * F), chunk = (g % (8 * F)) ^ (S::turn(row) << 2);
                at[k] = (uint32_t)row * pitch + (8 * chunk < beyond ? 16 * chunk : 0);
            }
        }
        step = INNER ? 2 * STEP : STEP * o.pitch;
        start = batch * o.batch + (INNER ? at0 * o.pitch : 2 * at0);
        segment = q.segments > 1 ? s / steps_in : 0;
        const int in = s - segment * steps_in;
        left = steps_in - in;
        p = o.plane[planes[segment]] + start + in * step;
    }
    __device__ __forceinline__ void next(const Product& q, const Operand16& o, const uint8_t* planes, int steps_in) {
        p += step;
        if (--left == 0 && segment + 1 < q.segments) {
            segment++;
            left = steps_in;
            p = o.plane[planes[segment]] + start;
        }
    }
    // The first of k that load k brings.
    __device__ __forceinline__ int k_of(int k) const {
        const int g = first + 64 * k;
        return INNER ? 8 * ((g % 8) ^ (g / 16 & 7)) : g / (8 * F);
    }
    // Load k of the step, to the wavefront's place. ENDS: what lies at or past `there` of the step's k is read from zeros.
    template <bool ENDS>
    __device__ __forceinline__ void load(int k, int64_t there, LdsAt to) const {
        const char* from = p + at[k];
        if (ENDS && k_of(k) >= there) from = (const char*)&g_zeros;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                         (__attribute__((address_space(3))) void*)(to + 1024 * k), 16, 0, 0);
    }
};

// A wavefront's reads of one operand's fragments: lane l has eight of k, from 8 (l / 32) on, of row or column l % 32.
template <int F, bool INNER>
struct Reads {
    typedef TileShape<F> S;
    uint32_t at[INNER ? 1 : F];

    __device__ __forceinline__ void set(int first, int lane) {
        if (INNER) {
            const int row = first + (lane & 31);
            at[0] = row * 2 * STEP + 16 * ((lane >> 5) ^ (row >> 1 & 7));
        } else {
            const int row = 8 * (lane >> 5) + ((lane & 15) >> 2);
#pragma unroll
            for (int m = 0; m < F; m++)
                at[m] = row * 2 * S::TILE +
                        ((2 * (first + 32 * m + (lane & 16) + 4 * (lane & 3))) ^ (S::turn(row) << 6));
        }
    }
    // Fragment m of the sixteen of k from 16 part on.
    template <class E8>
    __device__ __forceinline__ E8 take(LdsAt from, int part, int m) const {
        if constexpr (INNER) {
            typedef __attribute__((address_space(3))) E8* At;
            return *(At)(from + (at[0] ^ (part << 5)) + m * 32 * 2 * STEP);
        } else {
            typedef __attribute__((address_space(3))) s16x4* At;
            const LdsAt p = from + at[m] + part * 16 * 2 * S::TILE;
            // four rows on, the exchange of units is the same
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)(p + 4 * 2 * S::TILE));
            return __builtin_bit_cast(E8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// All loads but the last LEFT have arrived, in every wavefront, and every wavefront's reads.
template <int LEFT>
__device__ __forceinline__ void arrived() {
    static_assert(LEFT == 2 || LEFT == 4 || LEFT == 6 || LEFT == 8, "a step's loads of A");
    if constexpr (LEFT == 2) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)" ::: "memory");
    else if constexpr (LEFT == 4) asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
    else if constexpr (LEFT == 6) asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
}

template <class E, int F, bool AI, bool BI>
struct Tiles {
    typedef E E8 __attribute__((ext_vector_type(8)));
    typedef TileShape<F> S;
    const Product& q;
    Fetch<F, AI> fa;
    Fetch<F, BI> fb;
    Reads<F, AI> ra;
    Reads<F, BI> rb;
    int steps_in;  // of a segment

    __device__ __forceinline__ Tiles(const Product& product, int batch, int64_t i0, int64_t j0, int wave, int lane, int s)
        : q(product) {
        steps_in = (int)((q.k + STEP - 1) / STEP);
        fa.set(q, q.a, q.pa, batch, i0, wave, lane, s, steps_in);
        fb.set(q, q.b, q.pb, batch, j0, wave, lane, s, steps_in);
        ra.set((wave >> 1) * 32 * F, lane);
        rb.set((wave & 1) * 32 * F, lane);
    }
    __device__ __forceinline__ void next_a() { fa.next(q, q.a, q.pa, steps_in); }
    __device__ __forceinline__ void next_b() { fb.next(q, q.b, q.pb, steps_in); }
    // What of k is there at an operand's step.
    template <class Side>
    __device__ __forceinline__ int64_t there(const Side& f, bool any) const {
        return any ? q.k - int64_t(steps_in - f.left) * STEP : 0;
    }

    // One step: the tiles a and b, whose first fragments are in xa and xb; B's next tile is loaded to to_b, A's after next
    // to to_a, and the first fragments of the next step's tiles are read from na and nb once they have arrived. They are
    // different buffers: told so, the compiler lets reads pass loads in flight.
    template <bool ENDS>
    __device__ __forceinline__ void step(LdsAt __restrict__ a, LdsAt __restrict__ b, LdsAt __restrict__ na,
                                         LdsAt __restrict__ nb, LdsAt __restrict__ to_a, LdsAt __restrict__ to_b,
                                         int64_t there_a, int64_t there_b, E8 (&xa)[F], E8 (&xb)[F], f32x16 (&acc)[F][F]) {
        E8 ya[F], yb[F];
#pragma unroll
        for (int part = 0; part < 4; part++) {
            E8(&ca)[F] = part & 1 ? ya : xa;
            E8(&cb)[F] = part & 1 ? yb : xb;
            E8(&da)[F] = part & 1 ? xa : ya;
            E8(&db)[F] = part & 1 ? xb : yb;
#pragma unroll
            for (int m = 0; m < F; m++) {
                if (part == 0) {
                    fb.template load<ENDS>(2 * m, there_b, to_b);
                    fb.template load<ENDS>(2 * m + 1, there_b, to_b);
                } else if (part < 3) {
                    fa.template load<ENDS>((part - 1) * F + m, there_a, to_a);
                }
                if (part < 3) {
                    da[m] = ra.template take<E8>(a, part + 1, m);
                    db[m] = rb.template take<E8>(b, part + 1, m);
                }
#pragma unroll
                for (int n = 0; n < F; n++) acc[m][n] = mfma(ca[m], cb[n], acc[m][n]);
                __builtin_amdgcn_sched_barrier(0);
                if (part == 3) {
                    if (m == 0) arrived<S::PARTS>();
                    da[m] = ra.template take<E8>(na, 0, m);
                    db[m] = rb.template take<E8>(nb, 0, m);
                }
            }
        }
        next_a();
        next_b();
    }

    // Steps lo .. hi of the product.
    __device__ __forceinline__ void run(LdsAt base, int wave, int lo, int hi, f32x16 (&acc)[F][F]) {
        const LdsAt base_b = base + A_BUFFERS * S::SIDE;
        const int mine = wave * S::PARTS * 1024;
        // steps whose loads are whole: the last of a segment may not be
        const int whole = q.segments == 1 ? min(hi, (int)(q.k / STEP)) : q.k % STEP == 0 ? hi : 0;
        auto load_a = [&](int s, LdsAt to) {
            const int64_t n = there(fa, s < hi);
#pragma unroll
            for (int k = 0; k < S::PARTS; k++) fa.template load<true>(k, n, to + mine);
            next_a();
        };
        load_a(lo, base);
        {
            const int64_t n = there(fb, true);
#pragma unroll
            for (int k = 0; k < S::PARTS; k++) fb.template load<true>(k, n, base_b + mine);
            next_b();
        }
        load_a(lo + 1, base + S::SIDE);
        arrived<S::PARTS>();
        E8 xa[F], xb[F];
#pragma unroll
        for (int m = 0; m < F; m++) {
            xa[m] = ra.template take<E8>(base, 0, m);
            xb[m] = rb.template take<E8>(base_b, 0, m);
        }
        LdsAt a = base, na = base + S::SIDE, to = base + 2 * S::SIDE, b = base_b, nb = base_b + S::SIDE;
        auto turn = [&] {
            const LdsAt was = a;
            a = na, na = to, to = was;
            const LdsAt old = b;
            b = nb, nb = old;
        };
        int s = lo;
        for (; s + 2 < whole; s++, turn()) step<false>(a, b, na, nb, to + mine, nb + mine, STEP, STEP, xa, xb, acc);
        // the last steps load zeros past the end: the count of loads in flight stays the same
        for (; s < hi; s++, turn())
            step<true>(a, b, na, nb, to + mine, nb + mine, there(fa, s + 2 < hi), there(fb, s + 1 < hi), xa, xb, acc);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    }
};

// What a product's epilogue sees: eight values of row i from column j, n of them in the matrix.
// Raw is what it reads for them, before, if reads().
//   struct Epilogue {
//       bool reads() const;
//       Raw raw(int batch, int64_t i, int64_t j, int n) const;
//       void operator()(const Raw&, int batch, int64_t i, int64_t j, int n, float (&v)[8]) const;
//   };
// MIRROR: symmetric results; the epilogue also gets columns as rows.
// Workgroup `block` of `total` of a product.
template <class E, int F, bool AI, bool BI, class Epilogue>
__device__ __forceinline__ void product(const Product& p, const Epilogue& epilogue, char* lds, unsigned block,
                                        unsigned total) {
    typedef TileShape<F> S;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // Workgroups go round the eight XCDs; consecutive tiles, which share panels of both operands, go to one XCD's cache.
    const unsigned per = total / 8;
    const int id = block < per * 8 ? (block % 8) * per + block / 8 : block;
    const int tiles = p.triangle ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
    const int batch = id / (tiles * p.runs), run = id / tiles - batch * p.runs, tile = id % tiles;
    int ti, tj;
    if (p.triangle) {
        // column tj has tiles 0 .. tj
        tj = (int)((sqrtf(8.f * tile + 1.f) - 1.f) * 0.5f);
        while (tj * (tj + 1) / 2 > tile) tj--;
        while ((tj + 1) * (tj + 2) / 2 <= tile) tj++;
        ti = tile - tj * (tj + 1) / 2;
    } else {
        // four rows of tiles at a time: 32 neighbouring workgroups share 4 + 8 panels
        const int band = tile / (4 * p.tiles_n), high = min(4, p.tiles_m - 4 * band), in = tile - band * 4 * p.tiles_n;
        ti = 4 * band + in % high, tj = in / high;
    }
    const int64_t i0 = int64_t(ti) * S::TILE, j0 = int64_t(tj) * S::TILE;
    const int lo = run * p.run_steps, hi = min(lo + p.run_steps, p.steps);

    f32x16 acc[F][F] = {};
    if (lo < hi) {
        Tiles<E, F, AI, BI> tiles_of(p, batch, i0, j0, wave, lane, lo);
        tiles_of.run((LdsAt)lds, wave, lo, hi, acc);
    }

    // Through LDS to whole rows: a lane has one column of sixteen rows, memory wants eight columns of one.
    constexpr int WIDE = 32 * F, PITCH = WIDE + 4, CHUNKS = WIDE / 8, ROWS = 64 / CHUNKS;
    static_assert(32 * PITCH * 4 <= S::LDS / 4, "a wavefront's fragments of 32 rows fit its part");
    float* mine = (float*)(lds + wave * (S::LDS / 4));
    const int64_t wi = i0 + (wave >> 1) * WIDE, wj = j0 + (wave & 1) * WIDE, m_all = p.a.outer, n_all = p.b.outer;
    float* part = p.runs > 1 ? p.part + (int64_t(run) * p.batches + batch) * m_all * n_all : nullptr;
    auto sync = [] {  // a wavefront's own: its LDS accesses stay in order, and the compiler keeps them so
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int m = 0; m < F; m++) {
#pragma unroll
        for (int n = 0; n < F; n++)
#pragma unroll
            for (int k = 0; k < 16; k++)
                mine[(8 * (k / 4) + 4 * (lane >> 5) + k % 4) * PITCH + 32 * n + (lane & 31)] = acc[m][n][k];
        sync();
        // What the epilogue reads for a few rows goes before the first of them is written; where it reads nothing, a row
        // at a time is faster (16,384 x 4,096 x 4,096: 464 and 497 us; with a residual 625 and 587).
        constexpr int TURNS = (32 + ROWS - 1) / ROWS, SOME = sizeof(typename Epilogue::Raw) > 16 && F > 2 ? 2 : 4,
                      AT_ONCE = TURNS < SOME ? TURNS : SOME;
        const int c = 8 * (lane % CHUNKS);
        const int64_t j = wj + c;
        const int have = (int)max<int64_t>(0, min<int64_t>(8, n_all - j));
        auto there = [&](int r) {
            return have > 0 && wi + 32 * m + r < m_all && !(64 % CHUNKS && (lane >= ROWS * CHUNKS || r >= 32));
        };
        auto values = [&](int r, float(&v)[8]) {
            const float4 lo4 = *(const float4*)(mine + r * PITCH + c), hi4 = *(const float4*)(mine + r * PITCH + c + 4);
            v[0] = lo4.x, v[1] = lo4.y, v[2] = lo4.z, v[3] = lo4.w, v[4] = hi4.x, v[5] = hi4.y, v[6] = hi4.z, v[7] = hi4.w;
        };
        if (!part && epilogue.reads()) {
            for (int it = 0; it < TURNS; it += AT_ONCE) {
                typename Epilogue::Raw raw[AT_ONCE] = {};
                const int r = it * ROWS + lane / CHUNKS;
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++)
                    if (there(r + u * ROWS)) raw[u] = epilogue.raw(batch, wi + 32 * m + r + u * ROWS, j, have);
#pragma unroll
                for (int u = 0; u < AT_ONCE; u++) {
                    if (!there(r + u * ROWS)) continue;
                    float v[8];
                    values(r + u * ROWS, v);
                    epilogue(raw[u], batch, wi + 32 * m + r + u * ROWS, j, have, v);
                }
            }
        } else {
            for (int it = 0; it < TURNS; it++) {
                const int r = it * ROWS + lane / CHUNKS;
                if (!there(r)) continue;
                float v[8];
                values(r, v);
                if (part) store_n(part + (wi + 32 * m + r) * n_all + j, have, v);
                else epilogue({}, batch, wi + 32 * m + r, j, have, v);
            }
        }
        if (Epilogue::MIRROR && p.triangle && ti != tj && !part) {
            // a row of the other half: 32 of i, eight a lane
            for (int it = 0; it < WIDE / 16; it++) {
                const int c = it * 16 + lane / 4, r = 8 * (lane % 4);
                const int64_t i = wj + c, j = wi + 32 * m + r;
                if (i >= n_all || j >= m_all) continue;
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; u++) v[u] = mine[(r + u) * PITCH + c];
                const int n = (int)min<int64_t>(8, m_all - j);
                epilogue(epilogue.raw(batch, i, j, n), batch, i, j, n, v);
            }
        }
        sync();
    }
}

template <class E, int F, bool AI, bool BI, class Epilogue>
__global__ __launch_bounds__(PRODUCT_BLOCK, F > 2 ? 1 : 2) void k_product(Product p, Epilogue epilogue) {
    __shared__ __align__(16) char lds[TileShape<F>::LDS];
    product<E, F, AI, BI>(p, epilogue, lds, blockIdx.x, gridDim.x);
}

// Two products that do not wait for each other in one launch: the first's workgroups, and the second's, whose operands both
// have rows on k.
template <class E, int F, bool BI, class Epilogue, class Second>
__global__ __launch_bounds__(PRODUCT_BLOCK, 2) void k_products(Product p, Epilogue epilogue, unsigned blocks, Product q,
                                                               Second second) {
    __shared__ __align__(16) char lds[TileShape<F>::LDS];
    if (blockIdx.x < blocks) product<E, F, true, BI>(p, epilogue, lds, blockIdx.x, blocks);
    else product<E, F, false, false>(q, second, lds, blockIdx.x - blocks, gridDim.x - blocks);
}

// The runs' partial products added, in an order that does not change: eight elements of a row a thread, a quarter of
// the runs each wavefront.
template <class Epilogue>
__device__ __forceinline__ void product_sum(const Product& p, int64_t chunks, const Epilogue& epilogue, int64_t block) {
    typedef float Eight __attribute__((ext_vector_type(8)));
    __shared__ Eight quarters[3][64];
    const int quarter = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t m = p.a.outer, n = p.b.outer, at = block * 64 + lane, per_row = (n + 7) / 8;
    const bool there = at < chunks;
    const int64_t row = at / per_row, j = (at - row * per_row) * 8;  // a row of all matrices
    const int have = (int)min<int64_t>(8, n - j);
    const int64_t i = row % m, batch = row / m;
    // a symmetric result's lower tiles are read from their mirror images
    const bool lower = p.triangle && i / p.triangle > j / p.triangle;
    Eight s = {};
    if (there) {
        const float* from = p.part + batch * m * n;
        const int64_t stride = int64_t(p.batches) * m * n;
        for (int k = quarter; k < p.runs; k += 4) {
            float v[8] = {};
            if (!lower) {
                load_n(from + k * stride + i * n + j, have, 0.f, v);
            } else {
                for (int u = 0; u < have; u++) v[u] = from[k * stride + (j + u) * n + i];
            }
#pragma unroll
            for (int u = 0; u < 8; u++) s[u] += v[u];
        }
    }
    if (quarter) quarters[quarter - 1][lane] = s;
    __syncthreads();
    if (quarter || !there) return;
    s = (s + quarters[0][lane]) + (quarters[1][lane] + quarters[2][lane]);
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = s[u];
    epilogue(epilogue.raw((int)batch, i, j, have), (int)batch, i, j, have, v);
}

template <class Epilogue>
__global__ __launch_bounds__(PRODUCT_BLOCK) void k_product_sum(Product p, int64_t chunks, Epilogue epilogue) {
    product_sum(p, chunks, epilogue, blockIdx.x);
}

// ---------------------------------------------------------------- the host's side

inline int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A launch holds fewer than 2^32 threads: 2^24 workgroups, and two products may share it. Tiles of 256 stay below
// this for any result that fits the memory.
constexpr int64_t MOST_TILES = int64_t(1) << 23;

// How a product is cut: tiles of 64 F, and runs along k.
struct Cut {
    int f, runs, run_steps, steps;
    int64_t tiles_m, tiles_n;
    bool triangle;

    // of the runs' partial products; n all matrices' elements
    size_t bytes(int64_t n) const { return runs > 1 ? size_t(runs) * n * 4 : 0; }
};

// What a round of workgroups costs, in microseconds: a step with so many workgroups a CU, and all else (the start, the
// first loads, the epilogue, the end). Measured on products of 1 to 2,048 tiles and 1 to 64 steps; a tile of 256 reaches
// 1.41 PFLOP/s in its steps on all CUs, one of 192 1.3, of 128 1.12, of 64 0.59, but costs 15 us beside them, 11, 7 and 4.
struct RoundCost {
    int most;            // workgroups a CU
    double step[4], fixed[4];
};
inline const RoundCost& round_cost(int f) {
    static const RoundCost cost[4] = {{4, {0.33, 0.51, 0.72, 0.91}, {4.0, 4.6, 5.3, 6.0}},
                                      {2, {0.57, 1.0}, {6.8, 8.5}},
                                      {1, {0.95}, {11.5}},
                                      {1, {1.52}, {15.5}}};
    return cost[f - 1];
}

inline Cut cut_of(int64_t m, int64_t n, int64_t k, int segments, int cus, int64_t batches = 1, bool triangle = false) {
    Cut best = {};
    double least = -1;
    const int64_t steps = (k + STEP - 1) / STEP * segments;
    for (int f = 4; f >= 1; f--) {
        const RoundCost& cost = round_cost(f);
        const int64_t tile = 64 * f, tm = (m + tile - 1) / tile, tn = (n + tile - 1) / tile,
                      tiles = std::max<int64_t>(1, batches * (triangle ? tm * (tm + 1) / 2 : tm * tn));
        if (f < 4 && tiles > MOST_TILES) break;
        const int64_t slots = int64_t(cost.most) * cus;
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(steps / 2, 4 * slots / tiles));
        for (int64_t r = 1; r <= 128; r = r < 8 ? r + 1 : r * 5 / 4) {
            if (r > most) break;
            const int64_t per = (steps + r - 1) / r, runs = per ? (steps + per - 1) / per : 1;
            const int64_t full = tiles * runs / slots, rest = tiles * runs % slots, beside = (rest + cus - 1) / cus;
            double t = double(full) * (double(per) * cost.step[cost.most - 1] + cost.fixed[cost.most - 1]);
            if (rest) t += double(per) * cost.step[beside - 1] + cost.fixed[beside - 1];
            // the runs' products written, read and added by a launch of its own
            if (runs > 1) t += 4.0 + double(runs) * batches * m * n * 8 / 4.5e6;
            if (least >= 0 && t >= least) continue;
            least = t;
            best.f = f;
            best.runs = (int)std::max<int64_t>(1, runs);
            best.run_steps = (int)per;
            best.steps = (int)steps;
            best.tiles_m = tm;
            best.tiles_n = tn;
            best.triangle = triangle;
        }
    }
    return best;
}

template <class E, int F, class Epilogue>
void product_of(const Product& p, bool ai, bool bi, const Epilogue& e, hipStream_t s) {
    const int tiles = p.triangle ? p.tiles_m * (p.tiles_m + 1) / 2 : p.tiles_m * p.tiles_n;
    const dim3 grid((uint32_t)(tiles * p.runs * p.batches));
    if (ai && bi) k_product<E, F, true, true><<<grid, PRODUCT_BLOCK, 0, s>>>(p, e);
    else if (ai) k_product<E, F, true, false><<<grid, PRODUCT_BLOCK, 0, s>>>(p, e);
    else k_product<E, F, false, false><<<grid, PRODUCT_BLOCK, 0, s>>>(p, e);
}

// a, b, k, segments and batches are set.
inline Product cut_product(Product p, const Cut& cut, float* part) {
    p.tiles_m = (int)cut.tiles_m;
    p.tiles_n = (int)cut.tiles_n;
    p.runs = cut.runs;
    p.run_steps = cut.run_steps;
    p.steps = cut.steps;
    p.triangle = cut.triangle ? 64 * cut.f : 0;
    p.part = part;
    return p;
}
inline int64_t sum_chunks(const Product& p) { return p.batches * p.a.outer * ((p.b.outer + 7) / 8); }

template <class E, class Epilogue>
void launch_product(Product p, const Cut& cut, bool ai, bool bi, float* part, const Epilogue& e, hipStream_t s) {
    p = cut_product(p, cut, part);
    if (cut.f == 4) product_of<E, 4>(p, ai, bi, e, s);
    else if (cut.f == 3) product_of<E, 3>(p, ai, bi, e, s);
    else if (cut.f == 2) product_of<E, 2>(p, ai, bi, e, s);
    else product_of<E, 1>(p, ai, bi, e, s);
    if (cut.runs > 1)
        k_product_sum<<<dim3((uint32_t)((sum_chunks(p) + 63) / 64)), PRODUCT_BLOCK, 0, s>>>(p, sum_chunks(p), e);
}

}  // namespace
}  // namespace learn
}  // namespace wc
