// The weight gradient from activations kept in 8 bits, on the matrix cores (include/wc_learn.h).
//
// weight[i][j] = sum over rows r of a[r][i] g[r][j]: both operands have the
// summed index outermost, while a matrix instruction takes several values of
// it from one lane. Tiles go to LDS as they lie in memory, the 8-bit one
// expanded to the 16-bit type on the way, and come back through the transposing
// LDS read (four rows of sixteen columns become four values of one column per
// lane). A workgroup of four wavefronts owns a square tile of weight, each
// wavefront a quarter in its accumulators; two LDS buffers alternate, the next
// tile's global loads in registers meanwhile. Where the tiles are too few for
// the device the rows are cut into runs, whose partial products are added in
// order.
//
// On one MI355X: 512 x 384 over 49,371 rows 39 us (k_weight, 492 workgroups of
// which 41 share a tile) and 7 to add the runs; floor 17 us at the 1,142 TFLOP/s
// of a large library product. A step of 64 rows takes 1.45 us with two workgroups
// a CU, of which the matrix instructions are 0.42, arithmetic 0.4 and LDS 0.5 (a
// third of the cycles wait on barriers and counters). 4,096 x 4,096 over 16,384
// rows with GELU: 39 us to expand and 477 us (k_weight_big, 1.15 PFLOP/s); the
// library's product of the same 16-bit operands takes 559.
//
// A recomputed GELU or SiLU is rounded to the gradient's 16-bit type, whatever the
// result's: one matrix instruction a product instead of two. Half an ulp of the
// activation (2^-9 of it in bf16) is less than the 8 bits' own half step, 1/254 to
// 1/127 of the group's largest. Over 16,384 rows the sums are off by 1.5e-3 of their
// norm by it; a bf16 result's own rounding is 1.7e-3, both together 2.2e-3.
//
// A float32 gradient is three passes of k_weight over the rows, one step of loads
// ahead: 512 x 384 over 49,371 rows 133 us and 7 to add the runs (three bf16 products
// at the library's rate: 51), 4,096 x 4,096 over 16,384 rows 3,650 us (1,443).
#include <algorithm>

#include "ckpt8_dev.h"

namespace wc {
namespace learn {
namespace {

constexpr int BLOCK = 256;
constexpr int DEPTH = 64;  // rows per step

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// A lane's eight rows of a column added to s.
__device__ __forceinline__ float plus(bf16x8 v, float s) {
    typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{v[i], v[i + 1]}, one, s, false);
    return s;
}
__device__ __forceinline__ float plus(f16x8 v, float s) {
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(f16)1.f, (f16)1.f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) s = __builtin_amdgcn_fdot2(f16x2{v[i], v[i + 1]}, one, s, false);
    return s;
}

// The operand's type and how many parts a gradient element is taken in: a
// float32 is the sum of three bf16 (8 + 8 + 8 mantissa bits), whose products
// with a kept value (8 bits) are exact. The parts are three passes over the rows.
template <class T>
struct Operand {
    typedef T type;
    static constexpr int PARTS = 1;
};
template <>
struct Operand<float> {
    typedef bf16 type;
    static constexpr int PARTS = 3;
};

// The first of a float32's three parts is its upper half: cut, not rounded, so
// that a value past bf16's largest does not become infinite. (The mark of a quiet
// NaN, as arithmetic leaves it, is in that half too.)
__device__ __forceinline__ float cut(float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); }

// One of the three parts of eight values. What an infinity leaves is 0, not
// infinity less infinity: its products are infinite through the first part alone.
__device__ __forceinline__ bf16x8 part_of(const Vec8<float>::type& v, int part) {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float x = v[i];
        if (part > 0) {
            x -= cut(x);
            x = x == x ? x : 0.f;
        }
        if (part > 1) x -= cut(x);
        u[i] = __float_as_uint(x);
    }
    Words w;
#pragma unroll
    for (int i = 0; i < 4; i++) w[i] = __builtin_amdgcn_perm(u[2 * i + 1], u[2 * i], 0x07060302);  // both upper halves
    return __builtin_bit_cast(bf16x8, w);
}

// One tile: 2 x 2 wavefronts of F x F fragments of 32 x 32.
template <int F>
struct Shape {
    static constexpr int TILE = 64 * F;
    // Bytes from one row of a tile to the next. A transposing read takes 64 bytes
    // of four consecutive rows: row r's 64-byte units are exchanged by r modulo 4,
    // so that they lie in different banks.
    static constexpr int PITCH = 2 * TILE;
    static constexpr int A_CHUNKS = DEPTH * TILE / 16 / BLOCK;  // 16 kept values each
    static constexpr int B_CHUNKS = DEPTH * TILE / 8 / BLOCK;   // 8 gradient values each
};

struct Job {
    wc_ckpt_weight_args a;
    int64_t run;        // rows per run, a multiple of DEPTH
    int64_t open;       // the rows after which there is room for loads past a row's end
    int tiles_i, tiles_j, runs;
    float* part;        // runs x width x out, where there are several runs
    float* bias_part;   // runs x out, likewise
};

// Sixteen kept values of one row.
struct Kept {
    uint32_t q[4], e;
};

// From column c; zeros beyond the rows and the row.
__device__ __forceinline__ Kept load_kept(const wc_ckpt_weight_args& a, int64_t r, int64_t hi, int64_t c) {
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(1)));
    Kept k = {{0, 0, 0, 0}, 1};
    if (r < hi && c < a.width) {
        const int8_t* p = a.q + r * a.q_stride + c;
        k.e = a.exps[r * a.exps_stride + (c >> 5)];
        if (c + 16 <= a.width) {
            const Words w = *(const Words*)p;
#pragma unroll
            for (int i = 0; i < 4; i++) k.q[i] = w[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++)
                if (c + i < a.width) k.q[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
        }
    }
    return k;
}

// All of them there.
__device__ __forceinline__ Kept load_kept(const int8_t* q, const uint8_t* e) {
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(1)));
    const Words w = *(const Words*)q;
    return {{w[0], w[1], w[2], w[3]}, *e};
}

// Eight of them, in 16 bits.
template <class E>
struct Eight {
    typedef E type __attribute__((ext_vector_type(8)));
};
template <class E>
__device__ __forceinline__ typename Eight<E>::type expand(const Kept& k, const int act, int half) {
    const float step = step_of(k.e);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)(int8_t)(k.q[2 * half + (i >> 2)] >> (8 * (i & 3))) * step;
    if (may_pass<E>(k.e)) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = held<E>(v[i]);
    }
    act_values(v, act);
    typename Eight<E>::type o;
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = (E)v[i];
    return o;
}

// Eight gradient values of one row, from column c; zeros beyond the rows and the row.
template <class T>
__device__ __forceinline__ typename Vec8<T>::type load_grad(const wc_ckpt_weight_args& a, int64_t r, int64_t hi,
                                                            int64_t c) {
    typename Vec8<T>::type v = {};
    if (r < hi && c < a.out) {
        const T* p = (const T*)a.grad + r * a.grad_stride + c;
        if (c + 8 <= a.out) {
            v = *(const typename Vec8<T>::type*)p;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (c + i < a.out) v[i] = p[i];
        }
    }
    return v;
}

// A fragment's eight values for the lane: rows k0 + 8 (lane / 32) .. + 7 of
// column c0 + lane % 32, by two transposing reads of four rows.
template <class E8, int PITCH>
__device__ __forceinline__ E8 fragment(const char* tile, int k0, int c0, int lane) {
    typedef __attribute__((address_space(3))) s16x4* Lds;
    const int row = (lane & 15) >> 2;
    const char* p = tile + (k0 + 8 * (lane >> 5) + row) * PITCH + ((2 * (c0 + (lane & 16) + 4 * (lane & 3))) ^ (row << 6));
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * PITCH));
    return __builtin_bit_cast(E8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// What a workgroup of k_weight works on.
struct Tile {
    int64_t i0, j0, lo, hi, open;
    bool sums;
};

// The tile's products, and with `sums` the gradient's column sums, of half a
// fragment's rows a lane, by the wavefronts of the tile's first half.
//
// All steps but the last loads unchecked: where the tile reaches past the last
// column a lane loads columns before it, or past the row's end the next row's
// first bytes, and the products of what is no column are not stored. The last
// rows of all, after which nothing need follow, and a step that is not whole go
// through checked loads at the end. (Checks in the loop would be loads that the
// compiler cannot count, and so waits for at once; and several kilobytes of
// code that every workgroup would fetch.)
template <class T, int F, int ACT>
__device__ __forceinline__ void products(const wc_ckpt_weight_args& a, const Tile& tile, char* lds, f32x16 (&acc)[F][F],
                                         float (&bias)[F]) {
    typedef typename Operand<T>::type E;
    typedef E E8 __attribute__((ext_vector_type(8)));
    typedef Shape<F> S;
    constexpr int PARTS = Operand<T>::PARTS, TILE = S::TILE, PITCH = S::PITCH, SIDE = DEPTH * PITCH;
    constexpr int AR = BLOCK / (TILE / 16), BR = BLOCK / (TILE / 8);
    static_assert(AR % 4 == 0 && BR % 4 == 0, "a thread's rows have one place modulo 4");
    static_assert(DEPTH / 16 == S::B_CHUNKS && S::B_CHUNKS == 2 * S::A_CHUNKS, "four parts");
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int ac = (t % (TILE / 16)) * 16, ar = t / (TILE / 16);
    const int bc = (t % (TILE / 8)) * 8, br = t / (TILE / 8);
    const int wi = (wave >> 1) * 32 * F, wj = (wave & 1) * 32 * F;
    const int64_t lo = tile.lo, hi = tile.hi;
    const int whole = (int)(max<int64_t>(0, min(hi, tile.open) - lo) / DEPTH), all = whole * PARTS;

    // Loads of the next AHEAD steps wait in registers: a step is shorter than a load takes.
    constexpr int AHEAD = sizeof(T) == 2 ? 3 : 1;
    struct Loads {
        Kept a[S::A_CHUNKS];
        typename Vec8<T>::type g[S::B_CHUNKS];
    } ahead[AHEAD];
    const int64_t ca = min(tile.i0 + ac, (a.width - 1) / 16 * 16), cb = min(tile.j0 + bc, (a.out - 1) / 8 * 8);
    const int8_t* q0 = a.q + (lo + ar) * a.q_stride + ca;
    const uint8_t* e0 = a.exps + (lo + ar) * a.exps_stride + (ca >> 5);
    const T* g0 = (const T*)a.grad + (lo + br) * a.grad_stride + cb;
    auto first_row = [&](int s) {
        s = min(s, all - 1);  // past the end the last step's again: the count of loads stays the same
        return int64_t(PARTS == 1 ? s : s % whole) * DEPTH;
    };
    auto load_a = [&](Loads& l, int m, int64_t r0) {
        l.a[m] = load_kept(q0 + (r0 + m * AR) * a.q_stride, e0 + (r0 + m * AR) * a.exps_stride);
    };
    auto load_g = [&](Loads& l, int m, int64_t r0) {
        l.g[m] = *(const typename Vec8<T>::type*)(g0 + (r0 + m * BR) * a.grad_stride);
    };
    // A step's loads and LDS writes are in four parts, between its matrix instructions:
    // part k has chunk k of the gradient and half a chunk of the kept values.
    auto put = [&](const Loads& l, int k, char* to, int plane) {
        E8* p = (E8*)(to + (ar + k / 2 * AR) * PITCH + ((2 * ac) ^ ((ar & 3) << 6)));
        p[k % 2] = expand<E>(l.a[k / 2], ACT, k % 2);
        E8 o;
        if constexpr (PARTS == 1) {
            o = l.g[k];
        } else {
            o = part_of(l.g[k], plane);
        }
        *(E8*)(to + SIDE + (br + k * BR) * PITCH + ((2 * bc) ^ ((br & 3) << 6))) = o;
    };
    E8 fa[2][F], fb[2][F];
    auto take = [&](const char* from, int k) {
#pragma unroll
        for (int m = 0; m < F; m++) fa[k & 1][m] = fragment<E8, PITCH>(from, 16 * k, wi + 32 * m, lane);
#pragma unroll
        for (int n = 0; n < F; n++) fb[k & 1][n] = fragment<E8, PITCH>(from + SIDE, 16 * k, wj + 32 * n, lane);
    };
    auto multiply = [&](int k) {
#pragma unroll
        for (int m = 0; m < F; m++)
#pragma unroll
            for (int n = 0; n < F; n++) acc[m][n] = mfma(fa[k & 1][m], fb[k & 1][n], acc[m][n]);
        if (tile.sums && wi == 0) {
#pragma unroll
            for (int n = 0; n < F; n++) bias[n] = plus(fb[k & 1][n], bias[n]);
        }
    };

    if (all > 0) {
        auto load = [&](Loads& l, int s) {
            const int64_t r0 = first_row(s);
#pragma unroll
            for (int m = 0; m < S::A_CHUNKS; m++) load_a(l, m, r0);
#pragma unroll
            for (int m = 0; m < S::B_CHUNKS; m++) load_g(l, m, r0);
        };
        load(ahead[0], 0);
#pragma unroll
        for (int k = 0; k < 4; k++) put(ahead[0], k, lds, 0);
#pragma unroll
        for (int k = 0; k < AHEAD; k++) load(ahead[k], 1 + k);
        __syncthreads();
        for (int s0 = 0; s0 < all; s0 += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                const int s = s0 + u;
                if (s >= all) break;
                const char* from = lds + (s & 1) * 2 * SIDE;
                char* to = lds + (s + 1 & 1) * 2 * SIDE;
                const int64_t r0 = first_row(s + 1 + AHEAD);
                take(from, 0);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (k < 3) take(from, k + 1);
                    put(ahead[u], k, to, PARTS == 1 ? 0 : (s + 1) / whole);
                    if (k % 2) load_a(ahead[u], k / 2, r0);
                    load_g(ahead[u], k, r0);
                    multiply(k);
                }
                __syncthreads();
            }
        }
    }
    // what is left
    for (int64_t r0 = lo + int64_t(whole) * DEPTH; r0 < hi; r0 += DEPTH) {
        Loads& l = ahead[0];
#pragma unroll
        for (int m = 0; m < S::A_CHUNKS; m++) l.a[m] = load_kept(a, r0 + ar + m * AR, hi, tile.i0 + ac);
#pragma unroll
        for (int m = 0; m < S::B_CHUNKS; m++) l.g[m] = load_grad<T>(a, r0 + br + m * BR, hi, tile.j0 + bc);
        for (int plane = 0; plane < PARTS; plane++) {
#pragma unroll
            for (int k = 0; k < 4; k++) put(l, k, lds, plane);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                take(lds, k);
                multiply(k);
            }
            __syncthreads();
        }
    }
}

template <class T, int F, int ACT>
__global__ __launch_bounds__(BLOCK, 2) void k_weight(Job job) {
    typedef Shape<F> S;
    constexpr int TILE = S::TILE;
    __shared__ __align__(16) char lds[4 * DEPTH * S::PITCH];  // two buffers of a tile of each operand
    const wc_ckpt_weight_args& a = job.a;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // Workgroups go round the eight XCDs; consecutive tiles of a run, which share
    // rows of both operands, go to one XCD's cache.
    const int total = job.tiles_i * job.tiles_j * job.runs, per = total / 8;
    const int id = blockIdx.x < (unsigned)per * 8 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
    const int run = id / (job.tiles_i * job.tiles_j), at = id - run * (job.tiles_i * job.tiles_j);
    Tile tile;
    tile.i0 = int64_t(at % job.tiles_i) * TILE;
    tile.j0 = int64_t(at / job.tiles_i) * TILE;
    tile.lo = run * job.run;
    tile.hi = min(tile.lo + job.run, a.rows);
    tile.open = job.open;
    tile.sums = a.bias && tile.i0 == 0;
    f32x16 acc[F][F] = {};
    float bias[F] = {};
    if (tile.lo < tile.hi) products<T, F, ACT>(a, tile, lds, acc, bias);
    const int wi = (wave >> 1) * 32 * F, wj = (wave & 1) * 32 * F;
    const int64_t i0 = tile.i0, j0 = tile.j0;

    const bool last = job.runs == 1;
    float* part = job.part + int64_t(run) * a.width * a.out;
#pragma unroll
    for (int m = 0; m < F; m++)
#pragma unroll
        for (int n = 0; n < F; n++)
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const int64_t i = i0 + wi + 32 * m + 8 * (k / 4) + 4 * (lane >> 5) + k % 4, j = j0 + wj + 32 * n + (lane & 31);
                if (i >= a.width || j >= a.out) continue;
                if (!last) part[i * a.out + j] = acc[m][n][k];
                else if (a.weight_dtype == WC_DTYPE_F32) ((float*)a.weight)[i * a.weight_stride + j] = acc[m][n][k];
                else ((T*)a.weight)[i * a.weight_stride + j] = (T)acc[m][n][k];
            }
    if (tile.sums && wi == 0) {  // a column's rows are in two lanes
#pragma unroll
        for (int n = 0; n < F; n++) {
            const float s = bias[n] + __shfl_xor(bias[n], 32);
            const int64_t j = j0 + wj + 32 * n + lane;
            if (lane < 32 && j < a.out) (last ? a.bias : job.bias_part + int64_t(run) * a.out)[j] = s;
        }
    }
}

// --------------------------------------------------- large products, 16-bit

// Both operands in 16 bits with rows on 16 bytes: the kept values expanded once
// (an activation recomputed for every column tile would cost more than the
// products), the gradient as it is or copied. 256 x 256 tiles, four wavefronts
// of 128 x 128; tiles go from memory to LDS without passing registers, four
// buffers of 32 rows, three of them in flight. With a wait for all loads in each
// step, and these in one block before the matrix instructions, it took 663 us
// where it takes 477.
constexpr int BIG = 256, BIG_DEPTH = 32, BIG_ROW = 2 * BIG, BIG_SIDE = BIG_DEPTH * BIG_ROW, BUFFERS = 4;

static __device__ __align__(16) uint4 g_zeros;  // what rows past the end are read from

struct BigJob {
    Job job;
    const char* x;     // rows x width, x_pitch bytes a row
    const char* g;     // rows x out, g_pitch bytes a row
    int64_t x_pitch, g_pitch;
};

// LDS as the large product addresses it.
typedef __attribute__((address_space(3))) char* Lds;

// One wavefront's share of a step's tiles, from memory to LDS: eight rows of
// each, in four parts of two. A load's 64 lanes bring 16 bytes each to places
// in LDS that follow each other. A transposing read takes 64 bytes of four
// consecutive rows: so that they lie in different banks, row r's 64-byte units
// are exchanged by r modulo 4, by which lane loads what.
struct Fetch {
    const char *x, *g;  // the wavefront's first row: the same for all lanes
    int64_t x_pitch, g_pitch, rows;
    uint32_t ox[2], og[2];  // the lane's place in two rows, for the even parts and the odd ones
    int half;

    // ENDS: rows past the end are read from zeros.
    template <bool ENDS>
    __device__ __forceinline__ void part(int s, int m, Lds to) const {
        const int64_t r0 = int64_t(s) * BIG_DEPTH + 2 * m;
        const char* fx = x + r0 * x_pitch;
        const char* fg = g + r0 * g_pitch;
        if (ENDS) {
            const bool there = r0 + half < rows;
            load(there ? fx + ox[m & 1] : (const char*)&g_zeros, to + 2 * m * BIG_ROW);
            load(there ? fg + og[m & 1] : (const char*)&g_zeros, to + BIG_SIDE + 2 * m * BIG_ROW);
        } else {
            load(fx + ox[m & 1], to + 2 * m * BIG_ROW);
            load(fg + og[m & 1], to + BIG_SIDE + 2 * m * BIG_ROW);
        }
    }
    static __device__ __forceinline__ void load(const char* from, Lds to) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                         (__attribute__((address_space(3))) void*)to, 16, 0, 0);
    }
};

// Sixteen rows of a buffer: one fragment of each operand.
template <class E8>
__device__ __forceinline__ void take(Lds from, int at, int wi, int wj, E8& fa, E8& fb) {
    typedef __attribute__((address_space(3))) s16x4* Lds4;
    const Lds pa = from + at + 2 * wi, pb = from + at + 2 * wj + BIG_SIDE;
    const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)pa);
    const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(pa + 4 * BIG_ROW));
    const s16x4 b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)pb);
    const s16x4 b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds4)(pb + 4 * BIG_ROW));
    fa = __builtin_bit_cast(E8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
    fb = __builtin_bit_cast(E8, __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Of the 24 loads that three buffers take, the first 8 have arrived when 16 are left.
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(16) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
}

// One step: the buffer `from`, whose first fragments are in fa and fb, and the
// first of `next`; the loads of three steps on go to `to`. The three are
// different buffers: told so, the compiler lets reads pass loads in flight.
// Everything else goes between the matrix instructions, which take 32 cycles
// each: four of them, then the loads and reads of one part.
template <class E8, bool SUMS, bool ENDS>
__device__ __forceinline__ void step(Lds __restrict__ from, Lds __restrict__ next, Lds __restrict__ to,
                                     const Fetch& fetch, int s, const int (&at)[4], int wi, int wj, E8 (&fa)[4],
                                     E8 (&fb)[4], f32x16 (&acc)[4][4], float (&bias)[4]) {
    E8 na[4], nb[4];
#pragma unroll
    for (int m = 0; m < 4; m++) {
        fetch.part<ENDS>(s + 3, m, to);
        take(from + 16 * BIG_ROW, at[m], wi, wj, na[m], nb[m]);
#pragma unroll
        for (int n = 0; n < 4; n++) acc[m][n] = mfma(fa[m], fb[n], acc[m][n]);
        if (SUMS) bias[m] = plus(fb[m], bias[m]);
        __builtin_amdgcn_sched_barrier(0);
    }
    E8 oa[4], ob[4];
#pragma unroll
    for (int m = 0; m < 4; m++) {
#pragma unroll
        for (int n = 0; n < 4; n++) acc[m][n] = mfma(na[m], nb[n], acc[m][n]);
        if (SUMS) bias[m] = plus(nb[m], bias[m]);
        __builtin_amdgcn_sched_barrier(0);
        if (m == 0) arrived();  // the next buffer's, and every wavefront has read this one's
        take(next, at[m], wi, wj, oa[m], ob[m]);
    }
#pragma unroll
    for (int m = 0; m < 4; m++) fa[m] = oa[m], fb[m] = ob[m];
}

template <class E8, bool SUMS>
__device__ __forceinline__ void steps_of(Lds base, const Fetch& fetch, Lds mine, int64_t rows, const int (&at)[4],
                                         int wi, int wj, f32x16 (&acc)[4][4], float (&bias)[4]) {
    const int whole = (int)(rows / BIG_DEPTH), steps = (int)((rows + BIG_DEPTH - 1) / BIG_DEPTH);
    E8 fa[4], fb[4];
    for (int s = 0; s < 3; s++)
#pragma unroll
        for (int m = 0; m < 4; m++) fetch.part<true>(s, m, mine + s * 2 * BIG_SIDE);
    arrived();
#pragma unroll
    for (int m = 0; m < 4; m++) take(base, at[m], wi, wj, fa[m], fb[m]);
    int s = 0;
    for (; s + 3 < whole; s++)
        step<E8, SUMS, false>(base + (s & 3) * 2 * BIG_SIDE, base + (s + 1 & 3) * 2 * BIG_SIDE,
                              mine + (s + 3 & 3) * 2 * BIG_SIDE, fetch, s, at, wi, wj, fa, fb, acc, bias);
    // the last steps load zeros past the end: the count of loads in flight stays the same
    for (; s < steps; s++)
        step<E8, SUMS, true>(base + (s & 3) * 2 * BIG_SIDE, base + (s + 1 & 3) * 2 * BIG_SIDE,
                             mine + (s + 3 & 3) * 2 * BIG_SIDE, fetch, s, at, wi, wj, fa, fb, acc, bias);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// W: what is written, the weights' type or a run's float32 products.
template <class E, class W>
__global__ __launch_bounds__(BLOCK, 1) void k_weight_big(BigJob big) {
    typedef E E8 __attribute__((ext_vector_type(8)));
    __shared__ __align__(16) char lds[BUFFERS * 2 * BIG_SIDE];
    const Job& job = big.job;
    const wc_ckpt_weight_args& a = job.a;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles = job.tiles_i * job.tiles_j, per = tiles * job.runs / 8;
    const int id = blockIdx.x < (unsigned)per * 8 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
    const int run = id / tiles, tile = id - run * tiles;
    // four rows of tiles at a time: 32 neighbouring workgroups share 4 + 8 panels
    const int band = tile / (4 * job.tiles_j), high = min(4, job.tiles_i - 4 * band), in = tile - band * 4 * job.tiles_j;
    const int ti = 4 * band + in % high, tj = in / high;
    const int64_t i0 = int64_t(ti) * BIG, j0 = int64_t(tj) * BIG;
    const int64_t lo = run * job.run, hi = min(lo + job.run, a.rows);

    Fetch fetch;
    const int64_t first = lo + wave * 8;
    fetch.x = big.x + first * big.x_pitch + 2 * i0;
    fetch.g = big.g + first * big.g_pitch + 2 * j0;
    fetch.x_pitch = big.x_pitch;
    fetch.g_pitch = big.g_pitch;
    fetch.rows = hi - first;
    fetch.half = lane >> 5;
#pragma unroll
    for (int odd = 0; odd < 2; odd++) {
        const int chunk = (lane & 31) ^ ((2 * odd + (lane >> 5)) << 2);
        // past the last column any column will do: its products are not stored
        fetch.ox[odd] = (uint32_t)(fetch.half * big.x_pitch) + (i0 + 8 * chunk < a.width ? 16 * chunk : 0);
        fetch.og[odd] = (uint32_t)(fetch.half * big.g_pitch) + (j0 + 8 * chunk < a.out ? 16 * chunk : 0);
    }

    const int wi = (wave >> 1) * 128, wj = (wave & 1) * 128;
    const int row = 8 * (lane >> 5) + ((lane & 15) >> 2), turn = ((lane & 15) >> 2) << 6;
    int at[4];
#pragma unroll
    for (int m = 0; m < 4; m++) at[m] = row * BIG_ROW + ((64 * m + 2 * ((lane & 16) + 4 * (lane & 3))) ^ turn);

    f32x16 acc[4][4] = {};
    float bias[4] = {};
    const bool sums = a.bias && ti == 0 && wi == 0;
    const Lds base = (Lds)lds, mine = base + wave * 8 * BIG_ROW;
    if (sums) steps_of<E8, true>(base, fetch, mine, max<int64_t>(hi - lo, 0), at, wi, wj, acc, bias);
    else steps_of<E8, false>(base, fetch, mine, max<int64_t>(hi - lo, 0), at, wi, wj, acc, bias);

    const bool last = job.runs == 1;
    const int64_t stride = last ? a.weight_stride : a.out;
    W* to = last ? (W*)a.weight : (W*)(job.part + int64_t(run) * a.width * a.out);
    const int64_t i1 = i0 + wi + 4 * (lane >> 5), j1 = j0 + wj + (lane & 31);
    to += i1 * stride + j1;
#pragma unroll
    for (int m = 0; m < 4; m++)
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const int di = 32 * m + 8 * (k / 4) + k % 4;
#pragma unroll
            for (int n = 0; n < 4; n++)
                if (i1 + di < a.width && j1 + 32 * n < a.out) to[di * stride + 32 * n] = (W)acc[m][n][k];
        }
    if (sums) {  // a column's rows are in two lanes
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const float s = bias[n] + __shfl_xor(bias[n], 32);
            const int64_t j = j0 + wj + 32 * n + lane;
            if (lane < 32 && j < a.out) (last ? a.bias : job.bias_part + int64_t(run) * a.out)[j] = s;
        }
    }
}

// What the large product reads: act(kept) in 16 bits, rows of `pitch` elements.
template <class E>
__global__ __launch_bounds__(BLOCK) void k_expand(wc_ckpt_weight_args a, E* to, int64_t pitch, int64_t per_row) {
    typedef E E8 __attribute__((ext_vector_type(8)));
    const int64_t total = a.rows * per_row;
    for (int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x; i < total; i += int64_t(gridDim.x) * BLOCK) {
        const int64_t r = i / per_row, c = (i - r * per_row) * 16;
        const Kept k = load_kept(a, r, a.rows, c);
        E8* p = (E8*)(to + r * pitch + c);
        p[0] = expand<E>(k, a.act, 0);
        p[1] = expand<E>(k, a.act, 1);
    }
}

// A gradient whose rows do not start on 16 bytes, copied to rows that do.
template <class T>
__global__ __launch_bounds__(BLOCK) void k_align(wc_ckpt_weight_args a, T* to, int64_t pitch, int64_t per_row) {
    const int64_t total = a.rows * per_row;
    for (int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x; i < total; i += int64_t(gridDim.x) * BLOCK) {
        const int64_t r = i / per_row, c = (i - r * per_row) * 8;
        *(typename Vec8<T>::type*)(to + r * pitch + c) = load_grad<T>(a, r, a.rows, c);
    }
}

// The runs' partial products added, in an order that does not change: N
// elements a thread, a quarter of the runs each wavefront. The workgroups past
// the weights' add the bias's.
template <class W, int N>
__global__ __launch_bounds__(BLOCK) void k_weight_sum(Job job, int64_t weight_blocks) {
    typedef float Some __attribute__((ext_vector_type(N)));
    __shared__ Some quarters[BLOCK / 64][64];
    const wc_ckpt_weight_args& a = job.a;
    const bool bias = blockIdx.x >= weight_blocks;
    const int quarter = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t n = bias ? a.out : a.width * a.out, block = blockIdx.x - (bias ? weight_blocks : 0);
    const int64_t i = (block * 64 + lane) * N;
    const float* part = (bias ? job.bias_part : job.part) + i;
    Some s = {};
    if (i < n) {
        int k = quarter;
        for (; k + 28 < job.runs; k += 32) {
            Some v[8];
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] = *(const Some*)(part + (k + 4 * u) * n);
#pragma unroll
            for (int u = 0; u < 8; u++) s += v[u];
        }
        for (; k < job.runs; k += 4) s += *(const Some*)(part + k * n);
    }
    quarters[quarter][lane] = s;
    __syncthreads();
    if (quarter || i >= n) return;
    s = (s + quarters[1][lane]) + (quarters[2][lane] + quarters[3][lane]);
#pragma unroll
    for (int u = 0; u < N; u++) {
        const float v = s[u];
        if (bias) a.bias[i + u] = v;
        else ((W*)a.weight)[(i + u) / a.out * a.weight_stride + (i + u) % a.out] = (W)v;
    }
}

// Which kernel, its tiles and runs, and where its scratch lies.
struct Plan {
    bool big;
    int tiles_i, tiles_j, runs;
    int64_t run;
    bool copy;             // big: the gradient is copied to aligned rows
    int64_t xp, gp;        // big: elements from row to row
    size_t x, g, part, bias, bytes;
};

// Microseconds that a product takes, from measured parts: a step of a round of
// workgroups (alone on their CUs, or two to a CU), a round's start and end, the
// runs' products written and read, and what the large product's operands cost
// to lay out. Both kernels over 1 to 128 runs at fifteen shapes: the pick was
// the best of all at thirteen, 7 and 15% above it at two. For instance 512 x 384 x
// 49,371: small 45 us, large 61; with GELU 65 and 61; 4,096 x 4,096 x 16,384:
// small 728, large 484; 1,024 x 1,024 x 8,192: 43 and 51; 300 x 200 x 1,000: 16
// in eight runs, 24 in one.
Plan plan_of(const wc_ckpt_weight_args& a, int cus) {
    Plan best = {};
    double least = -1;
    // (a lane's offset in two rows is held in 32 bits)
    const bool aligned = a.out % 8 == 0 && a.grad_stride % 8 == 0 && ((uintptr_t)a.grad & 15) == 0 &&
                         a.grad_stride < (1 << 29);
    const bool value = a.act == WC_ACT_GELU || a.act == WC_ACT_SILU;
    for (int big = 0; big < 2; big++) {
        if (big && a.dtype == WC_DTYPE_F32) continue;
        const int tile = big ? BIG : Shape<2>::TILE, depth = big ? BIG_DEPTH : DEPTH;
        const int64_t ti = (a.width + tile - 1) / tile, tj = (a.out + tile - 1) / tile, tiles = ti * tj;
        const int64_t steps = std::max<int64_t>(1, (a.rows + depth - 1) / depth), slots = big ? cus : 2 * cus;
        const double one = big ? 0.8 : value ? 1.55 : 0.97, two = big ? 0.8 : value ? 2.6 : 1.58;
        const double lay = big ? 4.0 + double(a.rows) * a.width * 3 / 5e6 +
                                     (aligned ? 0.0 : 4.0 + double(a.rows) * a.out * 4 / 5e6)
                               : 0.0;
        // runs that fill one to eight times the device's CUs, a few, or as many as leave each a few steps
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(steps / (big ? 4 : 2), 4 * slots / tiles));
        for (int k = -3; k <= 8; k++) {
            const int64_t runs = std::min(most, std::max<int64_t>(1, k == 0 ? most : k < 0 ? -k : k * cus / tiles));
            const int64_t per = (steps + runs - 1) / runs, full = tiles * runs / slots, rest = tiles * runs % slots;
            const double t = lay + double(full) * (double(per) * two + 4.0) +
                             (rest ? double(per) * (rest <= cus ? one : two) + 4.0 : 0.0) +
                             (runs > 1 ? 4.0 + double(runs) * a.width * a.out * 8 / 9e6 : 0.0);
            if (least >= 0 && t >= least) continue;
            least = t;
            best = {};
            best.big = big;
            best.tiles_i = (int)ti;
            best.tiles_j = (int)tj;
            best.runs = (int)((steps + per - 1) / per);
            best.run = per * depth;
            best.copy = big && !aligned;
        }
    }
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += pad256(n);
        return here;
    };
    if (best.big) {
        best.xp = (a.width + 15) / 16 * 16;
        best.gp = best.copy ? (a.out + 7) / 8 * 8 : a.grad_stride;
        best.x = take(size_t(a.rows) * best.xp * 2);
        best.g = best.copy ? take(size_t(a.rows) * best.gp * 2) : 0;
    }
    if (best.runs > 1) {
        best.part = take(size_t(best.runs) * a.width * a.out * 4);
        best.bias = take(size_t(best.runs) * a.out * 4);
    }
    best.bytes = at;
    return best;
}

template <class T>
void weight(const wc_ckpt_weight_args& a, int cus, hipStream_t s) {
    const Plan p = plan_of(a, cus);
    char* w = (char*)a.workspace;
    // whole chunks of the last columns reach this far past a row's end, which the rows that follow must hold
    const int64_t past_q = (a.width + 15) / 16 * 16 - a.width, past_g = (a.out + 7) / 8 * 8 - a.out;
    auto rows_past = [&](int64_t past, int64_t stride) {
        return !past ? 0 : !stride ? a.rows : std::min(a.rows, (past + stride - 1) / stride);
    };
    const int64_t open = a.rows - std::max(rows_past(past_q, a.q_stride), rows_past(past_g, a.grad_stride));
    const Job job = {a, p.run, open, p.tiles_i, p.tiles_j, p.runs, (float*)(w + p.part), (float*)(w + p.bias)};
    const dim3 grid(p.tiles_i * p.tiles_j * p.runs);
    if constexpr (sizeof(T) == 2) {
        if (p.big) {
            auto lay_grid = [&](int64_t n) {
                return dim3((uint32_t)std::max<int64_t>(1, std::min<int64_t>((n + BLOCK - 1) / BLOCK, cus * 64)));
            };
            if (a.rows) {
                const int64_t x = p.xp / 16, g = p.gp / 8;
                k_expand<T><<<lay_grid(a.rows * x), BLOCK, 0, s>>>(a, (T*)(w + p.x), p.xp, x);
                if (p.copy) k_align<T><<<lay_grid(a.rows * g), BLOCK, 0, s>>>(a, (T*)(w + p.g), p.gp, g);
            }
            const BigJob big = {job, w + p.x, p.copy ? w + p.g : (const char*)a.grad, 2 * p.xp, 2 * p.gp};
            if (p.runs > 1 || a.weight_dtype == WC_DTYPE_F32) k_weight_big<T, float><<<grid, BLOCK, 0, s>>>(big);
            else k_weight_big<T, T><<<grid, BLOCK, 0, s>>>(big);
        }
    }
    if (!p.big) {
        if (a.act == WC_ACT_NONE) k_weight<T, 2, WC_ACT_NONE><<<grid, BLOCK, 0, s>>>(job);
        else if (a.act == WC_ACT_RELU) k_weight<T, 2, WC_ACT_RELU><<<grid, BLOCK, 0, s>>>(job);
        if constexpr (sizeof(T) == 2) {
            if (a.act == WC_ACT_GELU) k_weight<T, 2, WC_ACT_GELU><<<grid, BLOCK, 0, s>>>(job);
            else if (a.act == WC_ACT_SILU) k_weight<T, 2, WC_ACT_SILU><<<grid, BLOCK, 0, s>>>(job);
        }
    }
    if (p.runs > 1) {
        // 16-byte reads where every run's part starts on 16 bytes
        const int64_t n = a.out % 4 == 0 ? 4 : 1, blocks = (a.width * a.out + 64 * n - 1) / (64 * n);
        const dim3 g((uint32_t)(blocks + (a.bias ? (a.out + 64 * n - 1) / (64 * n) : 0)));
        if (a.weight_dtype == WC_DTYPE_F32) {
            if (n == 4) k_weight_sum<float, 4><<<g, BLOCK, 0, s>>>(job, blocks);
            else k_weight_sum<float, 1><<<g, BLOCK, 0, s>>>(job, blocks);
        } else {
            if (n == 4) k_weight_sum<T, 4><<<g, BLOCK, 0, s>>>(job, blocks);
            else k_weight_sum<T, 1><<<g, BLOCK, 0, s>>>(job, blocks);
        }
    }
}

}  // namespace

size_t ckpt_weight_scratch(const wc_ckpt_weight_args& a, int cus) { return plan_of(a, cus).bytes; }

void launch_ckpt_weight(const wc_ckpt_weight_args& a, int cus, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) weight<float>(a, cus, s);
    else if (a.dtype == WC_DTYPE_F16) weight<f16>(a, cus, s);
    else weight<bf16>(a, cus, s);
}

}  // namespace learn
}  // namespace wc
