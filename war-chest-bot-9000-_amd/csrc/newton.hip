// A matrix's singular values brought towards 1 by Newton-Schulz products (include/wc_learn.h).
//
//   X = U / (|U| + eps);  a few times: A = X X^T, B = b A + c A A, X = a X + B X  (X^T X and X B for a tall matrix)
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and written twice.
//
// X, A and B are held as sums of two f16 (22 bits), times 2^10, so that an element of 2^-13 still has all its bits. No
// element of X, A or B is larger than its largest singular value, s, s^2 and |b s^2 + c s^4|: below 63 each fits (f16 ends
// at 65504). A is what passes it first, at s = 7.9, or B, where the coefficients are large. A product is then three matrix
// products: the one of the two small parts is left out.
//
// For a bf16 result one product of the large parts is enough, with A and B in one f16 (11 bits), but X stays in 22: its
// rounding would fall on every direction, on small singular values that grow 500-fold too, where A's and B's fall on
// what is large already. A gradient with three large directions and 256 x 1,024 with 11-bit X comes out 8e-3 off (of its
// norm; all of it in bf16, 7e-2), with 22-bit X 9e-5; a random matrix 1.7e-3, as much as the result's own rounding.
// Up to 128 rows or columns (2.7e-3 at 40 x 200) the three products cost next to nothing, and are taken.
//
// 4,096 x 4,096 bf16, five steps: 1.57 ms, 874 TFLOP/s of the operations that symmetry leaves; the library's best large
// product reaches 1,528.
#include "learn.h"
#include "product_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

constexpr float HELD = 1024.f;
constexpr int SUM_BLOCKS = 1024;

// Where X, A or B lies: planes of rows of whole chunks of eight, zeros behind a row's end.
struct Held16 {
    f16* p;
    int64_t pitch, plane, batch;  // elements

    __device__ __forceinline__ void put(int planes, int batch_of, int64_t i, int64_t j, int n, const float (&v)[8]) const {
        f16x8 hi, lo;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const float x = u < n ? v[u] : 0.f;
            hi[u] = (f16)x;
            lo[u] = (f16)(x - (float)hi[u]);
        }
        f16* to = p + batch_of * batch + i * pitch + j;
        *(f16x8*)to = hi;
        if (planes > 1) *(f16x8*)(to + plane) = lo;
    }
    struct Eight {
        f16x8 hi, lo;
    };
    __device__ __forceinline__ Eight get(int planes, int batch_of, int64_t i, int64_t j) const {
        const f16* from = p + batch_of * batch + i * pitch + j;
        Eight e = {*(const f16x8*)from, f16x8{}};
        if (planes > 1) e.lo = *(const f16x8*)(from + plane);
        return e;
    }
};

// alpha v + beta (what `from` holds), to planes or to the result.
struct StepEpilogue {
    static constexpr bool MIRROR = true;
    Held16 from, to;
    int from_planes, to_planes, out_dtype;
    float alpha, beta;
    void* out;
    int64_t out_stride, out_batch;

    template <class T>
    __device__ __forceinline__ void result(int batch, int64_t i, int64_t j, int n, const float (&v)[8]) const {
        store_n((T*)out + batch * out_batch + i * out_stride + j, n, v);
    }
    __device__ __forceinline__ bool reads() const { return from.p != nullptr; }
    typedef Held16::Eight Raw;
    __device__ __forceinline__ Raw raw(int batch, int64_t i, int64_t j, int) const {
        return from.p ? from.get(from_planes, batch, i, j) : Raw{};
    }
    __device__ __forceinline__ void operator()(const Raw& r, int batch, int64_t i, int64_t j, int n, float (&v)[8]) const {
#pragma unroll
        for (int u = 0; u < 8; u++) {
            v[u] *= alpha;
            if (from.p) v[u] += beta * ((float)r.hi[u] + (float)r.lo[u]);
        }
        if (!out) to.put(to_planes, batch, i, j, n, v);
        else if (out_dtype == WC_DTYPE_F32) result<float>(batch, i, j, n, v);
        else if (out_dtype == WC_DTYPE_F16) result<f16>(batch, i, j, n, v);
        else result<bf16>(batch, i, j, n, v);
    }
};

template <class T>
struct Update {
    const T* u;
    int64_t stride, batch, rows, width;

    __device__ __forceinline__ void load(int b, int64_t chunk, int64_t per_row, float (&v)[8]) const {
        const int64_t r = chunk / per_row, c = 8 * (chunk - r * per_row);
        load_n(u + b * batch + r * stride + c, (int)min<int64_t>(8, width - c), 0.f, v);
    }
};

// Sum over a workgroup, the same in every thread.
__device__ __forceinline__ double all_of(double s, double (&lds)[4]) {
#pragma unroll
    for (int mask = 32; mask; mask >>= 1) s += __shfl_xor(s, mask);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Squares summed in 64 bits: they would leave float32's range from 2^64 on.
template <class T>
__global__ __launch_bounds__(256) void k_squares(Update<T> u, double* sums) {
    __shared__ double lds[4];
    const int64_t per_row = (u.width + 7) / 8, chunks = u.rows * per_row;
    double s = 0;
    for (int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x; at < chunks; at += int64_t(gridDim.x) * 256) {
        float v[8];
        u.load(blockIdx.y, at, per_row, v);
#pragma unroll
        for (int k = 0; k < 8; k++) s += (double)v[k] * (double)v[k];
    }
    s = all_of(s, lds);
    if (threadIdx.x == 0) sums[int64_t(blockIdx.y) * gridDim.x + blockIdx.x] = s;
}

template <class T>
__global__ __launch_bounds__(256) void k_start(Update<T> u, const double* sums, int blocks, float eps, Held16 to,
                                               int planes) {
    __shared__ double lds[4];
    double s = 0;
    for (int k = threadIdx.x; k < blocks; k += 256) s += sums[int64_t(blockIdx.y) * blocks + k];
    s = all_of(s, lds);
    const double rate = HELD / (sqrt(s) + (double)eps);
    const int64_t per_row = (u.width + 7) / 8, chunks = u.rows * per_row;
    for (int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x; at < chunks; at += int64_t(gridDim.x) * 256) {
        float v[8];
        u.load(blockIdx.y, at, per_row, v);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (float)((double)v[k] * rate);
        const int64_t r = at / per_row;
        to.put(planes, blockIdx.y, r, 8 * (at - r * per_row), 8, v);
    }
}

// ------------------------------------------------------------ small matrices

// A matrix whose X (in the form that is wide: small x large) and A fit in LDS, two parts each, in one launch: a workgroup
// of eight wavefronts a matrix. Fragments of 32 x 32, of A those on and above the diagonal only. B takes A's place, and X'
// X's, after a barrier. Vector arithmetic bounds it (splitting results into their parts, addresses): so the parts of eight
// elements lie beside each other, 16 bytes and 16 bytes, and one address serves both. 8 of 192 x 96, five steps: 45 us,
// 6.2 a step and 13 to load, norm and store; through memory, 17 launches, 123.
constexpr int SMALL_BLOCK = 512, SMALL_WAVES = SMALL_BLOCK / 64, SMALL_LDS = 160 * 1024, SMALL_TILES = 6;

struct SmallShape {
    int m, n, mp, np;  // small, large, and rounded up to whole fragments
    int px, pa;        // bytes from row to row: 16 more than the row has, so that rows lie in different banks

    __host__ __device__ SmallShape(int64_t small, int64_t large) {
        m = (int)small, n = (int)large;
        mp = (m + 31) / 32 * 32, np = (n + 31) / 32 * 32;
        px = 4 * np + 16, pa = 4 * mp + 16;
    }
    bool fits() const {
        return int64_t(mp) * (px + pa) <= SMALL_LDS && mp <= 128 &&
               (mp / 32) * (np / 32) <= SMALL_WAVES * SMALL_TILES;
    }
};

struct Pair16 {
    f16x8 hi, lo;
};

// Where element c of a row is.
__device__ __forceinline__ int place_of(int c) { return 4 * (c & ~7) + 2 * (c & 7); }

// Fragments along k, 16 at a time. Lane l's eight of k, from 8 (l / 32) on, of row first + l % 32, where rows have k inside.
struct ByRows {
    const char* p;

    __device__ __forceinline__ ByRows(const char* base, int pitch, int first, int lane)
        : p(base + (first + (lane & 31)) * pitch + 32 * (lane >> 5)) {}
    __device__ __forceinline__ Pair16 take(int part) const {
        return {*(const f16x8*)(p + 64 * part), *(const f16x8*)(p + 64 * part + 16)};
    }
    __device__ __forceinline__ void next() { p += 128; }  // 32 of k
};
// The same of column first + l % 32, where rows are on k.
struct ByColumns {
    const char *p, *q;  // four rows apart
    int pitch;

    __device__ __forceinline__ ByColumns(const char* base, int row, int first, int lane)
        : p(base + (8 * (lane >> 5) + ((lane & 15) >> 2)) * row + place_of(first + (lane & 16) + 4 * (lane & 3))),
          q(p + 4 * row), pitch(row) {}
    __device__ __forceinline__ Pair16 take(int part) const {
        return {eight(p + part * 16 * pitch, q + part * 16 * pitch),
                eight(p + part * 16 * pitch + 16, q + part * 16 * pitch + 16)};
    }
    __device__ __forceinline__ void next() { p += 32 * pitch, q += 32 * pitch; }
    static __device__ __forceinline__ f16x8 eight(const char* p, const char* q) {
        typedef __attribute__((address_space(3))) s16x4* At;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((At)q);
        return __builtin_bit_cast(f16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// c and the sum over k, a multiple of 32, of p's rows by q's columns; the next fragments are loaded beside each product.
template <class P, class Q>
__device__ __forceinline__ f32x16 sum_of(int all, f32x16 c, P p, Q q) {
    auto add = [&](const Pair16& a, const Pair16& b) {
        c = mfma(a.lo, b.hi, c);  // small by large, large by small, large by large
        c = mfma(a.hi, b.lo, c);
        c = mfma(a.hi, b.hi, c);
    };
    Pair16 a = p.take(0), b = q.take(0);
    for (int k = 32; k < all; k += 32) {
        const Pair16 a1 = p.take(1), b1 = q.take(1);
        p.next(), q.next();
        add(a, b);
        a = p.take(0), b = q.take(0);
        add(a1, b1);
    }
    const Pair16 a1 = p.take(1), b1 = q.take(1);
    add(a, b);
    add(a1, b1);
    return c;
}

typedef f16 f16x2 __attribute__((ext_vector_type(2)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// The parts of two elements.
__device__ __forceinline__ void split(float a, float b, f16x2& hi, f16x2& lo) {
    hi = __builtin_convertvector(f32x2{a, b}, f16x2);
    lo = __builtin_convertvector(f32x2{a - (float)hi[0], b - (float)hi[1]}, f16x2);
}

template <class T>
__global__ __launch_bounds__(SMALL_BLOCK, 2) void k_newton_small(Update<T> u, wc_orthogonalise_args o) {
    __shared__ __align__(16) char lds[SMALL_LDS];
    const bool tall = u.rows > u.width;
    const SmallShape s(tall ? u.width : u.rows, tall ? u.rows : u.width);
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    char* const x = lds;
    char* const a = lds + s.mp * s.px;
    const int wide = s.mp / 32, deep = s.np / 32, tiles = wide * deep, halves = wide * (wide + 1) / 2;

    // A wavefront's fragments of X stay in its registers in float32, and are what it adds to; LDS has what the products
    // read. Lane l has of a fragment column l % 32 and rows 8 (k / 4) + 4 (l / 32) + k % 4.
    f32x16 held[SMALL_TILES];
    const int down = 4 * (lane >> 5), across = lane & 31;
    auto each = [&](auto&& body) {
#pragma unroll
        for (int g = 0; g < SMALL_TILES; g++) {
            const int tile = wave + g * SMALL_WAVES;
            if (tile < tiles) body(held[g], 32 * (tile / deep), 32 * (tile % deep));
        }
    };
    // A fragment's parts to rows i0 .. of `to`; as rows of its mirror image too.
    auto put = [&](char* to, int pitch, const f32x16& c, int i0, int j0, bool mirror) {
        char* p = to + (i0 + down) * pitch + place_of(j0 + across);
        char* m = to + (j0 + across) * pitch + place_of(i0 + down);
#pragma unroll
        for (int q = 0; q < 4; q++) {
            f16x2 hi[2], lo[2];
#pragma unroll
            for (int k = 0; k < 2; k++) split(c[4 * q + 2 * k], c[4 * q + 2 * k + 1], hi[k], lo[k]);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                *(f16*)(p + k * pitch) = hi[k / 2][k % 2];
                *(f16*)(p + k * pitch + 16) = lo[k / 2][k % 2];
            }
            p += 8 * pitch;
            if (mirror) {  // eight rows on are the next sixteen bytes and sixteen
                *(f16x4*)(m + 32 * q) = __builtin_shufflevector(hi[0], hi[1], 0, 1, 2, 3);
                *(f16x4*)(m + 32 * q + 16) = __builtin_shufflevector(lo[0], lo[1], 0, 1, 2, 3);
            }
        }
    };

    // The matrix in chunks of eight of a row, as float32 where X's parts will be, and its norm: squares summed in 64 bits,
    // as in k_squares. Chunk c of a wide matrix is chunk c % per_row of a row, of a tall one a row's, rows first: then
    // neighbours write beside each other either way.
    const T* from = u.u + blockIdx.x * u.batch;
    const uint32_t width = (uint32_t)u.width, rows = (uint32_t)u.rows, per_row = (width + 7) / 8, chunks = rows * per_row;
    auto place = [&](uint32_t chunk, uint32_t& r, uint32_t& col) {
        const uint32_t by = tall ? rows : per_row, q = chunk / by, rest = chunk - q * by;
        r = tall ? rest : q, col = 8 * (tall ? q : rest);
    };
    for (int at = t * 16; at < s.mp * s.px; at += SMALL_BLOCK * 16) *(uint4*)(x + at) = uint4{};
    __syncthreads();
    double sum = 0;
    for (uint32_t first = t; first < chunks; first += 4 * SMALL_BLOCK) {
        float v[4][8] = {};
        uint32_t r[4], col[4];
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const uint32_t chunk = first + g * SMALL_BLOCK;
            place(chunk, r[g], col[g]);
            if (chunk < chunks) load_n(from + r[g] * u.stride + col[g], (int)min(8u, width - col[g]), 0.f, v[g]);
        }
#pragma unroll
        for (int g = 0; g < 4; g++) {
            if (first + g * SMALL_BLOCK >= chunks) break;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                sum += (double)v[g][k] * (double)v[g][k];
                if (col[g] + k < width) *(float*)(x + (tall ? (col[g] + k) * s.px + 4 * r[g] : r[g] * s.px + 4 * (col[g] + k))) = v[g][k];
            }
        }
    }
#pragma unroll
    for (int mask = 32; mask; mask >>= 1) sum += __shfl_xor(sum, mask);
    double* sums = (double*)a;
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < SMALL_WAVES; w++) sum += sums[w];
    const double rate = HELD / (sqrt(sum) + (double)o.eps);
    each([&](f32x16& c, int i0, int j0) {
        const char* p = x + (i0 + down) * s.px + 4 * (j0 + across);
#pragma unroll
        for (int k = 0; k < 16; k++) c[k] = (float)((double)*(const float*)(p + (8 * (k / 4) + k % 4) * s.px) * rate);
    });
    __syncthreads();
    each([&](f32x16& c, int i0, int j0) { put(x, s.px, c, i0, j0, false); });
    __syncthreads();

    // a wavefront's fragments of A and B, on or above the diagonal
    constexpr int HALVES = (10 + SMALL_WAVES - 1) / SMALL_WAVES;
    auto each_half = [&](f32x16(&c)[HALVES], auto&& body) {
#pragma unroll
        for (int g = 0; g < HALVES; g++) {
            const int tile = wave + g * SMALL_WAVES;
            if (tile >= halves) break;
            int tj = 0;
            while ((tj + 1) * (tj + 2) / 2 <= tile) tj++;
            body(c[g], 32 * (tile - tj * (tj + 1) / 2), 32 * tj);
        }
    };
    for (int step = 0; step < o.steps; step++) {
        f32x16 c[HALVES];
        // A = X X^T
        each_half(c, [&](f32x16& d, int i0, int j0) {
            d = sum_of(s.np, f32x16{}, ByRows(x, s.px, i0, lane), ByRows(x, s.px, j0, lane));
#pragma unroll
            for (int k = 0; k < 16; k++) d[k] *= 1.f / HELD;
            put(a, s.pa, d, i0, j0, i0 != j0);
        });
        __syncthreads();
        // B = b A + c A A
        each_half(c, [&](f32x16& d, int i0, int j0) {
            const f32x16 e = sum_of(s.mp, f32x16{}, ByRows(a, s.pa, i0, lane), ByRows(a, s.pa, j0, lane));
#pragma unroll
            for (int k = 0; k < 16; k++) d[k] = o.b * d[k] + o.c / HELD * e[k];
        });
        __syncthreads();
        each_half(c, [&](f32x16& d, int i0, int j0) { put(a, s.pa, d, i0, j0, i0 != j0); });
        __syncthreads();
        // X' = a X + B X
        each([&](f32x16& d, int i0, int j0) {
            const f32x16 e = sum_of(s.mp, f32x16{}, ByRows(a, s.pa, i0, lane), ByColumns(x, s.px, j0, lane));
#pragma unroll
            for (int k = 0; k < 16; k++) d[k] = o.a * d[k] + e[k] * (1.f / HELD);
        });
        __syncthreads();
        if (step + 1 == o.steps) break;
        each([&](f32x16& d, int i0, int j0) { put(x, s.px, d, i0, j0, false); });
        __syncthreads();
    }
    // and back the same way
    const float scale = o.scale / HELD;
    each([&](f32x16& c, int i0, int j0) {
        char* p = x + (i0 + down) * s.px + 4 * (j0 + across);
#pragma unroll
        for (int k = 0; k < 16; k++) *(float*)(p + (8 * (k / 4) + k % 4) * s.px) = c[k] * scale;
    });
    __syncthreads();
    for (uint32_t chunk = t; chunk < chunks; chunk += SMALL_BLOCK) {
        uint32_t r, col;
        place(chunk, r, col);
        const int have = (int)min(8u, width - col);
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const uint32_t c = min(col + k, width - 1);
            v[k] = *(const float*)(x + (tall ? c * s.px + 4 * r : r * s.px + 4 * c));
        }
        const int64_t to = blockIdx.x * o.out_batch + r * o.out_stride + col;
        if (o.out_dtype == WC_DTYPE_F32) store_n((float*)o.out + to, have, v);
        else if (o.out_dtype == WC_DTYPE_F16) store_n((f16*)o.out + to, have, v);
        else store_n((bf16*)o.out + to, have, v);
    }
}

// ----------------------------------------------------------- narrow matrices

// A = X X^T and B = b A + c A A where tiles of 64 would be few: a workgroup of eight wavefronts a fragment of 32 x 32 on
// or above the diagonal, each an eighth of k, straight from memory (rows have k inside: 16 bytes a lane), added in LDS.
// 256 x 1,024, one part: 7.8 us and 3.6, on tiles of 64 12 and 6. A call with 512 rows, and with 520 on tiles: 2,048
// columns 133 us and 187, 4,096 182 and 222, 8,192 280 and 284; in two parts 220 and 304, 315 and 378, 491 and 466.
constexpr int NARROW_BLOCK = 512, NARROW_WAVES = NARROW_BLOCK / 64;

struct NarrowJob {
    Held16 x;       // rows of k
    int64_t m, k;
    Held16 from, to;
    float alpha, beta;
};

template <int PARTS>
__global__ __launch_bounds__(NARROW_BLOCK) void k_narrow(NarrowJob o) {
    __shared__ float sums[NARROW_WAVES][32][33];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, batch = blockIdx.y;
    int tj = (int)((sqrtf(8.f * blockIdx.x + 1.f) - 1.f) * 0.5f);
    while (tj * (tj + 1) / 2 > (int)blockIdx.x) tj--;
    while ((tj + 1) * (tj + 2) / 2 <= (int)blockIdx.x) tj++;
    const int64_t i0 = 32 * (blockIdx.x - tj * (tj + 1) / 2), j0 = 32 * tj;
    // past the last row any row will do: its products are not stored
    const f16* base = o.x.p + batch * o.x.batch + 8 * (lane >> 5);
    const f16* pa = base + min(i0 + (lane & 31), o.m - 1) * o.x.pitch;
    const f16* pb = base + min(j0 + (lane & 31), o.m - 1) * o.x.pitch;
    const int steps = (int)((o.k + 15) / 16), each = (steps + NARROW_WAVES - 1) / NARROW_WAVES;
    const int lo = wave * each, hi = min(lo + each, steps);
    f32x16 c = {};
#pragma unroll 8
    for (int s = lo; s < hi; s++) {
        f16x8 a[PARTS], b[PARTS];
        const bool there = 16 * s + 8 * (lane >> 5) < o.k;  // whole eights, zeros in the last
#pragma unroll
        for (int u = 0; u < PARTS; u++) {
            a[u] = there ? *(const f16x8*)(pa + 16 * s + u * o.x.plane) : f16x8{};
            b[u] = there ? *(const f16x8*)(pb + 16 * s + u * o.x.plane) : f16x8{};
        }
        if constexpr (PARTS > 1) {
            c = mfma(a[1], b[0], c);
            c = mfma(a[0], b[1], c);
        }
        c = mfma(a[0], b[0], c);
    }
#pragma unroll
    for (int k = 0; k < 16; k++) sums[wave][8 * (k / 4) + 4 * (lane >> 5) + k % 4][lane & 31] = c[k];
    __syncthreads();
    const int r = threadIdx.x / 16, col = threadIdx.x % 16 * 2;
    const int64_t padded = (o.m + 7) & ~int64_t(7);
#pragma unroll
    for (int u = 0; u < 2; u++) {
        const int64_t i = i0 + r, j = j0 + col + u;
        float v = 0.f;
        if (i < o.m && j < o.m) {
            for (int w = 0; w < NARROW_WAVES; w++) v += sums[w][r][col + u];
            v *= o.alpha;
            if (o.from.p) {
                const f16* from = o.from.p + batch * o.from.batch + i * o.from.pitch + j;
                v += o.beta * ((float)from[0] + (PARTS > 1 ? (float)from[o.from.plane] : 0.f));
            }
        }
        const f16 hi = (f16)v, low = (f16)(v - (float)hi);
        f16* to = o.to.p + batch * o.to.batch;
        if (i < o.m && j < padded) {
            to[i * o.to.pitch + j] = hi;
            if (PARTS > 1) to[i * o.to.pitch + j + o.to.plane] = low;
        }
        if (i0 != j0 && j < o.m && i < padded) {
            to[j * o.to.pitch + i] = hi;
            if (PARTS > 1) to[j * o.to.pitch + i + o.to.plane] = low;
        }
    }
}

// A tall matrix turned, as X's parts, and back as the result: eight of a row a thread, rows first.
template <class T>
__global__ __launch_bounds__(256) void k_start_turned(Update<T> u, const double* sums, int blocks, float eps, Held16 to) {
    __shared__ double lds[4];
    double s = 0;
    for (int k = threadIdx.x; k < blocks; k += 256) s += sums[int64_t(blockIdx.y) * blocks + k];
    s = all_of(s, lds);
    const double rate = HELD / (sqrt(s) + (double)eps);
    const int64_t rows = to.pitch, chunks = rows * ((u.width + 7) / 8);  // with zeros to the end of to's rows
    for (int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x; at < chunks; at += int64_t(gridDim.x) * 256) {
        const int64_t c = at / rows * 8, r = at % rows;
        float v[8] = {};
        if (r < u.rows) load_n(u.u + blockIdx.y * u.batch + r * u.stride + c, (int)min<int64_t>(8, u.width - c), 0.f, v);
        f16* p = to.p + blockIdx.y * to.batch + c * to.pitch + r;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            if (c + k >= u.width) break;
            const float x = (float)((double)v[k] * rate);
            const f16 hi = (f16)x;
            p[k * to.pitch] = hi;
            p[k * to.pitch + to.plane] = (f16)(x - (float)hi);
        }
    }
}

template <class T>
__global__ __launch_bounds__(256) void k_finish_turned(Held16 x, int64_t rows, int64_t width, float scale, T* out,
                                                       int64_t stride, int64_t batch) {
    const int64_t chunks = rows * ((width + 7) / 8);
    for (int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x; at < chunks; at += int64_t(gridDim.x) * 256) {
        const int64_t c = at / rows * 8, r = at % rows;
        const f16* p = x.p + blockIdx.y * x.batch + c * x.pitch + r;
        float v[8] = {};
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (c + k < width) v[k] = scale * ((float)p[k * x.pitch] + (float)p[k * x.pitch + x.plane]);
        store_n(out + blockIdx.y * batch + r * stride + c, (int)min<int64_t>(8, width - c), v);
    }
}

struct Plan {
    int planes, segments, blocks;  // planes of A and B, and of X in products; X has two
    int64_t small, pitch, pitch_small, x_plane, a_plane;  // elements
    bool narrow, turned;  // narrow: k_narrow, for which a tall matrix is turned
    int64_t x_rows, x_cols;
    Cut gram, square, step;
    size_t x[2], a, b, sums, part, bytes;
};

Plan plan_of(const wc_orthogonalise_args& o, int cus) {
    Plan p = {};
    const bool tall = o.rows > o.width;
    p.small = tall ? o.width : o.rows;
    p.planes = o.out_dtype == WC_DTYPE_BF16 && p.small > 128 ? 1 : 2;
    p.segments = p.planes == 1 ? 1 : 3;
    const int64_t large = tall ? o.rows : o.width;
    const int64_t fragments = (p.small + 31) / 32;
    p.narrow = p.small <= 512 && large <= 4096 && fragments * (fragments + 1) / 2 * o.batch <= 2 * int64_t(cus);
    p.turned = p.narrow && tall;
    p.x_rows = p.turned ? o.width : o.rows;
    p.x_cols = p.turned ? o.rows : o.width;
    p.pitch = up(p.x_cols, 8);
    p.pitch_small = up(p.small, 8);
    p.x_plane = p.x_rows * p.pitch;
    p.a_plane = p.small * p.pitch_small;
    p.gram = cut_of(p.small, p.small, large, p.segments, cus, o.batch, true);
    p.square = cut_of(p.small, p.small, p.small, p.segments, cus, o.batch, true);
    p.step = cut_of(p.x_rows, p.x_cols, p.small, p.segments, cus, o.batch);
    const int64_t chunks = o.rows * ((o.width + 7) / 8);
    p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>((chunks + 1023) / 1024, SUM_BLOCKS));
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += pad256(n);
        return here;
    };
    const size_t each = size_t(o.batch) * p.planes * 2;
    p.x[0] = take(size_t(o.batch) * 4 * p.x_plane);
    p.x[1] = take(size_t(o.batch) * 4 * p.x_plane);
    p.a = take(each * p.a_plane);
    p.b = take(each * p.a_plane);
    p.sums = take(size_t(o.batch) * p.blocks * 8);
    const int64_t small = p.narrow ? 0 : o.batch * p.small * p.small;
    p.part = take(std::max({p.gram.bytes(small), p.square.bytes(small), p.step.bytes(o.batch * o.rows * o.width)}));
    p.bytes = at;
    return p;
}

Operand16 operand(const Held16& h, int planes, int64_t outer) {
    Operand16 o = {};
    for (int k = 0; k < planes; k++) o.plane[k] = (const char*)(h.p + k * h.plane);
    o.pitch = 2 * h.pitch;
    o.batch = 2 * h.batch;
    o.outer = outer;
    return o;
}

// Matrices of a launch, unless each is a workgroup's: 2^20 elements in a row are 2^12 tiles of 256, and a launch holds
// fewer than 2^24 workgroups of 256.
constexpr int64_t MOST_MATRICES = 2048;

bool small_enough(const wc_orthogonalise_args& o) {
    const int64_t small = std::min(o.rows, o.width), large = std::max(o.rows, o.width);
    return small <= 128 && large <= 4096 && SmallShape(small, large).fits();
}

template <class T>
void start(const wc_orthogonalise_args& o, const Plan& p, const Held16& x, hipStream_t s) {
    const Update<T> u = {(const T*)o.update, o.update_stride, o.update_batch, o.rows, o.width};
    if (small_enough(o)) {
        k_newton_small<T><<<dim3((uint32_t)o.batch), SMALL_BLOCK, 0, s>>>(u, o);
        return;
    }
    double* sums = (double*)((char*)o.workspace + p.sums);
    const dim3 grid((uint32_t)p.blocks, (uint32_t)o.batch);
    k_squares<T><<<grid, 256, 0, s>>>(u, sums);
    const int64_t chunks = p.x_rows * (p.pitch / 8);
    const dim3 wide((uint32_t)std::min<int64_t>((chunks + 255) / 256, 4096), (uint32_t)o.batch);
    if (p.turned) k_start_turned<T><<<wide, 256, 0, s>>>(u, sums, p.blocks, o.eps, x);
    else k_start<T><<<wide, 256, 0, s>>>(u, sums, p.blocks, o.eps, x, 2);
}

}  // namespace

// The plan of a launch's matrices; the last launch may have fewer.
static Plan launch_plan(const wc_orthogonalise_args& o, int cus) {
    wc_orthogonalise_args some = o;
    some.batch = std::min(o.batch, MOST_MATRICES);
    return plan_of(some, cus);
}

size_t orthogonalise_scratch(const wc_orthogonalise_args& o, int cus) {
    return small_enough(o) ? 0 : launch_plan(o, cus).bytes;
}

static void orthogonalise(const wc_orthogonalise_args& o, const Plan& p, hipStream_t s) {
    char* w = (char*)o.workspace;
    Held16 x[2], a = {(f16*)(w + p.a), p.pitch_small, p.a_plane, p.a_plane * p.planes}, b = a;
    b.p = (f16*)(w + p.b);
    for (int k = 0; k < 2; k++) x[k] = {(f16*)(w + p.x[k]), p.pitch, p.x_plane, p.x_plane * 2};
    if (o.dtype == WC_DTYPE_F32) start<float>(o, p, x[0], s);
    else if (o.dtype == WC_DTYPE_F16) start<f16>(o, p, x[0], s);
    else start<bf16>(o, p, x[0], s);
    if (small_enough(o)) return;

    const bool tall = o.rows > o.width && !p.turned;
    float* part = (float*)(w + p.part);
    for (int k = 0; k < o.steps; k++) {
        const Held16 &from = x[k & 1], &to = x[k + 1 & 1];
        Product m = {};
        m.segments = p.segments;
        m.batches = (int)o.batch;
        if (p.planes > 1) {
            m.pa[0] = 1, m.pb[1] = 1;  // small by large, large by small, large by large
        }
        StepEpilogue e = {};
        e.from_planes = e.to_planes = p.planes;
        if (p.narrow) {
            const int64_t fragments = (p.small + 31) / 32;
            const dim3 grid((uint32_t)(fragments * (fragments + 1) / 2), (uint32_t)o.batch);
            auto narrow = [&](const NarrowJob& job) {
                if (p.planes == 1) k_narrow<1><<<grid, NARROW_BLOCK, 0, s>>>(job);
                else k_narrow<2><<<grid, NARROW_BLOCK, 0, s>>>(job);
            };
            narrow({from, p.small, p.x_cols, {}, a, 1.f / HELD, 0.f});
            narrow({a, p.small, p.small, a, b, o.c / HELD, o.b});
        } else {
            // A
            m.a = m.b = operand(from, p.planes, p.small);
            m.k = tall ? o.rows : o.width;
            e.to = a;
            e.alpha = 1.f / HELD;
            launch_product<f16>(m, p.gram, !tall, !tall, part, e, s);
            // b A + c A A
            m.a = m.b = operand(a, p.planes, p.small);
            m.k = p.small;
            e.from = a;
            e.to = b;
            e.alpha = o.c / HELD;
            e.beta = o.b;
            launch_product<f16>(m, p.square, true, true, part, e, s);
        }
        m.k = p.small;
        // a X + B X, or X B
        const Operand16 ob = operand(b, p.planes, p.small), ox = operand(from, p.planes, tall ? o.rows : p.x_cols);
        m.a = tall ? ox : ob;
        m.b = tall ? ob : ox;
        e.from = from;
        e.to = to;
        e.from_planes = e.to_planes = 2;
        e.alpha = 1.f / HELD;
        e.beta = o.a;
        if (k + 1 == o.steps && !p.turned) {
            e.alpha *= o.scale / HELD;
            e.beta *= o.scale / HELD;
            e.out = o.out;
            e.out_dtype = o.out_dtype;
            e.out_stride = o.out_stride;
            e.out_batch = o.out_batch;
        }
        launch_product<f16>(m, p.step, true, tall, part, e, s);
    }
    if (p.turned) {
        const int64_t chunks = o.rows * ((o.width + 7) / 8);
        const dim3 grid((uint32_t)std::min<int64_t>((chunks + 255) / 256, 4096), (uint32_t)o.batch);
        auto finish = [&](auto* out) {
            k_finish_turned<<<grid, 256, 0, s>>>(x[o.steps & 1], o.rows, o.width, o.scale / HELD, out, o.out_stride, o.out_batch);
        };
        if (o.out_dtype == WC_DTYPE_F32) finish((float*)o.out);
        else if (o.out_dtype == WC_DTYPE_F16) finish((f16*)o.out);
        else finish((bf16*)o.out);
    }
}

void launch_orthogonalise(const wc_orthogonalise_args& o, int cus, hipStream_t s) {
    if (!o.batch) return;
    const Plan p = launch_plan(o, cus);
    if (small_enough(o)) return orthogonalise(o, p, s);
    for (int64_t lo = 0; lo < o.batch; lo += MOST_MATRICES) {
        wc_orthogonalise_args some = o;
        some.batch = std::min(o.batch - lo, MOST_MATRICES);
        some.update = (const char*)o.update + lo * o.update_batch * (o.dtype == WC_DTYPE_F32 ? 4 : 2);
        some.out = (char*)o.out + lo * o.out_batch * (o.out_dtype == WC_DTYPE_F32 ? 4 : 2);
        orthogonalise(some, p, s);
    }
}

}  // namespace learn
}  // namespace wc
