// A layer's product with bias, activation and residual in its epilogue, and its gradients (include/wc_learn.h), for one
// element type: linear_f32.hip, linear_f16.hip and linear_bf16.hip build one each.
//
//   y = act(x W + b) + residual;  d_pre = d_y act'(pre);  d_x = d_pre W^T;  d_W = x^T d_pre;  d_b = column sums of d_pre
//
// The three products differ in which index of each operand is summed; one kernel takes all (product_dev.h). Sums, bias,
// activation and residual are float32 and rounded once, to the output's type. d_pre is rounded to the 16-bit type for
// its two products (as it would be between two operators): its own half ulp, 2^-9 of an element in bf16, against the
// same for every element of the result, which is then 2.3e-3 of its norm off in place of 1.7e-3. Pre-activations are kept
// in float32: in 16 bits their rounding would be 10^4 times that of the float32 sums of d_b (1.3e-3 of its norm in bf16).
//
// float32 operands are taken as three bf16 parts (8 + 8 + 8 bits), and of their nine products the six that matter:
// the matrix cores' own float32 rate is a sixteenth of the 16-bit one. Small ones, whose launches cost more than their
// products, are left as they are (direct_dev.h).
#pragma once

#include "ckpt8_dev.h"
#include "direct_dev.h"
#include "learn.h"
#include "product_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

// The 16-bit type that products are taken in, and the parts of an element.
template <class T>
struct Parts {
    typedef T type;
    static constexpr int COUNT = 1;
};
template <>
struct Parts<float> {
    typedef bf16 type;
    static constexpr int COUNT = 3;
};

// Each part is what is left rounded to bf16; the third is exact, and the products that are left out are below 2^-25 of
// the whole. A first part that would round past bf16's largest is cut, and the second too: together they are no
// larger than x, in whatever order they are added. What an infinity leaves is 0.
__device__ __forceinline__ bf16 cut_bf16(float x) { return __builtin_bit_cast(bf16, (uint16_t)(__float_as_uint(x) >> 16)); }
__device__ __forceinline__ void parts_of(float x, bf16 (&o)[3]) {
    o[0] = (bf16)x;
    const bool past = fabsf((float)o[0]) == INFINITY;
    if (past) o[0] = cut_bf16(x);
    x -= (float)o[0];
    x = x == x ? x : 0.f;
    o[1] = past ? cut_bf16(x) : (bf16)x;
    o[2] = (bf16)(x - (float)o[1]);
}

// Eight values to a row of an operand's planes.
template <class T>
__device__ __forceinline__ void put_parts(char* to, int64_t plane, const float (&v)[8]) {
    typedef typename Parts<T>::type E;
    typedef E E8 __attribute__((ext_vector_type(8)));
    if constexpr (Parts<T>::COUNT == 1) {
        E8 o;
#pragma unroll
        for (int u = 0; u < 8; u++) {
            o[u] = (E)v[u];
            // what float32 holds and would round past bf16's largest
            if constexpr (__is_same(E, bf16))
                if (fabsf((float)o[u]) == INFINITY && fabsf(v[u]) != INFINITY) o[u] = cut_bf16(v[u]);
        }
        *(E8*)to = o;
    } else {
        E8 o[3];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            bf16 part[3];
            parts_of(v[u], part);
#pragma unroll
            for (int k = 0; k < 3; k++) o[k][u] = part[k];
        }
#pragma unroll
        for (int k = 0; k < 3; k++) *(E8*)(to + k * plane) = o[k];
    }
}

// What a product reads of a matrix: the matrix itself, or a copy of it in the workspace, in parts, on 16-byte rows, with
// zeros up to whole steps where there are several parts.
struct Laid {
    bool copy;
    int64_t rows, cols, pitch, plane;  // of the copy: rows and columns with the zeros, bytes
    size_t at;

    size_t bytes(int parts) const { return copy ? size_t(plane) * parts : 0; }
};

template <class T>
Laid laid(const void* p, int64_t stride, int64_t rows, int64_t cols) {
    Laid l = {};
    constexpr bool one = Parts<T>::COUNT == 1;
    // (a lane's place in a tile is held in 32 bits)
    const bool whole = cols % 8 == 0 && ((uintptr_t)p & 15) == 0 && (rows <= 1 || (stride % 8 == 0 && stride < (1 << 22)));
    l.copy = !one || !whole;
    if (!l.copy) {
        l.rows = rows;
        l.cols = cols;
        l.pitch = rows <= 1 ? 2 * cols : 2 * stride;
        return l;
    }
    l.rows = one ? rows : up(rows, STEP);
    l.cols = up(cols, one ? 8 : STEP);
    l.pitch = 2 * l.cols;
    l.plane = l.pitch * l.rows;
    return l;
}

struct Source {
    const void* p;
    int64_t stride, rows, cols;
    char* to;
    int64_t to_rows, to_cols, plane;
};

// Up to two matrices copied into planes, a chunk of eight a thread, by workgroup `block` of `blocks`.
template <class T>
__device__ __forceinline__ void lay_chunks(const Source& one, const Source& two, int64_t block, int64_t blocks) {
    const int64_t n1 = one.to_rows * (one.to_cols / 8), n2 = two.to_rows * (two.to_cols / 8);
    for (int64_t at = block * 256 + threadIdx.x; at < n1 + n2; at += blocks * 256) {
        const Source& s = at < n1 ? one : two;
        const int64_t chunk = at < n1 ? at : at - n1, per_row = s.to_cols / 8, r = chunk / per_row, c = 8 * (chunk - r * per_row);
        float v[8] = {};
        if (r < s.rows && c < s.cols) load_n((const T*)s.p + r * s.stride + c, (int)min<int64_t>(8, s.cols - c), 0.f, v);
        put_parts<T>(s.to + 2 * (r * s.to_cols + c), s.plane, v);
    }
}
template <class T>
__global__ __launch_bounds__(256) void k_lay(Source one, Source two) {
    lay_chunks<T>(one, two, blockIdx.x, gridDim.x);
}

// y = act(v + bias) + residual, and the kept v + bias.
template <class T>
struct LayerEpilogue {
    static constexpr bool MIRROR = false;
    const void* bias;
    bool bias_f32;
    const T* residual;
    int64_t residual_stride;
    float* pre;
    int64_t pre_stride;
    T* y;
    int64_t y_stride;
    int act;

    // The same from row lo on.
    LayerEpilogue from(int64_t lo) const {
        LayerEpilogue e = *this;
        if (residual) e.residual += lo * residual_stride;
        if (pre) e.pre += lo * pre_stride;
        e.y += lo * y_stride;
        return e;
    }
    __device__ __forceinline__ bool reads() const { return residual != nullptr; }
    typedef typename Vec8<T>::type Raw;
    __device__ __forceinline__ Raw raw(int, int64_t i, int64_t j, int n) const {
        return residual ? load_some<8>(residual + i * residual_stride + j, n) : Raw{};
    }
    __device__ __forceinline__ void operator()(const Raw& r, int, int64_t i, int64_t j, int n, float (&v)[8]) const {
        if (bias) {
            float b[8];
            if (bias_f32) load_n((const float*)bias + j, n, 0.f, b);
            else load_n((const T*)bias + j, n, 0.f, b);
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] += b[u];
        }
        if (pre) store_n(pre + i * pre_stride + j, n, v);
        act_values(v, act);
        if (residual) {
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] += (float)r[u];
        }
        store_n(y + i * y_stride + j, n, v);
    }
};

// A gradient, as the product is or times a number in memory.
template <class T>
struct GradEpilogue {
    static constexpr bool MIRROR = false;
    T* y;
    int64_t y_stride;
    const float* rate;  // null: 1

    struct Raw {};
    __device__ __forceinline__ bool reads() const { return false; }
    __device__ __forceinline__ Raw raw(int, int64_t, int64_t, int) const { return {}; }
    __device__ __forceinline__ void operator()(const Raw&, int, int64_t i, int64_t j, int n, float (&v)[8]) const {
        if (rate) {
            const float by = *rate;
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] *= by;
        }
        store_n(y + i * y_stride + j, n, v);
    }
};

template <class T>
Operand16 operand(const Laid& l, const void* p, char* workspace, int64_t outer) {
    Operand16 o = {};
    for (int k = 0; k < Parts<T>::COUNT; k++) o.plane[k] = l.copy ? workspace + l.at + k * l.plane : (const char*)p;
    o.pitch = l.pitch;
    o.outer = outer;
    return o;
}

// The segments of a product whose a, b and k are set.
template <class T>
Product segments_of(Product p) {
    if (Parts<T>::COUNT == 3) {
        // the largest last: what is small is added to what is small
        static constexpr uint8_t pa[] = {2, 1, 0, 1, 0, 0}, pb[] = {0, 1, 2, 0, 1, 0};
        p.segments = 6;
        for (int k = 0; k < 6; k++) p.pa[k] = pa[k], p.pb[k] = pb[k];
    } else {
        p.segments = 1;
    }
    p.batches = 1;
    return p;
}

template <class T, class Epilogue>
void multiply(const Product& p, const Cut& cut, bool ai, bool bi, float* part, const Epilogue& e, hipStream_t s) {
    launch_product<typename Parts<T>::type>(segments_of<T>(p), cut, ai, bi, part, e, s);
}

inline dim3 lay_grid(int64_t chunks, int cus) {
    return dim3((uint32_t)std::max<int64_t>(1, std::min<int64_t>((chunks + 255) / 256, int64_t(cus) * 32)));
}

// Where a matrix is copied to; nothing where it is read as it lies.
inline Source copy_of(const Laid& l, Source s, char* workspace) {
    if (!l.copy) return {};
    s.to = workspace + l.at;
    s.to_rows = l.rows;
    s.to_cols = l.cols;
    s.plane = l.plane;
    return s;
}
inline int64_t chunks_of(const Source& a, const Source& b) { return a.to_rows * (a.to_cols / 8) + b.to_rows * (b.to_cols / 8); }

template <class T>
void lay(const Source& a, const Source& b, int cus, hipStream_t s) {
    if (const int64_t n = chunks_of(a, b)) k_lay<T><<<lay_grid(n, cus), 256, 0, s>>>(a, b);
}

// ------------------------------------------------------------------ few rows

// A few rows against a weight: the weight is read once, and nothing else matters. No matrix instruction, no copy: a lane
// has 16 bytes of a weight's row at a time, eight rows of it, times eight of k of every row of x. A wavefront's loads are
// whole lines of 128 bytes, eight of them in flight while the last eight are multiplied. 4,096 x 16,384 bf16, one row: 28
// us, 4.8 TB/s (a large copy moves 5.16; the tiles of 64, with split sums, take 33).
//
// Where rows of the weight are on k (IN_OUT) a wavefront has eight lanes across, 128 bytes of columns, and 64 of k, the
// workgroup's wavefronts follow each other along k and add up at the end. Where they are outputs (OUT_IN) a wavefront has
// eight outputs and all lanes along k.
constexpr int FEW_BLOCK = 512, FEW_WAVES = FEW_BLOCK / 64;

struct FewJob {
    int64_t rows, width, out, x_stride, w_stride, run;  // run: of k, a multiple of 512
    int runs;
    float* part;
};

template <class T, int R, bool IO, class Epilogue>
__global__ __launch_bounds__(FEW_BLOCK) void k_few(const T* x, const T* w, FewJob job, Epilogue epilogue) {
    constexpr int E = 16 / sizeof(T);
    typedef typename VecN<T, E>::type Chunk;
    __shared__ float lds[IO ? FEW_WAVES : 1][R][8 * E];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int groups = gridDim.x / job.runs, run = blockIdx.x / groups, group = blockIdx.x - run * groups;
    const int64_t lo = run * job.run, hi = min(lo + job.run, job.width);
    const T* rows[R];
#pragma unroll
    for (int r = 0; r < R; r++) rows[r] = x + min<int64_t>(r, job.rows - 1) * job.x_stride;  // what is not there is not stored
    auto to = [&](int64_t r, int64_t j, int n, float (&v)[8]) {
        if (job.runs > 1) store_n(job.part + (run * job.rows + r) * job.out + j, n, v);
        else epilogue(epilogue.raw(0, r, j, n), 0, r, j, n, v);
    };

    if constexpr (IO) {
        const int64_t j = int64_t(group) * 8 * E + (lane & 7) * E;
        const int have = (int)max<int64_t>(0, min<int64_t>(E, job.out - j));
        float acc[R][E] = {};
        const T* at = w + (lo + wave * 64 + (lane >> 3) * 8) * job.w_stride + (have == E ? j : 0);
        auto add = [&](int64_t k, const Chunk (&c)[8], int there) {
            float v[R][8];
#pragma unroll
            for (int r = 0; r < R; r++) load_n(rows[r] + k, there, 0.f, v[r]);
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float f = (float)c[i][e];
#pragma unroll
                    for (int r = 0; r < R; r++) acc[r][e] += v[r][i] * f;
                }
        };
        int64_t k = lo + wave * 64 + (lane >> 3) * 8;
        if (have == E) {
            Chunk c[8];
            auto load = [&](const T* p, Chunk (&d)[8]) {
#pragma unroll
                for (int i = 0; i < 8; i++) d[i] = *(const Chunk*)(p + i * job.w_stride);
            };
            bool whole = k + 8 <= hi;
            if (whole) load(at, c);
            while (whole) {
                const int64_t next = k + 64 * FEW_WAVES;
                at += 64 * FEW_WAVES * job.w_stride;
                whole = next + 8 <= hi;
                Chunk d[8];
                if (whole) load(at, d);
                add(k, c, 8);
#pragma unroll
                for (int i = 0; i < 8; i++) c[i] = d[i];
                k = next;
            }
        }
        // the last of k, and the last columns
        for (; k < hi && have; k += 64 * FEW_WAVES) {
            const int there = (int)min<int64_t>(8, hi - k);
            Chunk c[8] = {};
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < there) c[i] = load_some<E>(w + (k + i) * job.w_stride + j, have);
            add(k, c, there);
        }
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                float s = acc[r][e];
#pragma unroll
                for (int mask = 8; mask < 64; mask <<= 1) s += __shfl_xor(s, mask);
                if (lane < 8) lds[wave][r][lane * E + e] = s;
            }
        __syncthreads();
        if (threadIdx.x >= 8 * R) return;
        const int r = threadIdx.x / 8, at_e = threadIdx.x % 8 * E;
        if (r >= job.rows || j >= job.out) return;
        float v[8] = {};
#pragma unroll
        for (int e = 0; e < E; e++)
            for (int u = 0; u < FEW_WAVES; u++) v[e] += lds[u][r][at_e + e];
        to(r, j, have, v);
    } else {
        const int64_t j = (int64_t(group) * FEW_WAVES + wave) * 8;  // eight outputs
        const int have = (int)max<int64_t>(0, min<int64_t>(8, job.out - j));
        float acc[R][8] = {};
        auto add = [&](int64_t k, const Chunk (&c)[8], int there) {
            float v[R][E];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const Chunk d = load_some<E>(rows[r] + k, there);
#pragma unroll
                for (int e = 0; e < E; e++) v[r][e] = (float)d[e];
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float f = (float)c[i][e];
#pragma unroll
                    for (int r = 0; r < R; r++) acc[r][i] += v[r][e] * f;
                }
        };
        auto load = [&](int64_t k, int there, Chunk (&d)[8]) {
#pragma unroll
            for (int i = 0; i < 8; i++)  // past the last output the last again
                d[i] = load_some<E>(w + min<int64_t>(j + i, job.out - 1) * job.w_stride + k, there);
        };
        Chunk c[8];
        int64_t k = lo + lane * E;
        auto there = [&](int64_t at) { return (int)max<int64_t>(0, min<int64_t>(E, hi - at)); };
        if (have) {
            load(k, there(k), c);
            while (k < hi) {
                const int64_t next = k + 64 * E;
                Chunk d[8] = {};
                if (next < hi) load(next, there(next), d);
                add(k, c, there(k));
#pragma unroll
                for (int i = 0; i < 8; i++) c[i] = d[i];
                k = next;
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                v[i] = acc[r][i];
#pragma unroll
                for (int mask = 1; mask < 64; mask <<= 1) v[i] += __shfl_xor(v[i], mask);
            }
            if (lane == r && r < job.rows && have) to(r, j, have, v);
        }
    }
}

// Whether a product is of few rows. Microseconds of k_few and of the tiles, IN_OUT: bf16 4,096 x 16,384 28 and 46 (1 row),
// 40 and 46 (8); 4,096 x 4,096 12.6 and 12.6 (2), 15.1 and 12.6 (4); 1,024 x 1,024 5.9 and 7.1 (2), 8.3 and 7.1 (4).
// float32, whose tiles read three parts of six products: 4,096 x 4,096 16.6 and 66 (1), 36.6 and 66 (16); OUT_IN 24 and 65
// (8), 54 and 65 (16), but 1,024 x 1,024 16.4 and 19.2 (8), 39 and 19.2 (16).
// Its runs: two workgroups a CU, or one where the columns give that many already and the second launch that adds the runs
// is not needed.
struct Few {
    bool is;
    int lanes_rows, runs;  // rows a lane has
    int64_t groups, run;
};

template <class T>
Few few_of(const wc_linear_args& a, int cus) {
    constexpr int64_t E = 16 / sizeof(T);
    const bool io = a.weight_layout == WC_WEIGHT_IN_OUT;
    Few f = {};
    f.is = sizeof(T) == 4 ? a.rows <= (io ? 16 : 8) : a.rows <= (a.width * a.out >= 1 << 25 ? 8 : 2);
    if (!f.is) return f;
    f.lanes_rows = a.rows <= 1 ? 1 : a.rows <= 2 ? 2 : a.rows <= 4 ? 4 : a.rows <= 8 ? 8 : 16;
    const int64_t each = io ? 8 * E : 8 * FEW_WAVES;
    f.groups = (a.out + each - 1) / each;
    const int64_t most = std::max<int64_t>(1, a.width / 1024);
    const int64_t want = f.groups * 4 >= int64_t(cus) * 3 ? 1 : (2 * int64_t(cus) + f.groups - 1) / f.groups;
    const int64_t runs = std::min(most, want);
    f.run = up((a.width + runs - 1) / runs, 512);
    f.runs = (int)((a.width + f.run - 1) / f.run);
    return f;
}

// ------------------------------------------------------------------ direct

// A float32 product made straight from memory, in how many runs along k, and the microseconds that it takes (within 20%
// from 64 x 64 x 64 to 1,024 x 1,024 x 1,024).
//
// Microseconds of it and of the tiles of parts: forward 567 x 129 x 128 4.3 and 12.1, 512 x 512 x 512 8.1 and 19, 64 x 4,096 x
// 4,096 40 and 65, 1,024 x 1,024 x 1,024 37 and 35, 8,192 x 64 x 8,192 265 and 135. Both gradients through a GELU, with
// the bias's: 8.3 and 23.4, 16.7 and 34.8, 161 and 104, 105 and 61; 4,096 x 128 x 128 18 and 32, 1,024 x 512 x 512 43 and 40.
// The slopes are computed again in each tile: 1.45 times the products' time.
struct DirectCut {
    int runs;
    int64_t run;
    double us;

    size_t bytes(int64_t n) const { return runs > 1 ? pad256(size_t(runs) * n * 4) : 0; }
};

inline DirectCut direct_cut(int64_t m, int64_t n, int64_t k, bool slopes, int cus) {
    const int64_t tiles = ((m + 31) / 32) * ((n + 31) / 32);
    DirectCut best = {1, k, -1};
    for (int64_t r = 1; r <= 64; r = r < 4 ? r + 1 : r * 3 / 2) {
        const int64_t run = std::max<int64_t>(8 * DIRECT_WAVES, up((k + r - 1) / r, 8 * DIRECT_WAVES)),
                      runs = std::max<int64_t>(1, (k + run - 1) / run);
        if (r > 1 && (run < 128 || tiles * runs > 2 * cus)) break;
        const double rounds = double(tiles * runs) / cus, each = 0.0035 + 0.006 * std::max(1.0, rounds),
                     us = 3.5 + 0.75 * std::max(0.0, rounds - 2.0) + double(std::min(run, k)) * each * (slopes ? 1.45 : 1.0) + (runs > 1 ? 4.5 : 0.0);
        if (best.us < 0 || us < best.us) best = {(int)runs, run, us};
    }
    return best;
}

// Fragments of a launch, and the rows of a product that they are (width or out is at most 2^20): 2^22 workgroups are 2^31
// threads, and a launch, which two products may share, holds fewer than 2^32.
constexpr int64_t MOST_DIRECT = int64_t(1) << 22;
inline int64_t direct_rows(int64_t n) { return 32 * (MOST_DIRECT / ((n + 31) / 32)); }

inline Direct direct_of(const DirectSide& a, const DirectSide& b, int64_t k, int act, const DirectCut& cut, float* part, float* sums) {
    const int64_t tiles_n = (b.outer + 31) / 32;
    return {a, b, k, cut.run, tiles_n, act, cut.runs, (unsigned)(((a.outer + 31) / 32) * tiles_n * cut.runs), part, sums};
}

// What adds the runs' products.
inline Product direct_parts(const Direct& d) {
    Product m = {};
    m.a.outer = d.a.outer;
    m.b.outer = d.b.outer;
    m.runs = d.runs;
    m.batches = 1;
    m.part = d.part;
    return m;
}
template <class Epilogue>
void direct_sum(const Direct& d, const Epilogue& e, hipStream_t s) {
    if (d.runs <= 1) return;
    const Product m = direct_parts(d);
    k_product_sum<<<dim3((uint32_t)((sum_chunks(m) + 63) / 64)), PRODUCT_BLOCK, 0, s>>>(m, sum_chunks(m), e);
}

// What the other way costs: its launches and steps at the sizes in question, and the copies in parts of so many elements.
inline bool direct_pays(double us, int products, double copied) {
    return us < (products > 1 ? 30.0 : 25.0) + copied * 10 / 4.5e6;
}

// ------------------------------------------------------------------ forward

struct LinearPlan {
    Few few;
    bool direct;
    DirectCut one;
    Laid x, w;
    Cut cut;
    int64_t k;
    size_t part, bytes;
};

template <class T>
LinearPlan linear_plan(const wc_linear_args& a, int cus) {
    constexpr int parts = Parts<T>::COUNT;
    LinearPlan p = {};
    const bool io = a.weight_layout == WC_WEIGHT_IN_OUT;
    p.few = few_of<T>(a, cus);
    if (p.few.is) {
        p.bytes = p.few.runs > 1 ? pad256(size_t(p.few.runs) * a.rows * a.out * 4) : 0;
        return p;
    }
    if (parts > 1) p.one = direct_cut(a.rows, a.out, a.width, false, cus);
    p.direct = parts > 1 && direct_pays(p.one.us, 1, double(a.rows + a.out) * a.width);
    if (p.direct) {
        p.bytes = p.one.bytes(a.rows * a.out);
        return p;
    }
    p.x = laid<T>(a.x, a.x_stride, a.rows, a.width);
    p.w = io ? laid<T>(a.weight, a.weight_stride, a.width, a.out) : laid<T>(a.weight, a.weight_stride, a.out, a.width);
    p.k = parts > 1 ? up(a.width, STEP) : a.width;
    p.cut = cut_of(a.rows, a.out, p.k, parts > 1 ? 6 : 1, cus);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += pad256(n);
        return here;
    };
    p.x.at = take(p.x.bytes(parts));
    p.w.at = take(p.w.bytes(parts));
    p.part = take(p.cut.bytes(a.rows * a.out));
    p.bytes = at;
    return p;
}

template <class T>
void linear(const wc_linear_args& a, int cus, hipStream_t s) {
    if (!a.rows) return;
    const LinearPlan p = linear_plan<T>(a, cus);
    char* w = (char*)a.workspace;
    const bool io = a.weight_layout == WC_WEIGHT_IN_OUT;
    const LayerEpilogue<T> e = {a.bias, a.bias_dtype == WC_DTYPE_F32, (const T*)a.residual, a.residual_stride,
                                a.pre, a.pre_stride, (T*)a.y, a.y_stride, a.act};
    if (p.few.is) {
        const FewJob job = {a.rows, a.width, a.out, a.x_stride, a.weight_stride, p.few.run, p.few.runs, (float*)w};
        const dim3 grid((uint32_t)(p.few.groups * p.few.runs));
        auto run = [&](auto rows) {
            if (io) k_few<T, rows(), true><<<grid, FEW_BLOCK, 0, s>>>((const T*)a.x, (const T*)a.weight, job, e);
            else if constexpr (rows() <= 8)
                k_few<T, rows(), false><<<grid, FEW_BLOCK, 0, s>>>((const T*)a.x, (const T*)a.weight, job, e);
        };
        if (p.few.lanes_rows == 1) run(std::integral_constant<int, 1>());
        else if (p.few.lanes_rows == 2) run(std::integral_constant<int, 2>());
        else if (p.few.lanes_rows == 4) run(std::integral_constant<int, 4>());
        else if (p.few.lanes_rows == 8) run(std::integral_constant<int, 8>());
        else if constexpr (sizeof(T) == 4) run(std::integral_constant<int, 16>());
        if (p.few.runs > 1) {
            Product m = {};
            m.a.outer = a.rows;
            m.b.outer = a.out;
            m.runs = p.few.runs;
            m.batches = 1;
            m.part = (float*)w;
            const int64_t chunks = a.rows * ((a.out + 7) / 8);
            k_product_sum<<<dim3((uint32_t)((chunks + 63) / 64)), PRODUCT_BLOCK, 0, s>>>(m, chunks, e);
        }
        return;
    }
    if constexpr (sizeof(T) == 4) {
        if (p.direct) {
            // (runs are of few fragments: all in one launch)
            const int64_t most = direct_rows(a.out);
            for (int64_t lo = 0; lo < a.rows; lo += most) {
                const Direct d = direct_of({(const float*)a.x + lo * a.x_stride, a.x_stride, std::min(most, a.rows - lo)},
                                           {(const float*)a.weight, a.weight_stride, a.out}, a.width, 0, p.one, (float*)w, nullptr);
                const auto el = e.from(lo);
                if (io) k_direct<false><<<dim3(d.blocks), DIRECT_BLOCK, 0, s>>>(d, el);
                else k_direct<true><<<dim3(d.blocks), DIRECT_BLOCK, 0, s>>>(d, el);
                direct_sum(d, el, s);
            }
            return;
        }
    }
    lay<T>(copy_of(p.x, {a.x, a.x_stride, a.rows, a.width}, w),
           copy_of(p.w, {a.weight, a.weight_stride, io ? a.width : a.out, io ? a.out : a.width}, w), cus, s);
    Product m = {};
    m.a = operand<T>(p.x, a.x, w, a.rows);
    m.b = operand<T>(p.w, a.weight, w, a.out);
    m.k = p.k;
    multiply<T>(m, p.cut, true, !io, (float*)(w + p.part), e, s);
}

// ----------------------------------------------------------------- backward

// d_pre = d_out act'(pre), eight columns of a row.
template <class T>
__device__ __forceinline__ void slope_values(const wc_linear_back_args& a, int64_t r, int64_t c, int have, float (&v)[8]) {
    load_n((const T*)a.d_out + r * a.d_out_stride + c, have, 0.f, v);
    if (a.act == WC_ACT_NONE) return;
    float z[8];
    load_n((const float*)a.pre + r * a.pre_stride + c, have, 0.f, z);
    act_slopes(z, a.act);
#pragma unroll
    for (int u = 0; u < 8; u++) v[u] = u < have ? v[u] * z[u] : 0.f;
}

// d_pre in the parts that its products read (`to` may be null: not needed), and its column sums, from the unrounded
// float32 values: 32 chunks of eight columns by eight rows a workgroup, over `per` rows. Memory bounds it: 16,384 x 4,096
// bf16 through a GELU 110 us for 537 MB, 4.9 TB/s. past (f16): marks the workgroups that found what f16 does not hold.
template <class T>
__global__ __launch_bounds__(256) void k_slope(wc_linear_back_args a, Source d, int64_t per, float* sums, uint32_t* past) {
    __shared__ float4 add[256][2];
    const int64_t c = (int64_t(blockIdx.x) * 32 + threadIdx.x % 32) * 8, lo = int64_t(blockIdx.y) * per;
    const int64_t rows = d.to ? d.to_rows : a.rows, hi = min(lo + per, rows);
    const int lane = threadIdx.x / 32, have = (int)min<int64_t>(8, a.out - c);
    float sum[8] = {};
    bool found = false;
    for (int64_t r = lo + lane; r < hi; r += 8) {
        float v[8] = {};
        if (r < a.rows && have > 0) {
            slope_values<T>(a, r, c, have, v);
#pragma unroll
            for (int u = 0; u < 8; u++) sum[u] += v[u];
            if constexpr (__is_same(T, f16))
#pragma unroll
                for (int u = 0; u < 8; u++) found |= fabsf(v[u]) > 65504.f && fabsf(v[u]) != INFINITY;
        }
        if (d.to && c < d.to_cols) put_parts<T>(d.to + 2 * (r * d.to_cols + c), d.plane, v);
    }
    if constexpr (__is_same(T, f16))
        if (past) {
            const int any = __syncthreads_or(found);
            if (threadIdx.x == 0) past[blockIdx.y * gridDim.x + blockIdx.x] = any;
        }
    if (!sums) return;
    add[threadIdx.x][0] = {sum[0], sum[1], sum[2], sum[3]};
    add[threadIdx.x][1] = {sum[4], sum[5], sum[6], sum[7]};
    __syncthreads();
    // one column a thread
    const int64_t j = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (j >= a.out) return;
    const float* one = (const float*)add + (threadIdx.x / 8) * 8 + threadIdx.x % 8;
    float s = 0.f;
#pragma unroll
    for (int u = 0; u < 8; u++) s += one[u * 32 * 8];
    sums[int64_t(blockIdx.y) * a.out + j] = s;
}

// A GELU's slope is up to 1.13, a SiLU's 1.10: of an f16 d_out from 58,000 on d_pre may pass f16's largest. Where the first
// pass marked any, all of it is written again by halves, and the products' results are doubled (rate); the halves of less
// than 2^-13 lose a bit, which is why it is done for these only. In the launch that copies x and the weight, whose `first`
// workgroups those are (both gradients of 4,099 x 1,153 x 567 57.4 us, 58.1 without it and with the forward pass's epilogue);
// with nothing to copy it is a launch more (4,096 x 256 x 1,024: 29.6 and 26.7).
struct Half {
    Source d;
    int64_t per;
    const uint32_t* past;
    int marks, across;
    float* rate;
};
static __global__ __launch_bounds__(256) void k_lay_half(Source one, Source two, unsigned first, wc_linear_back_args a, Half h) {
    if (blockIdx.x < first) return lay_chunks<f16>(one, two, blockIdx.x, first);
    const unsigned block = blockIdx.x - first;
    bool found = false;
    for (int k = threadIdx.x; k < h.marks; k += 256) found |= h.past[k] != 0;
    const int any = __syncthreads_or(found);
    if (block == 0 && threadIdx.x == 0) *h.rate = any ? 2.f : 1.f;
    if (!any) return;
    const int64_t c = (int64_t(block % h.across) * 32 + threadIdx.x % 32) * 8, lo = block / h.across * h.per, hi = min(lo + h.per, a.rows);
    const int have = (int)min<int64_t>(8, a.out - c);
    if (have <= 0) return;
    for (int64_t r = lo + threadIdx.x / 32; r < hi; r += 8) {
        float v[8];
        slope_values<f16>(a, r, c, have, v);
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] *= 0.5f;
        put_parts<f16>(h.d.to + 2 * (r * h.d.to_cols + c), h.d.plane, v);
    }
}

// The row blocks' column sums added in order: a sixteenth of them each group of sixteen threads.
struct ColumnSums {
    const float* sums;
    int64_t out;
    int blocks;
    float* to;
};
__device__ __forceinline__ void column_sums(const ColumnSums& c, int64_t block) {
    const float* sums = c.sums;
    const int64_t out = c.out;
    const int blocks = c.blocks;
    __shared__ float some[16][17];
    const int64_t j = block * 16 + threadIdx.x % 16;
    const int q = threadIdx.x / 16;
    float s = 0.f;
    if (j < out) {
        int k = q;
        for (; k + 48 < blocks; k += 64) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = sums[(k + 16 * u) * out + j];
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
        for (; k < blocks; k += 16) s += sums[k * out + j];
    }
    some[q][threadIdx.x % 16] = s;
    __syncthreads();
    if (q || j >= out) return;
    for (int u = 1; u < 16; u++) s += some[u][threadIdx.x];
    c.to[j] = s;
}
static __global__ __launch_bounds__(256) void k_slope_sum(ColumnSums c) { column_sums(c, blockIdx.x); }

// The weight gradient's runs and the bias's blocks, in one launch.
template <class Epilogue>
__global__ __launch_bounds__(PRODUCT_BLOCK) void k_back_sum(Product p, int64_t chunks, Epilogue epilogue, unsigned blocks,
                                                            ColumnSums c) {
    if (blockIdx.x < blocks) product_sum(p, chunks, epilogue, blockIdx.x);
    else column_sums(c, blockIdx.x - blocks);
}

struct LinearBackPlan {
    Laid d, x, w;
    Cut cut_x, cut_w;
    int64_t out_k, rows_k, per;
    int blocks;
    bool slope, direct;
    DirectCut one_x, one_w;
    size_t sums, past, part_x, part, bytes;
    int marks;  // of what f16 does not hold, a workgroup of k_slope each; 0: d_pre is no larger than d_out
    bool together;
};

template <class T>
LinearBackPlan linear_back_plan(const wc_linear_back_args& a, int cus) {
    constexpr int parts = Parts<T>::COUNT;
    LinearBackPlan p = {};
    const bool io = a.weight_layout == WC_WEIGHT_IN_OUT;
    if (parts > 1 && (a.d_weight || (a.d_x && !a.d_bias))) {  // (the bias's alone is column sums, and nothing to multiply)
        const bool slopes = a.act != WC_ACT_NONE;
        if (a.d_x) p.one_x = direct_cut(a.rows, a.width, a.out, slopes, cus);
        if (a.d_weight) p.one_w = direct_cut(a.width, a.out, a.rows, slopes, cus);
        const double copied = double(a.rows) * a.out + (a.d_x ? double(a.width) * a.out : 0.0) + (a.d_weight ? double(a.rows) * a.width : 0.0);
        p.direct = direct_pays(p.one_x.us + p.one_w.us, (a.d_x != nullptr) + (a.d_weight != nullptr), copied) &&
                   (!a.d_weight || ((a.width + 31) / 32) * ((a.out + 31) / 32) * p.one_w.runs <= MOST_DIRECT);
        if (p.direct) {
            p.part_x = 0;
            p.part = p.part_x + p.one_x.bytes(a.rows * a.width);
            p.sums = p.part + p.one_w.bytes(a.width * a.out);
            p.bytes = p.sums + p.one_w.bytes(a.out);
            return p;
        }
    }
    p.d = laid<T>(a.d_out, a.d_out_stride, a.rows, a.out);
    if (a.act != WC_ACT_NONE && !p.d.copy) {
        p.d.copy = true;
        p.d.rows = a.rows;
        p.d.cols = up(a.out, 8);
        p.d.pitch = 2 * p.d.cols;
        p.d.plane = p.d.pitch * p.d.rows;
    }
    const bool products = a.d_x || a.d_weight;
    p.slope = (p.d.copy && products) || a.d_bias;
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += pad256(n);
        return here;
    };
    if (products) p.d.at = take(p.d.bytes(parts));
    if (a.d_x) {
        p.w = io ? laid<T>(a.weight, a.weight_stride, a.width, a.out) : laid<T>(a.weight, a.weight_stride, a.out, a.width);
        p.w.at = take(p.w.bytes(parts));
        p.out_k = parts > 1 ? up(a.out, STEP) : a.out;
        p.cut_x = cut_of(a.rows, a.width, p.out_k, parts > 1 ? 6 : 1, cus);
    }
    if (a.d_weight) {
        p.x = laid<T>(a.x, a.x_stride, a.rows, a.width);
        p.x.at = take(p.x.bytes(parts));
        p.rows_k = parts > 1 ? up(a.rows, STEP) : a.rows;
        p.cut_w = cut_of(io ? a.width : a.out, io ? a.out : a.width, p.rows_k, parts > 1 ? 6 : 1, cus);
    }
    // Small tiles of both: one launch, whose second product starts where the first leaves CUs free.
    p.together = a.d_x && a.d_weight && a.rows && p.cut_x.f == p.cut_w.f && p.cut_x.f <= 2;
    const size_t px = a.d_x ? p.cut_x.bytes(a.rows * a.width) : 0, pw = a.d_weight ? p.cut_w.bytes(a.width * a.out) : 0;
    if (p.together) {
        p.part_x = take(px);
        p.part = take(pw);
    } else {
        p.part_x = p.part = take(std::max(px, pw));  // one after the other in it
    }
    if (p.slope) {
        const int64_t across = (a.out + 255) / 256;
        const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((a.rows + 31) / 32, 8 * int64_t(cus) / across + 1));
        p.per = up((std::max<int64_t>(p.d.copy ? p.d.rows : a.rows, 1) + blocks - 1) / blocks, 8);
        p.blocks = (int)((std::max<int64_t>(p.d.copy ? p.d.rows : a.rows, 1) + p.per - 1) / p.per);
        if (a.d_bias) p.sums = take(size_t(p.blocks) * a.out * 4);
        if (__is_same(T, f16) && products && a.rows && (a.act == WC_ACT_GELU || a.act == WC_ACT_SILU)) {
            p.marks = (int)((p.d.cols + 255) / 256) * p.blocks;
            p.past = take(4 * (size_t(p.marks) + 1));  // and the rate behind them
        }
    }
    p.bytes = at;
    return p;
}

template <class T>
void linear_back(const wc_linear_back_args& a, int cus, hipStream_t s) {
    const LinearBackPlan p = linear_back_plan<T>(a, cus);
    char* w = (char*)a.workspace;
    const bool io = a.weight_layout == WC_WEIGHT_IN_OUT, products = a.d_x || a.d_weight;
    if constexpr (sizeof(T) == 4) {
        if (p.direct) {
            const float* z = a.act == WC_ACT_NONE ? nullptr : a.pre;
            const float* d = (const float*)a.d_out;
            Direct dw = {};
            if (a.d_weight) {
                const DirectSide side = {d, a.d_out_stride, a.out, z, a.pre_stride}, x = {(const float*)a.x, a.x_stride, a.width};
                float* sums = !a.d_bias || p.one_w.runs == 1 ? a.d_bias : (float*)(w + p.sums);
                dw = direct_of(io ? x : side, io ? side : x, a.rows, a.act, p.one_w, (float*)(w + p.part), sums);
            }
            const GradEpilogue<float> ew = {(float*)a.d_weight, a.d_weight_stride, nullptr};
            // x's gradient in parts that a launch holds, the weight's beside the first
            const int64_t rows_x = a.d_x ? a.rows : 0, most = direct_rows(a.width);
            for (int64_t lo = 0; lo == 0 || lo < rows_x; lo += most) {
                Direct dx = {};
                if (rows_x)
                    dx = direct_of({d + lo * a.d_out_stride, a.d_out_stride, std::min(most, rows_x - lo), z ? z + lo * a.pre_stride : nullptr,
                                    a.pre_stride},
                                   {(const float*)a.weight, a.weight_stride, a.width}, a.out, a.act, p.one_x, (float*)(w + p.part_x),
                                   nullptr);
                const Direct beside = lo ? Direct{} : dw;
                const GradEpilogue<float> ex = {rows_x ? (float*)a.d_x + lo * a.d_x_stride : nullptr, a.d_x_stride, nullptr};
                const dim3 grid(dx.blocks + beside.blocks);
                if (!grid.x) return;
                if (io) k_direct_back<true><<<grid, DIRECT_BLOCK, 0, s>>>(dx, ex, beside, ew);
                else k_direct_back<false><<<grid, DIRECT_BLOCK, 0, s>>>(dx, ex, beside, ew);
                direct_sum(dx, ex, s);
            }
            if (dw.runs > 1) {
                const Product m = direct_parts(dw);
                const uint32_t blocks = (uint32_t)((sum_chunks(m) + 63) / 64);
                const ColumnSums bias = {dw.sums, a.out, dw.runs, a.d_bias};
                k_back_sum<<<dim3(blocks + (a.d_bias ? (uint32_t)((a.out + 15) / 16) : 0)), PRODUCT_BLOCK, 0, s>>>(
                    m, sum_chunks(m), ew, blocks, bias);
            }
            return;
        }
    }
    uint32_t* const past = p.marks ? (uint32_t*)(w + p.past) : nullptr;
    const Source d_pre = products ? copy_of(p.d, {}, w) : Source{};
    if (p.slope) {
        float* sums = a.d_bias ? (float*)(w + p.sums) : nullptr;
        const int64_t across = ((d_pre.to ? p.d.cols : a.out) + 255) / 256;
        k_slope<T><<<dim3((uint32_t)across, (uint32_t)p.blocks), 256, 0, s>>>(a, d_pre, p.per, sums, past);
    }
    const float* rate = past ? (const float*)(past + p.marks) : nullptr;
    const ColumnSums bias = {(const float*)(w + p.sums), a.out, p.blocks, a.d_bias};
    const uint32_t bias_blocks = a.d_bias ? (uint32_t)((a.out + 15) / 16) : 0;
    if (!a.d_weight || p.cut_w.runs == 1) {
        if (bias_blocks) k_slope_sum<<<dim3(bias_blocks), 256, 0, s>>>(bias);
    }
    if (!products) return;
    // copies of x and the weight, in one launch
    const Source to_x = copy_of(p.x, {a.x, a.x_stride, a.rows, a.width}, w),
                 to_w = copy_of(p.w, {a.weight, a.weight_stride, io ? a.width : a.out, io ? a.out : a.width}, w);
    if (!p.marks) {
        lay<T>(to_x, to_w, cus, s);
    } else if constexpr (__is_same(T, f16)) {
        const int64_t n = chunks_of(to_x, to_w);
        const unsigned first = n ? lay_grid(n, cus).x : 0;
        const Half h = {d_pre, p.per, past, p.marks, p.marks / p.blocks, (float*)(past + p.marks)};
        k_lay_half<<<dim3(first + (unsigned)p.marks), 256, 0, s>>>(to_x, to_w, first, a, h);
    }
    const bool with_x = a.d_x && a.rows;
    Product mx = {}, mw = {};
    if (with_x) {
        mx.a = operand<T>(p.d, a.d_out, w, a.rows);
        mx.b = operand<T>(p.w, a.weight, w, a.width);
        mx.k = p.out_k;
        mx = cut_product(segments_of<T>(mx), p.cut_x, (float*)(w + p.part_x));
    }
    const GradEpilogue<T> ex = {(T*)a.d_x, a.d_x_stride, rate};
    if (!a.d_weight) {
        if (with_x) multiply<T>(mx, p.cut_x, true, io, mx.part, ex, s);
        return;
    }
    const Operand16 x = operand<T>(p.x, a.x, w, a.width), d = operand<T>(p.d, a.d_out, w, a.out);
    mw.a = io ? x : d;
    mw.b = io ? d : x;
    mw.k = p.rows_k;
    mw = cut_product(segments_of<T>(mw), p.cut_w, (float*)(w + p.part));
    auto both = [&](const auto& ew) {
        typedef typename Parts<T>::type E;
        auto sums = [&] {
            const int64_t chunks = sum_chunks(mw);
            const uint32_t blocks = (uint32_t)((chunks + 63) / 64);
            if (p.cut_w.runs > 1) k_back_sum<<<dim3(blocks + bias_blocks), PRODUCT_BLOCK, 0, s>>>(mw, chunks, ew, blocks, bias);
        };
        const uint32_t nx = (uint32_t)(mx.tiles_m * mx.tiles_n * mx.runs), nw = (uint32_t)(mw.tiles_m * mw.tiles_n * mw.runs);
        auto together = [&](auto f) {
            if (io) k_products<E, f(), true><<<dim3(nx + nw), PRODUCT_BLOCK, 0, s>>>(mx, ex, nx, mw, ew);
            else k_products<E, f(), false><<<dim3(nx + nw), PRODUCT_BLOCK, 0, s>>>(mx, ex, nx, mw, ew);
        };
        if (with_x && p.together) {
            if (p.cut_x.f == 2) together(std::integral_constant<int, 2>());
            else together(std::integral_constant<int, 1>());
            if (p.cut_x.runs > 1)
                k_product_sum<<<dim3((uint32_t)((sum_chunks(mx) + 63) / 64)), PRODUCT_BLOCK, 0, s>>>(mx, sum_chunks(mx), ex);
        } else {
            if (with_x) multiply<T>(mx, p.cut_x, true, io, mx.part, ex, s);
            if (p.cut_w.f == 4) product_of<E, 4>(mw, false, false, ew, s);
            else if (p.cut_w.f == 3) product_of<E, 3>(mw, false, false, ew, s);
            else if (p.cut_w.f == 2) product_of<E, 2>(mw, false, false, ew, s);
            else product_of<E, 1>(mw, false, false, ew, s);
        }
        sums();
    };
    if (a.grad_dtype == a.dtype) {
        both(GradEpilogue<T>{(T*)a.d_weight, a.d_weight_stride, rate});
    } else if constexpr (Parts<T>::COUNT == 1) {
        both(GradEpilogue<float>{(float*)a.d_weight, a.d_weight_stride, rate});
    }
}

}  // namespace
}  // namespace learn
}  // namespace wc
