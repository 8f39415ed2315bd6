// A matrix's singular values brought towards 1 by Newton-Schulz products (include/wc_learn.h).
//
//   X = U / (|U| + eps);  a few times: A = X X^T, B = b A + c A A, X = a X + B X  (X^T X and X B for a tall matrix)
//
// A and A A are symmetric: only tiles on and above the diagonal are computed, and written twice.
//
// X, A and B are held as sums of two f16 (22 bits), times 2^10: no element of X or A is larger than the largest singular
// value and its square, so that nothing overflows below 60, and an element of 2^-13 still has all its bits. A product is
// then three matrix products: the one of the two small parts is left out.
//
// For a bf16 result one product of the large parts is enough, with A and B in one f16 (11 bits), but X stays in 22: its
// rounding would fall on every direction, on small singular values that grow 500-fold too, where A's and B's fall on
// what is large already. A gradient with three large directions and 256 x 1,024 with 11-bit X comes out 8e-3 off (of its
// norm; all of it in bf16, 7e-2), with 22-bit X 9e-5; a random matrix 1.7e-3, as much as the result's own rounding.
// Up to 128 rows or columns (2.7e-3 at 40 x 200) the three products cost next to nothing, and are taken.
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
    __device__ __forceinline__ void get(int planes, int batch_of, int64_t i, int64_t j, float (&v)[8]) const {
        const f16* from = p + batch_of * batch + i * pitch + j;
        const f16x8 hi = *(const f16x8*)from;
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = (float)hi[u];
        if (planes > 1) {
            const f16x8 lo = *(const f16x8*)(from + plane);
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] += (float)lo[u];
        }
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
    __device__ __forceinline__ void operator()(int batch, int64_t i, int64_t j, int n, float (&v)[8]) const {
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] *= alpha;
        if (from.p) {
            float x[8];
            from.get(from_planes, batch, i, j, x);
#pragma unroll
            for (int u = 0; u < 8; u++) v[u] += beta * x[u];
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

struct Plan {
    int planes, segments, blocks;  // planes of A and B, and of X in products; X has two
    int64_t small, pitch, pitch_small, x_plane, a_plane;  // elements
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
    p.pitch = up(o.width, 8);
    p.pitch_small = up(p.small, 8);
    p.x_plane = o.rows * p.pitch;
    p.a_plane = p.small * p.pitch_small;
    p.gram = cut_of(p.small, p.small, large, p.segments, cus, o.batch, true);
    p.square = cut_of(p.small, p.small, p.small, p.segments, cus, o.batch, true);
    p.step = cut_of(o.rows, o.width, p.small, p.segments, cus, o.batch);
    const int64_t chunks = o.rows * (p.pitch / 8);
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
    p.part = take(std::max({p.gram.bytes(o.batch * p.small * p.small), p.square.bytes(o.batch * p.small * p.small),
                            p.step.bytes(o.batch * o.rows * o.width)}));
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

template <class T>
void start(const wc_orthogonalise_args& o, const Plan& p, const Held16& x, hipStream_t s) {
    const Update<T> u = {(const T*)o.update, o.update_stride, o.update_batch, o.rows, o.width};
    double* sums = (double*)((char*)o.workspace + p.sums);
    const dim3 grid((uint32_t)p.blocks, (uint32_t)o.batch);
    k_squares<T><<<grid, 256, 0, s>>>(u, sums);
    const int64_t chunks = o.rows * (p.pitch / 8);
    const dim3 wide((uint32_t)std::min<int64_t>((chunks + 255) / 256, 4096), (uint32_t)o.batch);
    k_start<T><<<wide, 256, 0, s>>>(u, sums, p.blocks, o.eps, x, 2);
}

}  // namespace

size_t orthogonalise_scratch(const wc_orthogonalise_args& o, int cus) { return plan_of(o, cus).bytes; }

void launch_orthogonalise(const wc_orthogonalise_args& o, int cus, hipStream_t s) {
    if (!o.batch) return;
    const Plan p = plan_of(o, cus);
    char* w = (char*)o.workspace;
    Held16 x[2], a = {(f16*)(w + p.a), p.pitch_small, p.a_plane, p.a_plane * p.planes}, b = a;
    b.p = (f16*)(w + p.b);
    for (int k = 0; k < 2; k++) x[k] = {(f16*)(w + p.x[k]), p.pitch, p.x_plane, p.x_plane * 2};
    if (o.dtype == WC_DTYPE_F32) start<float>(o, p, x[0], s);
    else if (o.dtype == WC_DTYPE_F16) start<f16>(o, p, x[0], s);
    else start<bf16>(o, p, x[0], s);

    const bool tall = o.rows > o.width;
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
        // a X + B X, or X B
        const Operand16 ob = operand(b, p.planes, p.small), ox = operand(from, p.planes, tall ? o.rows : o.width);
        m.a = tall ? ox : ob;
        m.b = tall ? ob : ox;
        e.from = from;
        e.to = to;
        e.from_planes = e.to_planes = 2;
        e.alpha = 1.f / HELD;
        e.beta = o.a;
        if (k + 1 == o.steps) {
            e.alpha *= o.scale / HELD;
            e.beta *= o.scale / HELD;
            e.out = o.out;
            e.out_dtype = o.out_dtype;
            e.out_stride = o.out_stride;
            e.out_batch = o.out_batch;
        }
        launch_product<f16>(m, p.step, true, tall, part, e, s);
    }
}

}  // namespace learn
}  // namespace wc
