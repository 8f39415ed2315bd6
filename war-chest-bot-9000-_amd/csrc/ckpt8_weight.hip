// The weight gradient from activations kept in 8 bits, on the matrix cores (include/wc_learn.h).
#include <algorithm>

#include "ckpt8_dev.h"

namespace wc {
namespace learn {
namespace {

constexpr int BLOCK = 256, TILE = 64, DEPTH = 32, LD = DEPTH + 8;

typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The operand's type and how many parts a gradient element is taken in: a
// float32 is the sum of three bf16 (8 + 8 + 8 mantissa bits), whose products
// with a kept value (8 bits) are exact.
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


// One 64 x 64 tile of weight over one run of rows; part: runs x width x out.
template <class T>
__global__ __launch_bounds__(BLOCK) void k_weight(wc_ckpt_weight_args a, int64_t run, float* part) {
    typedef typename Operand<T>::type E;
    typedef E E8 __attribute__((ext_vector_type(8)));
    constexpr int PARTS = Operand<T>::PARTS;
    __shared__ __align__(16) E as[TILE][LD];
    __shared__ __align__(16) E bs[PARTS][TILE][LD];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int64_t i0 = int64_t(blockIdx.x) * TILE, j0 = int64_t(blockIdx.y) * TILE;
    const int64_t lo = int64_t(blockIdx.z) * run, hi = min(lo + run, a.rows);
    const int kk = t >> 3, cc = (t & 7) * 8;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    const int na = (int)min<int64_t>(8, max<int64_t>(0, a.width - i0 - cc));
    const int nb = (int)min<int64_t>(8, max<int64_t>(0, a.out - j0 - cc));
    f32x4 acc[2][2] = {};
    for (int64_t k0 = lo; k0 < hi; k0 += DEPTH) {
        const int64_t r = k0 + kk;
        float z[8] = {}, g[8] = {};
        if (r < hi && na > 0) {
            const float step = step_of(a.exps[r * a.exps_stride + ((i0 + cc) >> 5)]);
            for (int k = 0; k < na; k++) z[k] = act_value(held<E>((float)a.q[r * a.q_stride + i0 + cc + k] * step), a.act);
        }
        if (r < hi) load_n((const T*)a.grad + r * a.grad_stride + j0 + cc, nb, 0.f, g);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 8; k++) {
            as[cc + k][kk] = (E)z[k];
            float rest = g[k];
#pragma unroll
            for (int p = 0; p < PARTS; p++) {
                const E e = (E)rest;
                bs[p][cc + k][kk] = e;
                rest -= (float)e;
            }
        }
        __syncthreads();
        E8 fa[2], fb[2];
#pragma unroll
        for (int m = 0; m < 2; m++) fa[m] = *(const E8*)&as[wi + 16 * m + (lane & 15)][(lane >> 4) * 8];
#pragma unroll
        for (int p = 0; p < PARTS; p++) {
#pragma unroll
            for (int n = 0; n < 2; n++) fb[n] = *(const E8*)&bs[p][wj + 16 * n + (lane & 15)][(lane >> 4) * 8];
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int n = 0; n < 2; n++) acc[m][n] = mfma(fa[m], fb[n], acc[m][n]);
        }
    }
#pragma unroll
    for (int m = 0; m < 2; m++)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int64_t i = i0 + wi + 16 * m + (lane >> 4) * 4 + k, j = j0 + wj + 16 * n + (lane & 15);
                if (i < a.width && j < a.out) part[(int64_t(blockIdx.z) * a.width + i) * a.out + j] = acc[m][n][k];
            }
}

template <class W>
__global__ __launch_bounds__(BLOCK) void k_weight_sum(const float* part, int runs, int64_t width, int64_t out,
                                                      W* weight, int64_t stride) {
    const int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x;
    if (i >= width * out) return;
    float s = 0.f;
    for (int k = 0; k < runs; k++) s += part[k * width * out + i];
    weight[i / out * stride + i % out] = (W)s;
}

// Column sums of grad over one run of rows, and their sum.
template <class T>
__global__ __launch_bounds__(BLOCK) void k_bias(const T* grad, int64_t stride, int64_t rows, int64_t out, int64_t run,
                                                float* part) {
    const int64_t j = int64_t(blockIdx.x) * BLOCK + threadIdx.x;
    if (j >= out) return;
    const int64_t lo = int64_t(blockIdx.y) * run, hi = min(lo + run, rows);
    float s = 0.f;
    for (int64_t r = lo; r < hi; r++) s += (float)grad[r * stride + j];
    part[int64_t(blockIdx.y) * out + j] = s;
}

constexpr int BIAS_RUNS = 64;

int runs_of(const wc_ckpt_weight_args& a, int cus) {
    const int64_t tiles = ((a.width + TILE - 1) / TILE) * ((a.out + TILE - 1) / TILE);
    const int64_t want = std::max<int64_t>(1, 4 * cus / tiles), most = std::max<int64_t>(1, a.rows / 256);
    return (int)std::min(want, most);
}

template <class T>
void weight(const wc_ckpt_weight_args& a, int cus, hipStream_t s) {
    const int runs = runs_of(a, cus);
    const int64_t run = ((a.rows + runs - 1) / runs + DEPTH - 1) / DEPTH * DEPTH;
    float* part = (float*)a.workspace;
    float* bias = (float*)((uint8_t*)a.workspace + pad256(size_t(runs) * a.width * a.out * 4));
    k_weight<T><<<dim3((uint32_t)((a.width + TILE - 1) / TILE), (uint32_t)((a.out + TILE - 1) / TILE), runs), BLOCK, 0,
                  s>>>(a, run, part);
    const dim3 g((uint32_t)((a.width * a.out + BLOCK - 1) / BLOCK));
    if (a.weight_dtype == WC_DTYPE_F32)
        k_weight_sum<float><<<g, BLOCK, 0, s>>>(part, runs, a.width, a.out, (float*)a.weight, a.weight_stride);
    else
        k_weight_sum<T><<<g, BLOCK, 0, s>>>(part, runs, a.width, a.out, (T*)a.weight, a.weight_stride);
    if (a.bias) {
        const int64_t brun = (a.rows + BIAS_RUNS - 1) / BIAS_RUNS;
        const dim3 bg((uint32_t)((a.out + BLOCK - 1) / BLOCK), BIAS_RUNS);
        k_bias<T><<<bg, BLOCK, 0, s>>>((const T*)a.grad, a.grad_stride, a.rows, a.out, brun, bias);
        k_weight_sum<float><<<dim3((uint32_t)((a.out + BLOCK - 1) / BLOCK)), BLOCK, 0, s>>>(bias, BIAS_RUNS, 1, a.out,
                                                                                           a.bias, a.out);
    }
}

}  // namespace

size_t ckpt_weight_scratch(const wc_ckpt_weight_args& a, int cus) {
    return pad256(size_t(runs_of(a, cus)) * a.width * a.out * 4) + pad256(size_t(BIAS_RUNS) * a.out * 4);
}

void launch_ckpt_weight(const wc_ckpt_weight_args& a, int cus, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) weight<float>(a, cus, s);
    else if (a.dtype == WC_DTYPE_F16) weight<f16>(a, cus, s);
    else weight<bf16>(a, cus, s);
}

}  // namespace learn
}  // namespace wc
