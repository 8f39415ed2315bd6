// The residual update between two norms, forward and backward (include/wc_learn.h).
#include <algorithm>

#include "learn.h"
#include "learn_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

// Eight values of a parameter vector from column c; `fill` where there is none.
__device__ __forceinline__ void load_param(const void* p, int dtype, int64_t c, int n, float fill, float (&v)[8]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = fill;
    } else if (dtype == WC_DTYPE_F32) {
        load_n((const float*)p + c, n, 0.f, v);
    } else if (dtype == WC_DTYPE_F16) {
        load_n((const f16*)p + c, n, 0.f, v);
    } else {
        load_n((const bf16*)p + c, n, 0.f, v);
    }
}

// Sums over the G threads that hold a row, the same bits in each of them: a
// butterfly inside a wavefront, then the wavefronts' sums in order through LDS.
// Two slots alternate, so one barrier per sum is enough: a wavefront writes a
// slot again only after a barrier that every reader of its last use has passed.
// `lds` is the row's own slots: a workgroup of several such rows has as many.
template <int G>
struct RowSum {
    static constexpr int WAVES = G > 64 ? G / 64 : 1;
    typedef float2 Slots[2][WAVES];
    Slots& lds;
    int slot = 0;

    __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
        for (int mask = (G < 64 ? G : 64) / 2; mask; mask >>= 1) {
            a += __shfl_xor(a, mask);
            b += __shfl_xor(b, mask);
        }
        if constexpr (G > 64) {
            if ((threadIdx.x & 63) == 0) lds[slot][threadIdx.x % G >> 6] = make_float2(a, b);
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                a += lds[slot][w].x;
                b += lds[slot][w].y;
            }
            slot ^= 1;
        }
        return make_float2(a, b);
    }
};

// act(g), and its slope in *d.
__device__ __forceinline__ float gate_of(float g, int act, float* d) {
    if (act == WC_GATE_SIGMOID) {
        const float s = 1.f / (1.f + expf(-g));
        *d = s * (1.f - s);
        return s;
    }
    if (act == WC_GATE_TANH) {
        const float t = tanhf(g);
        *d = 1.f - t * t;
        return t;
    }
    *d = 1.f;
    return g;
}

template <int G>
constexpr int block_of() {
    return G < 256 ? 256 : G;
}

// Mean (0 for RMS) and 1 / sqrt(variance + eps) of the row's values, from two
// passes over registers.
template <int G, int NV>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][8], const int (&n)[NV], int width, bool layer,
                                            float eps, RowSum<G>& sum) {
    float mean = 0.f;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) s += v[k][i];  // 0 beyond the row's end
        mean = sum(s, 0.f).x / (float)width;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float d = i < n[k] ? v[k][i] - mean : 0.f;
            q += d * d;
        }
    const float var = sum(q, 0.f).x / (float)width;
    return make_float2(mean, 1.f / sqrtf(var + eps));
}

template <class T, int G, int NV>
__global__ __launch_bounds__(block_of<G>()) void k_norm(wc_norm_args a) {
    constexpr int PER = block_of<G>() / G;
    __shared__ typename RowSum<G>::Slots lds[PER];
    RowSum<G> sum{lds[threadIdx.x / G]};
    const int lane = threadIdx.x % G;
    const int width = (int)a.width;
    int n[NV];
#pragma unroll
    for (int k = 0; k < NV; k++) n[k] = min(8, max(0, width - 8 * (lane + k * G)));
    for (int64_t r0 = int64_t(blockIdx.x) * PER; r0 < a.rows; r0 += int64_t(gridDim.x) * PER) {
        const int64_t row = r0 + threadIdx.x / G;
        const bool here = row < a.rows;  // the others go along: the sums are taken by whole wavefronts
        const int64_t r = here ? row : a.rows - 1;
        float u[NV][8], x[NV][8];
#pragma unroll
        for (int k = 0; k < NV; k++) load_n((const T*)a.block + r * a.block_stride + 8 * (lane + k * G), n[k], 0.f, u[k]);
#pragma unroll
        for (int k = 0; k < NV; k++) load_n((const T*)a.stream + r * a.stream_stride + 8 * (lane + k * G), n[k], 0.f, x[k]);
        const float2 s1 = row_stats<G, NV>(u, n, width, a.norm == WC_NORM_LAYER, a.eps, sum);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = 8 * (lane + k * G);
            float g[8], b[8], w[8];
            load_param(a.post_gain, a.param_dtype, c, n[k], 1.f, g);
            load_param(a.post_bias, a.param_dtype, c, n[k], 0.f, b);
            if (a.gate && a.gate_stride) load_n((const T*)a.gate + r * a.gate_stride + c, n[k], 0.f, w);
            else load_param(a.gate, a.param_dtype, c, n[k], 1.f, w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                float slope;
                const float gate = a.gate ? gate_of(w[i], a.gate_act, &slope) : 1.f;
                x[k][i] = i < n[k] ? x[k][i] + a.scale * gate * ((u[k][i] - s1.x) * s1.y * g[i] + b[i]) : 0.f;
            }
            if (here) store_n((T*)a.new_stream + r * a.new_stream_stride + c, n[k], x[k]);
        }
        const float2 s2 = row_stats<G, NV>(x, n, width, a.norm == WC_NORM_LAYER, a.eps, sum);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = 8 * (lane + k * G);
            float g[8], b[8];
            load_param(a.pre_gain, a.param_dtype, c, n[k], 1.f, g);
            load_param(a.pre_bias, a.param_dtype, c, n[k], 0.f, b);
#pragma unroll
            for (int i = 0; i < 8; i++) g[i] = (x[k][i] - s2.x) * s2.y * g[i] + b[i];
            if (here) store_n((T*)a.out + r * a.out_stride + c, n[k], g);
        }
        if (a.stats && here && lane == 0) ((float4*)a.stats)[r] = make_float4(s1.x, s1.y, s2.x, s2.y);
    }
}

// The parameters' gradients in the order their column sums are kept.
constexpr int SUMS = 5;  // post gain, post bias, gate vector, pre gain, pre bias

// One workgroup takes rows blockIdx.x * PER, + gridDim.x * PER, ... and writes
// its column sums to part[blockIdx.x][SUMS][width].
template <class T, int G, int NV>
__global__ __launch_bounds__(block_of<G>()) void k_norm_back(wc_norm_back_args a, float* part) {
    constexpr int PER = block_of<G>() / G;
    __shared__ typename RowSum<G>::Slots lds[PER];
    __shared__ float cols[PER > 1 ? G * NV * 8 : 1];
    RowSum<G> sum{lds[threadIdx.x / G]};
    const int lane = threadIdx.x % G;
    const int width = (int)a.width;
    const bool layer = a.norm == WC_NORM_LAYER, vector = a.gate && !a.gate_stride;
    const float inv = 1.f / (float)width;
    int n[NV];
    float acc[SUMS][NV][8];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        n[k] = min(8, max(0, width - 8 * (lane + k * G)));
#pragma unroll
        for (int q = 0; q < SUMS; q++)
#pragma unroll
            for (int i = 0; i < 8; i++) acc[q][k][i] = 0.f;
    }
    for (int64_t r0 = int64_t(blockIdx.x) * PER; r0 < a.rows; r0 += int64_t(gridDim.x) * PER) {
        const int64_t row = r0 + threadIdx.x / G;
        const bool here = row < a.rows;
        const int64_t r = here ? row : a.rows - 1;
        const float4 st = ((const float4*)a.stats)[r];
        // norm of the block, the update's factor, and the stream after it, as the forward computed them
        float uh[NV][8], xh[NV][8], fac[NV][8], dx[NV][8];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = 8 * (lane + k * G);
            float g[8], b[8], w[8], d[8], pg[8];
            load_n((const T*)a.block + r * a.block_stride + c, n[k], 0.f, uh[k]);
            load_n((const T*)a.stream + r * a.stream_stride + c, n[k], 0.f, xh[k]);
            if (a.d_out) load_n((const T*)a.d_out + r * a.d_out_stride + c, n[k], 0.f, d);
            load_param(a.post_gain, a.param_dtype, c, n[k], 1.f, g);
            load_param(a.post_bias, a.param_dtype, c, n[k], 0.f, b);
            load_param(a.pre_gain, a.param_dtype, c, n[k], 1.f, pg);
            if (a.gate && a.gate_stride) load_n((const T*)a.gate + r * a.gate_stride + c, n[k], 0.f, w);
            else load_param(a.gate, a.param_dtype, c, n[k], 1.f, w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = i < n[k];
                float slope;
                const float gate = a.gate ? gate_of(w[i], a.gate_act, &slope) : 1.f;
                uh[k][i] = in ? (uh[k][i] - st.x) * st.y : 0.f;
                fac[k][i] = a.scale * gate;
                const float x = xh[k][i] + fac[k][i] * (uh[k][i] * g[i] + b[i]);
                xh[k][i] = in ? (x - st.z) * st.w : 0.f;
                const float dh = a.d_out && in ? d[i] : 0.f;
                if (here) {
                    acc[3][k][i] += dh * xh[k][i];
                    acc[4][k][i] += dh;
                }
                dx[k][i] = dh * pg[i];
                s1 += dx[k][i];
                s2 += dx[k][i] * xh[k][i];
            }
        }
        float2 m = sum(s1, s2);
        m.x *= inv;
        m.y *= inv;
        if (!layer) m.x = 0.f;
        s1 = s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = 8 * (lane + k * G);
            float g[8], b[8], w[8], d[8], dg[8];
            if (a.d_new_stream) load_n((const T*)a.d_new_stream + r * a.d_new_stream_stride + c, n[k], 0.f, d);
            load_param(a.post_gain, a.param_dtype, c, n[k], 1.f, g);
            load_param(a.post_bias, a.param_dtype, c, n[k], 0.f, b);
            if (a.gate && a.gate_stride) load_n((const T*)a.gate + r * a.gate_stride + c, n[k], 0.f, w);
            else load_param(a.gate, a.param_dtype, c, n[k], 1.f, w);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const bool in = i < n[k];
                float slope = 0.f;
                if (a.gate) gate_of(w[i], a.gate_act, &slope);
                const float v = st.w * (dx[k][i] - m.x - xh[k][i] * m.y) + (a.d_new_stream ? d[i] : 0.f);
                d[i] = v;
                const float dn = in ? fac[k][i] * v : 0.f;
                dg[i] = a.scale * slope * v * (uh[k][i] * g[i] + b[i]);
                if (here) {
                    acc[0][k][i] += dn * uh[k][i];
                    acc[1][k][i] += dn;
                    if (vector) acc[2][k][i] += in ? dg[i] : 0.f;
                }
                dx[k][i] = dn * g[i];
                s1 += dx[k][i];
                s2 += dx[k][i] * uh[k][i];
            }
            if (here) {
                store_n((T*)a.d_stream + r * a.d_stream_stride + c, n[k], d);
                if (a.d_gate && a.gate_stride) store_n((T*)a.d_gate + r * a.d_gate_stride + c, n[k], dg);
            }
        }
        m = sum(s1, s2);
        m.x *= inv;
        m.y *= inv;
        if (!layer) m.x = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int64_t c = 8 * (lane + k * G);
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = st.y * (dx[k][i] - m.x - uh[k][i] * m.y);
            if (here) store_n((T*)a.d_block + r * a.d_block_stride + c, n[k], o);
        }
    }
    // the workgroup's column sums: its row groups in order
    for (int q = 0; q < SUMS; q++) {
        float* to = part + (size_t(blockIdx.x) * SUMS + q) * width;
        if constexpr (PER == 1) {
#pragma unroll
            for (int k = 0; k < NV; k++)
                if (n[k] > 0) store_n(to + 8 * (lane + k * G), n[k], acc[q][k]);
        } else {
            for (int g = 0; g < PER; g++) {
                __syncthreads();
                if ((int)threadIdx.x / G == g) {
#pragma unroll
                    for (int k = 0; k < NV; k++)
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const int c = 8 * (lane + k * G) + i;
                            cols[c] = (g ? cols[c] : 0.f) + acc[q][k][i];
                        }
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < width; c += block_of<G>()) to[c] = cols[c];
        }
    }
}

struct ColumnSums {
    float* out[SUMS];
};

// Sums the workgroups' column sums in order: 64 columns by 4 interleaved runs.
__global__ __launch_bounds__(256) void k_norm_cols(const float* part, int blocks, int width, ColumnSums o) {
    __shared__ float lds[4][64];
    const int q = blockIdx.y, c = blockIdx.x * 64 + (threadIdx.x & 63), run = threadIdx.x >> 6;
    if (!o.out[q]) return;
    float s = 0.f;
    if (c < width)
        for (int b = run; b < blocks; b += 4) s += part[(size_t(b) * SUMS + q) * width + c];
    lds[run][threadIdx.x & 63] = s;
    __syncthreads();
    if (run == 0 && c < width) o.out[q][c] = (lds[0][c & 63] + lds[1][c & 63]) + (lds[2][c & 63] + lds[3][c & 63]);
}

// Threads per row: eight channels each, a power of two.
int group_of(int64_t width) {
    int g = 8;
    while (g < 1024 && 8 * g < width) g *= 2;
    return g;
}

int back_blocks(int64_t rows, int64_t width, int cus) {
    const int g = group_of(width), per = g < 256 ? 256 / g : 1;
    const int64_t want = (rows + per - 1) / per;
    return (int)std::max<int64_t>(1, std::min<int64_t>(want, int64_t(cus) * std::max(1, 1024 / std::max(256, g))));
}

template <class T, int G, int NV>
void norm_at(const wc_norm_args& a, int cus, hipStream_t s) {
    constexpr int PER = block_of<G>() / G;
    const int64_t want = (a.rows + PER - 1) / PER;
    k_norm<T, G, NV><<<dim3((uint32_t)std::min<int64_t>(want, 1 << 20)), block_of<G>(), 0, s>>>(a);
}

template <class T, int G, int NV>
void back_at(const wc_norm_back_args& a, int blocks, hipStream_t s) {
    k_norm_back<T, G, NV><<<dim3(blocks), block_of<G>(), 0, s>>>(a, (float*)a.workspace);
}

template <class T>
void norm(const wc_norm_args& a, int cus, hipStream_t s) {
    switch (group_of(a.width)) {
        case 8: return norm_at<T, 8, 1>(a, cus, s);
        case 16: return norm_at<T, 16, 1>(a, cus, s);
        case 32: return norm_at<T, 32, 1>(a, cus, s);
        case 64: return norm_at<T, 64, 1>(a, cus, s);
        case 128: return norm_at<T, 128, 1>(a, cus, s);
        case 256: return norm_at<T, 256, 1>(a, cus, s);
        case 512: return norm_at<T, 512, 1>(a, cus, s);
        default: return a.width <= 8192 ? norm_at<T, 1024, 1>(a, cus, s) : norm_at<T, 1024, 2>(a, cus, s);
    }
}

template <class T>
void norm_back(const wc_norm_back_args& a, int cus, hipStream_t s) {
    const int blocks = back_blocks(a.rows, a.width, cus);
    switch (group_of(a.width)) {
        case 8: back_at<T, 8, 1>(a, blocks, s); break;
        case 16: back_at<T, 16, 1>(a, blocks, s); break;
        case 32: back_at<T, 32, 1>(a, blocks, s); break;
        case 64: back_at<T, 64, 1>(a, blocks, s); break;
        case 128: back_at<T, 128, 1>(a, blocks, s); break;
        case 256: back_at<T, 256, 1>(a, blocks, s); break;
        case 512: back_at<T, 512, 1>(a, blocks, s); break;
        default:
            if (a.width <= 8192) back_at<T, 1024, 1>(a, blocks, s);
            else back_at<T, 1024, 2>(a, blocks, s);
    }
    const ColumnSums o = {{a.d_post_gain, a.d_post_bias, a.gate && !a.gate_stride ? (float*)a.d_gate : nullptr,
                           a.d_pre_gain, a.d_pre_bias}};
    k_norm_cols<<<dim3((uint32_t)(a.width + 63) / 64, SUMS), 256, 0, s>>>((const float*)a.workspace, blocks,
                                                                        (int)a.width, o);
}

}  // namespace

size_t norm_back_scratch(const wc_norm_back_args& a, int cus) {
    return pad256(size_t(back_blocks(a.rows, a.width, cus)) * SUMS * size_t(a.width) * 4);
}

void launch_norm(const wc_norm_args& a, int cus, hipStream_t s) {
    if (!a.rows) return;
    if (a.dtype == WC_DTYPE_F32) norm<float>(a, cus, s);
    else if (a.dtype == WC_DTYPE_F16) norm<f16>(a, cus, s);
    else norm<bf16>(a, cus, s);
}

void launch_norm_back(const wc_norm_back_args& a, int cus, hipStream_t s) {
    if (a.dtype == WC_DTYPE_F32) norm_back<float>(a, cus, s);
    else if (a.dtype == WC_DTYPE_F16) norm_back<f16>(a, cus, s);
    else norm_back<bf16>(a, cus, s);
}

}  // namespace learn
}  // namespace wc
