// Activations kept in 8 bits: writing, reading, and the activation's backward (include/wc_learn.h).
//
// One pass each, bound by memory: five bytes a value in 16 bits (write: the
// value in, 8 bits and act(value) out; backward: 8 bits and the gradient in, the
// gradient out) against some 30 operations for GELU. A thread takes eight values,
// 16 bytes in 16 bits; a group of 32 is four neighbouring lanes, whose largest
// magnitude two exchanges find. 16,384 x 8,192 bf16 with GELU on one MI355X:
// write 112 us (6.0 TB/s), backward 133 us (5.0 TB/s); a large copy moves 5.09.
#include <algorithm>

#include "ckpt8_dev.h"

namespace wc {
namespace learn {
namespace {

constexpr int BLOCK = 256;

typedef int8_t i8x8 __attribute__((ext_vector_type(8), aligned(1)));

// Where a thread's eight channels are: rows are padded to whole groups of 32,
// so that a group is four neighbouring lanes.
struct Place {
    int64_t row, col;
    int n;  // channels of the eight that the row has
};

__device__ __forceinline__ Place place_of(int64_t i, int64_t per_row, int64_t width) {
    Place p;
    p.row = i / per_row;
    p.col = (i - p.row * per_row) * 8;
    p.n = (int)min<int64_t>(8, max<int64_t>(0, width - p.col));
    return p;
}

template <class T>
__global__ __launch_bounds__(BLOCK) void k_ckpt_write(wc_ckpt_args a, int64_t per_row) {
    const int64_t total = a.rows * per_row;
    for (int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x; i < total; i += int64_t(gridDim.x) * BLOCK) {
        const Place p = place_of(i, per_row, a.width);
        float v[8];
        load_n((const T*)a.x + p.row * a.x_stride + p.col, p.n, 0.f, v);
        // the largest magnitude as bits: ordered like the numbers, and infinity and NaN above them all
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
        top = max(top, (uint32_t)__shfl_xor((int)top, 1));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2));
        // 127 * 2^k = 1.984375 * 2^(k + 6): the biased exponent less 6, one more if the mantissa is above 0x7E0000
        const int f = (int)(top >> 23), up = (top & 0x7FFFFFu) > 0x7E0000u;
        const bool lost = f == 255;
        const int e = max(1, f - 6 + up);
        const float back = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e)
        if (p.n > 0) {
            i8x8 q;
#pragma unroll
            for (int k = 0; k < 8; k++) q[k] = lost ? (int8_t)1 : (int8_t)(int)rintf(v[k] * back);
            int8_t* to = a.q + p.row * a.q_stride + p.col;
            if (p.n == 8) {
                *(i8x8*)to = q;
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (k < p.n) to[k] = q[k];
            }
            if ((p.col & 31) == 0) a.exps[p.row * a.exps_stride + (p.col >> 5)] = lost ? 255 : (uint8_t)e;
            if (a.y) {
                act_values(v, a.act);
                store_n((T*)a.y + p.row * a.y_stride + p.col, p.n, v);
            }
        }
    }
}

// y = act(kept), or with BACK y = x act'(kept).
template <class T, bool BACK>
__global__ __launch_bounds__(BLOCK) void k_ckpt_read(wc_ckpt_args a, int64_t per_row) {
    const int64_t total = a.rows * per_row;
    for (int64_t i = int64_t(blockIdx.x) * BLOCK + threadIdx.x; i < total; i += int64_t(gridDim.x) * BLOCK) {
        const Place p = place_of(i, per_row, a.width);
        if (p.n <= 0) continue;
        const uint32_t e = a.exps[p.row * a.exps_stride + (p.col >> 5)];
        const float step = step_of(e);
        const int8_t* from = a.q + p.row * a.q_stride + p.col;
        i8x8 q = {};
        if (p.n == 8) {
            q = *(const i8x8*)from;
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < p.n) q[k] = from[k];
        }
        float v[8], g[8];
        if (BACK) load_n((const T*)a.x + p.row * a.x_stride + p.col, p.n, 0.f, g);
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (float)q[k] * step;
        if (may_pass<T>(e)) {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = held<T>(v[k]);
        }
        if (BACK) {
            act_slopes(v, a.act);
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] *= g[k];
        } else {
            act_values(v, a.act);
        }
        store_n((T*)a.y + p.row * a.y_stride + p.col, p.n, v);
    }
}

int64_t chunks_of(int64_t width) { return (width + 31) / 32 * 4; }

dim3 grid_of(const wc_ckpt_args& a, int cus) {
    const int64_t want = (a.rows * chunks_of(a.width) + BLOCK - 1) / BLOCK;
    return dim3((uint32_t)std::max<int64_t>(1, std::min<int64_t>(want, int64_t(cus) * 64)));
}

}  // namespace

void launch_ckpt_write(const wc_ckpt_args& a, int cus, hipStream_t s) {
    if (!a.rows) return;
    const dim3 g = grid_of(a, cus);
    if (a.dtype == WC_DTYPE_F32) k_ckpt_write<float><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
    else if (a.dtype == WC_DTYPE_F16) k_ckpt_write<f16><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
    else k_ckpt_write<bf16><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
}

void launch_ckpt_read(const wc_ckpt_args& a, int cus, hipStream_t s) {
    if (!a.rows) return;
    const dim3 g = grid_of(a, cus);
    if (a.dtype == WC_DTYPE_F32) k_ckpt_read<float, false><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
    else if (a.dtype == WC_DTYPE_F16) k_ckpt_read<f16, false><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
    else k_ckpt_read<bf16, false><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
}

void launch_ckpt_act_back(const wc_ckpt_args& a, int cus, hipStream_t s) {
    if (!a.rows) return;
    const dim3 g = grid_of(a, cus);
    if (a.dtype == WC_DTYPE_F32) k_ckpt_read<float, true><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
    else if (a.dtype == WC_DTYPE_F16) k_ckpt_read<f16, true><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
    else k_ckpt_read<bf16, true><<<g, BLOCK, 0, s>>>(a, chunks_of(a.width));
}

}  // namespace learn
}  // namespace wc
