// float32 products straight from memory, for layers so small that launches are what they cost (linear_dev.h):
// C[m x n] = sum over k of A[i][k] B[k][j] by the matrix cores' float32 instruction, without copies in parts.
//
// One launch for a product, and one for both gradients with the bias's, where the way in parts has three and five; what
// bounds it then is the loads' latency (512 x 512 x 512 8.1 us, 33 TFLOP/s), and on all CUs that neighbouring
// fragments load the same rows again: 1,024 x 1,024 x 1,024 takes 37 us, as long as in parts.
//
// A workgroup of eight wavefronts has a fragment of 32 x 32, each wavefront every eighth eight of k: a lane loads four of k at a
// time, of one row of A and one column of B, and four instructions take one of them each. The eighths are added in LDS
// in an order that does not change.
#pragma once

#include "ckpt8_dev.h"
#include "learn.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

constexpr int DIRECT_BLOCK = 512, DIRECT_WAVES = DIRECT_BLOCK / 64, DIRECT_PITCH = 36;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32acc __attribute__((ext_vector_type(16)));

// One operand: `outer` rows of A or columns of B. With `pre`, what is read is times the activation's slope there.
struct DirectSide {
    const float* p;
    int64_t stride, outer;
    const float* pre;
    int64_t pre_stride;
};

struct Direct {
    DirectSide a, b;
    int64_t k, run, tiles_n;  // run: of k, what a workgroup sums
    int act, runs;
    unsigned blocks;          // of all runs
    float* part;              // runs > 1: runs x m x n partial products
    float* sums;              // of the slopes' side over each run, one for each of its rows or columns; may be null
};

// Four of k from `at` on, n of them there.
template <bool INNER>
__device__ __forceinline__ f32x4 direct_four(const float* p, int64_t stride, int64_t o, int64_t at, int n) {
    if (INNER) return load_some<4>(p + o * stride + at, n);
    f32x4 v = {};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n) v[i] = p[(at + i) * stride + o];
    return v;
}
template <bool INNER>
__device__ __forceinline__ f32x4 direct_side(const DirectSide& s, int act, int64_t o, int64_t at, int n) {
    f32x4 v = direct_four<INNER>(s.p, s.stride, o, at, n);
    if (!s.pre) return v;
    const f32x4 z = direct_four<INNER>(s.pre, s.pre_stride, o, at, n);
    float d[8] = {z[0], z[1], z[2], z[3]};
    act_slopes(d, act);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = i < n ? v[i] * d[i] : 0.f;
    return v;
}

typedef float DirectLds[DIRECT_WAVES][32][DIRECT_PITCH];

// SUMS: whose sums over k are wanted, 0 none, 1 A's, 2 B's.
template <bool AI, bool BI, int SUMS, class Epilogue>
__device__ __forceinline__ void direct_product(const Direct& p, const Epilogue& epilogue, DirectLds& lds, float (&some)[DIRECT_WAVES][32],
                                               int64_t block) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t tiles = p.blocks / p.runs, run = block / tiles, tile = block - run * tiles;
    const int64_t ti = tile / p.tiles_n, tj = tile - ti * p.tiles_n, i0 = 32 * ti, j0 = 32 * tj;
    const int64_t lo = run * p.run, hi = min(lo + p.run, p.k);
    // past the last row any row will do: its products are not stored
    const int64_t i = min(i0 + (lane & 31), p.a.outer - 1), j = min(j0 + (lane & 31), p.b.outer - 1);
    f32acc c = {};
    f32x4 total = {};
#pragma unroll 4
    for (int64_t first = lo + 8 * wave; first < hi; first += 8 * DIRECT_WAVES) {
        const int64_t at = first + 4 * (lane >> 5);
        const int n = (int)max<int64_t>(0, min<int64_t>(4, hi - at));
        const f32x4 a = direct_side<AI>(p.a, p.act, i, at, n), b = direct_side<BI>(p.b, p.act, j, at, n);
        if (SUMS == 1) total += a;
        if (SUMS == 2) total += b;
#pragma unroll
        for (int u = 0; u < 4; u++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[u], b[u], c, 0, 0, 0);
    }
#pragma unroll
    for (int k = 0; k < 16; k++) lds[wave][8 * (k / 4) + 4 * (lane >> 5) + k % 4][lane & 31] = c[k];
    if (SUMS) {
        float s = (total[0] + total[1]) + (total[2] + total[3]);
        s += __shfl_xor(s, 32);
        if (lane < 32) some[wave][lane] = s;
    }
    __syncthreads();
    if (SUMS && p.sums && (SUMS == 1 ? tj : ti) == 0 && threadIdx.x >= DIRECT_BLOCK - 32) {
        const int t = threadIdx.x & 31;
        const int64_t at = (SUMS == 1 ? i0 : j0) + t;
        float s = 0.f;
        for (int w = 0; w < DIRECT_WAVES; w++) s += some[w][t];
        const int64_t all = SUMS == 1 ? p.a.outer : p.b.outer;
        if (at < all) p.sums[run * all + at] = s;
    }
    if (threadIdx.x >= 128) return;
    const int r = threadIdx.x / 4, col = threadIdx.x % 4 * 8;
    const int have = (int)min<int64_t>(8, p.b.outer - j0 - col);
    if (i0 + r >= p.a.outer || have <= 0) return;
    float v[8] = {};
    typename Epilogue::Raw raw = {};
    if (p.runs == 1) raw = epilogue.raw(0, i0 + r, j0 + col, have);
    for (int w = 0; w < DIRECT_WAVES; w++) {
        const f32x4 lo = *(const f32x4*)&lds[w][r][col], hi = *(const f32x4*)&lds[w][r][col + 4];
#pragma unroll
        for (int u = 0; u < 4; u++) v[u] += lo[u], v[u + 4] += hi[u];
    }
    if (p.runs > 1) store_n(p.part + (run * p.a.outer + i0 + r) * p.b.outer + j0 + col, have, v);
    else epilogue(raw, 0, i0 + r, j0 + col, have, v);
}

template <bool BI, class Epilogue>
__global__ __launch_bounds__(DIRECT_BLOCK) void k_direct(Direct p, Epilogue epilogue) {
    __shared__ __align__(16) DirectLds lds;
    __shared__ float some[DIRECT_WAVES][32];
    direct_product<true, BI, 0>(p, epilogue, lds, some, blockIdx.x);
}

// A layer's gradients: x's, from the gradient at the pre-activations by the weight's rows or columns, and the weight's with
// the bias's, in one launch. Either may have no workgroups.
template <bool IO, class Epilogue>
__global__ __launch_bounds__(DIRECT_BLOCK) void k_direct_back(Direct x, Epilogue ex, Direct w, Epilogue ew) {
    __shared__ __align__(16) DirectLds lds;
    __shared__ float some[DIRECT_WAVES][32];
    if (blockIdx.x < x.blocks) direct_product<true, IO, 0>(x, ex, lds, some, blockIdx.x);
    else direct_product<false, false, IO ? 2 : 1>(w, ew, lds, some, blockIdx.x - x.blocks);
}

}  // namespace
}  // namespace learn
}  // namespace wc
