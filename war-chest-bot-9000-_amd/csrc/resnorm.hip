// The residual update between two norms, forward and backward (include/wc_learn.h).
//
// Memory bounds both: the forward reads two matrices and writes two, the
// backward reads four and writes two (a gate with a row each: one more read,
// and one more written). Each is read once: a row's values stay in registers,
// eight to a thread, from the load through both norms to the store. A
// workgroup takes row after row with the parameters in registers and the next
// row's loads in flight, and in the backward with the columns' sums of all its
// rows; a small kernel adds the workgroups' sums in order.
//
// On one MI355X (a large copy: 5.09 TB/s): 16,384 x 4,096 bf16 with a gate
// vector, forward 94 us (5.7 TB/s), backward 153 us and 5 for the column sums
// (5.1 TB/s); one workgroup a row and parameters read for each took 171 and 406.
// 4,099 x 1,153 f16 with a gate a row, LayerNorm: 18 and 28 us (2.6 TB/s): three
// to eight rows a workgroup, with four dependent sums each in the forward and
// two in the backward;
// rows at odd addresses cost nothing (1,152 and 1,153 columns take the same).
#include <algorithm>

#include "learn.h"
#include "learn_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {
namespace {

// Eight elements from p as they are; NARROW: the first n, and zeros.
template <class T, bool NARROW>
__device__ __forceinline__ typename Vec8<T>::type raw8(const T* p, int n) {
    typename Vec8<T>::type v = {};
    if (!NARROW) return *(const typename Vec8<T>::type*)p;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) v[i] = p[i];
    return v;
}

template <class T, bool NARROW>
__device__ __forceinline__ void put8(T* p, int n, const float (&v)[8]) {
    store_n(p, NARROW ? n : 8, v);
}

// Eight values of a parameter vector from column c; `fill` where there is none.
template <bool NARROW>
__device__ __forceinline__ void load_param(const void* p, int dtype, int64_t c, int n, float fill, float (&v)[8]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = fill;
    } else if (dtype == WC_DTYPE_F32) {
        const auto r = raw8<float, NARROW>((const float*)p + c, n);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = r[i];
    } else if (dtype == WC_DTYPE_F16) {
        const auto r = raw8<f16, NARROW>((const f16*)p + c, n);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)r[i];
    } else {
        const auto r = raw8<bf16, NARROW>((const bf16*)p + c, n);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)r[i];
    }
}

constexpr int MOST_WAVES = 16;

// Sums over the threads that hold a row, the same bits in each of them: over G
// lanes of a wavefront by a butterfly, or with G 0 over the workgroup: then
// the wavefronts' sums, in order, through LDS. Two slots alternate, so one
// barrier per sum is enough: a wavefront writes a slot again only after a
// barrier that every reader of its last use has passed.
template <int G>
struct RowSum {
    float2* lds;  // 2 x MOST_WAVES
    int waves, slot = 0;

    __device__ __forceinline__ float2 operator()(float a, float b) {
#pragma unroll
        for (int mask = (G ? G : 64) / 2; mask; mask >>= 1) {
            a += __shfl_xor(a, mask);
            b += __shfl_xor(b, mask);
        }
        if constexpr (G == 0) {
            float2* at = lds + slot * MOST_WAVES;
            if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = make_float2(a, b);
            __syncthreads();
            a = b = 0.f;
            for (int w = 0; w < waves; w++) {
                const float2 o = at[w];
                a += o.x;
                b += o.y;
            }
            slot ^= 1;
        }
        return make_float2(a, b);
    }
};

// Eight gate values through their function, chosen once for all.
__device__ __forceinline__ void gates(float (&w)[8], int act) {
    if (act == WC_GATE_SIGMOID) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = __builtin_amdgcn_rcpf(1.f + fast_exp(-w[i]));
    } else if (act == WC_GATE_TANH) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = tanhf(w[i]);
    }
}

// The function's slope from its value.
__device__ __forceinline__ float gate_slope(float w, int act) {
    return act == WC_GATE_SIGMOID ? w * (1.f - w) : act == WC_GATE_TANH ? 1.f - w * w : 1.f;
}

// How a workgroup's threads hold rows: G lanes a row, or with G 0 all of them,
// a chunk of eight columns each (NV: and one every `step` threads on). The last
// chunk of a width that eight does not divide is moved back to end with the
// row: its first columns are then the chunk before's too. Both threads compute
// and write the same values there; sums over the row leave out the second's
// (`skip` of them, or all eight of a thread past the end). So every load is a
// whole one. NARROW, of rows of less than eight: single elements.
template <int G, int NV, bool NARROW>
struct Layout {
    int lane, group, per;  // of the row; which row; rows at once
    int col[NV], skip[NV], n;

    __device__ __forceinline__ explicit Layout(int width) {
        const int step = G ? G : blockDim.x;
        lane = G ? threadIdx.x % (G ? G : 1) : threadIdx.x;
        group = G ? threadIdx.x / (G ? G : 1) : 0;
        per = G ? blockDim.x / (G ? G : 1) : 1;
        n = width;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            const int c = 8 * (lane + k * step);
            col[k] = NARROW ? 0 : min(c, width - 8);
            skip[k] = NARROW ? (lane ? 8 : 0) : min(c - col[k], 8);
        }
    }
    __device__ __forceinline__ bool counts(int k, int i) const { return i >= skip[k] && (!NARROW || i < n); }
    __device__ __forceinline__ bool holds(int k) const { return skip[k] < 8; }
};

// Mean (0 for RMS) and 1 / sqrt(variance + eps) of the row's values, from two
// passes over registers.
template <int G, int NV, bool LAYER, class L>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][8], const L& at, float width, float eps,
                                            RowSum<G>& sum) {
    float mean = 0.f, q = 0.f;
    if (LAYER) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++)
#pragma unroll
            for (int i = 0; i < 8; i++) s += at.counts(k, i) ? v[k][i] : 0.f;
        mean = sum(s, 0.f).x / width;
    }
#pragma unroll
    for (int k = 0; k < NV; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float d = at.counts(k, i) ? v[k][i] - mean : 0.f;
            q += d * d;
        }
    return make_float2(mean, 1.f / sqrtf(sum(q, 0.f).x / width + eps));
}

// The update of a column is gain * norm(block) + bias, with the scale, the gate
// vector and the parameters folded together where the gate is not the row's own.
template <bool NARROW, class A>
__device__ __forceinline__ void fold(const A& a, bool token, int col, int n, float (&gain)[8], float (&bias)[8]) {
    float g[8];
    load_param<NARROW>(a.post_gain, a.param_dtype, col, n, 1.f, gain);
    load_param<NARROW>(a.post_bias, a.param_dtype, col, n, 0.f, bias);
    load_param<NARROW>(token ? nullptr : a.gate, a.param_dtype, col, n, 1.f, g);
    if (a.gate && !token) gates(g, a.gate_act);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        gain[i] *= a.scale * g[i];
        bias[i] *= a.scale * g[i];
    }
}

template <class T, int G, int NV, bool LAYER, bool TOKEN, bool NARROW>
__global__ __launch_bounds__(G ? 256 : 1024) void k_norm(wc_norm_args a) {
    typedef typename Vec8<T>::type Raw;
    __shared__ float2 lds[2 * MOST_WAVES];
    const Layout<G, NV, NARROW> at((int)a.width);
    RowSum<G> sum{lds, (int)blockDim.x / 64};
    const float width = (float)(int)a.width;
    float g1[NV][8], b1[NV][8], g2[NV][8], b2[NV][8];
#pragma unroll
    for (int k = 0; k < NV; k++) {
        fold<NARROW>(a, TOKEN, at.col[k], at.n, g1[k], b1[k]);
        load_param<NARROW>(a.pre_gain, a.param_dtype, at.col[k], at.n, 1.f, g2[k]);
        load_param<NARROW>(a.pre_bias, a.param_dtype, at.col[k], at.n, 0.f, b2[k]);
    }
    const int64_t stride = int64_t(gridDim.x) * at.per;
    Raw ru[NV], rx[NV], rg[TOKEN ? NV : 1];
    auto load = [&](int64_t row) {
        const int64_t r = min(row, a.rows - 1);  // rows past the end go along: the sums are taken by whole wavefronts
#pragma unroll
        for (int k = 0; k < NV; k++) {
            ru[k] = raw8<T, NARROW>((const T*)a.block + r * a.block_stride + at.col[k], at.n);
            rx[k] = raw8<T, NARROW>((const T*)a.stream + r * a.stream_stride + at.col[k], at.n);
            if (TOKEN) rg[k] = raw8<T, NARROW>((const T*)a.gate + r * a.gate_stride + at.col[k], at.n);
        }
    };
    int64_t r = int64_t(blockIdx.x) * at.per + at.group;
    load(r);
    for (int64_t r0 = int64_t(blockIdx.x) * at.per; r0 < a.rows; r0 += stride, r += stride) {
        float u[NV][8], x[NV][8];
        Raw g[TOKEN ? NV : 1];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            // a chunk moved back may be read here and written, as the next thread's, by another wavefront
            if (G == 0) settle(rx[k]);
#pragma unroll
            for (int i = 0; i < 8; i++) u[k][i] = (float)ru[k][i], x[k][i] = (float)rx[k][i];
            if (TOKEN) g[k] = rg[k];
        }
        if (r0 + stride < a.rows) load(r + stride);
        const bool here = r < a.rows;
        const float2 s1 = row_stats<G, NV, LAYER>(u, at, width, a.eps, sum);
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = TOKEN ? (float)g[TOKEN ? k : 0][i] : 1.f;
            if (TOKEN) gates(w, a.gate_act);
#pragma unroll
            for (int i = 0; i < 8; i++) x[k][i] += w[i] * ((u[k][i] - s1.x) * s1.y * g1[k][i] + b1[k][i]);
            if (here && at.holds(k)) put8<T, NARROW>((T*)a.new_stream + r * a.new_stream_stride + at.col[k], at.n, x[k]);
        }
        const float2 s2 = row_stats<G, NV, LAYER>(x, at, width, a.eps, sum);
#pragma unroll
        for (int k = 0; k < NV; k++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[k][i] = (x[k][i] - s2.x) * s2.y * g2[k][i] + b2[k][i];
            if (here && at.holds(k)) put8<T, NARROW>((T*)a.out + r * a.out_stride + at.col[k], at.n, x[k]);
        }
        if (a.stats && here && at.lane == 0) ((float4*)a.stats)[r] = make_float4(s1.x, s1.y, s2.x, s2.y);
    }
}

// The parameters' gradients: which of them are wanted, and where the column
// sums go. The workgroups' sums lie one wanted parameter after the other.
constexpr int SUMS = 5;  // post gain, post bias, gate vector, pre gain, pre bias
struct ColumnSums {
    float* out[SUMS];
    int at[SUMS];  // the parameter's place among the wanted, or -1
    int wanted;
};

// With v what arrives at stream' in all and w the update's factor of a column,
// the parameters' gradients are of four sums over the rows: of w v norm(block)
// and w v, of d_out norm(stream') and d_out. A factor that is the column's own
// stays out of the sums: the gate vector's gradient is of the same two.
// MOST: threads of the widest workgroup; 512 leave a thread the registers that
// it needs, 1,024 do not: 2,048 x 8,192 bf16 with a gate a row 115 us (parameters
// in registers too: 172), floor 53; past 8,192 columns 1,024 x 16,384 255 us, floor 40.
template <class T, int G, int NV, bool LAYER, bool TOKEN, bool NARROW, int MOST>
__global__ __launch_bounds__(G ? 256 : MOST, MOST == 1024 ? 4 : TOKEN ? 2 : 3) void k_norm_back(wc_norm_back_args a, ColumnSums sums, float* part) {
    typedef typename Vec8<T>::type Raw;
    __shared__ float2 lds[2 * MOST_WAVES];
    __shared__ float cols[G ? G * NV * 8 : 1];
    const Layout<G, NV, NARROW> at((int)a.width);
    RowSum<G> sum{lds, (int)blockDim.x / 64};
    const float width = (float)(int)a.width;
    // Workgroups of 1,024 have 128 registers a thread: there the parameters wait
    // in LDS, each thread's own, and are read as a row needs them.
    constexpr bool STAGED = MOST == 1024 && NV == 1;
    __shared__ float4 stage[STAGED ? 6 * MOST : 1];
    float g1[NV][8], b1[NV][8], g2[NV][8], acc[4][NV][8] = {};
#pragma unroll
    for (int k = 0; k < NV; k++) {
        fold<NARROW>(a, TOKEN, at.col[k], at.n, g1[k], b1[k]);
        load_param<NARROW>(a.pre_gain, a.param_dtype, at.col[k], at.n, 1.f, g2[k]);
    }
    auto staged = [&](int q, float (&v)[8], bool put) {
        float4* to = stage + 2 * q * MOST + threadIdx.x;
        if (put) {
            to[0] = make_float4(v[0], v[1], v[2], v[3]);
            to[MOST] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            asm volatile("" ::: "memory");  // read here, not held from the row before
            const float4 lo = to[0], hi = to[MOST];
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
        }
    };
    if constexpr (STAGED) staged(0, g1[0], true), staged(1, b1[0], true), staged(2, g2[0], true);
    const int64_t stride = int64_t(gridDim.x) * at.per;
    Raw ru[NV], rx[NV], rh[NV], rd[NV], rg[TOKEN ? NV : 1];
    float4 rs;
    auto load = [&](int64_t row) {
        const int64_t r = min(row, a.rows - 1);
        rs = ((const float4*)a.stats)[r];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            ru[k] = raw8<T, NARROW>((const T*)a.block + r * a.block_stride + at.col[k], at.n);
            rx[k] = raw8<T, NARROW>((const T*)a.stream + r * a.stream_stride + at.col[k], at.n);
            rh[k] = Raw{}, rd[k] = Raw{};
            if (a.d_out) rh[k] = raw8<T, NARROW>((const T*)a.d_out + r * a.d_out_stride + at.col[k], at.n);
            if (a.d_new_stream)
                rd[k] = raw8<T, NARROW>((const T*)a.d_new_stream + r * a.d_new_stream_stride + at.col[k], at.n);
            if (TOKEN) rg[k] = raw8<T, NARROW>((const T*)a.gate + r * a.gate_stride + at.col[k], at.n);
        }
    };
    int64_t r = int64_t(blockIdx.x) * at.per + at.group;
    if (a.rows) load(r);
    for (int64_t r0 = int64_t(blockIdx.x) * at.per; r0 < a.rows; r0 += stride, r += stride) {
        const bool here = r < a.rows;
        const float4 st = rs;
        // the block's norm, and the stream's after the update, as the forward computed them
        float uh[NV][8], xh[NV][8], dx[NV][8], w[NV][8];
        Raw d[NV];
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            d[k] = rd[k];
            if (G == 0) settle(d[k]);  // as in the forward
#pragma unroll
            for (int i = 0; i < 8; i++) w[k][i] = TOKEN ? (float)rg[TOKEN ? k : 0][i] : 1.f;
            if (TOKEN) gates(w[k], a.gate_act);
            if constexpr (STAGED) staged(0, g1[k], false), staged(1, b1[k], false), staged(2, g2[k], false);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                uh[k][i] = ((float)ru[k][i] - st.x) * st.y;
                const float x = (float)rx[k][i] + w[k][i] * (uh[k][i] * g1[k][i] + b1[k][i]);
                xh[k][i] = (x - st.z) * st.w;
                const float dh = here ? (float)rh[k][i] : 0.f;
                acc[2][k][i] += dh * xh[k][i];
                acc[3][k][i] += dh;
                dx[k][i] = dh * g2[k][i];
                const float t = at.counts(k, i) ? dx[k][i] : 0.f;
                s1 += t;
                s2 += t * xh[k][i];
            }
        }
        if (r0 + stride < a.rows) load(r + stride);
        float2 m = sum(s1, s2);
        const float c1 = LAYER ? m.x / width : 0.f, c2 = m.y / width;
        s1 = s2 = 0.f;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float o[8], dg[8];
            if constexpr (STAGED) {
                staged(0, g1[k], false);
                if (TOKEN) staged(1, b1[k], false);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float v = st.w * (dx[k][i] - c1 - xh[k][i] * c2) + (float)d[k][i];
                o[i] = v;
                const float wv = here ? w[k][i] * v : 0.f;
                if (TOKEN) dg[i] = gate_slope(w[k][i], a.gate_act) * v * (uh[k][i] * g1[k][i] + b1[k][i]);
                acc[0][k][i] += wv * uh[k][i];
                acc[1][k][i] += wv;
                dx[k][i] = wv * g1[k][i];
                const float t = at.counts(k, i) ? dx[k][i] : 0.f;
                s1 += t;
                s2 += t * uh[k][i];
            }
            if (here && at.holds(k)) {
                put8<T, NARROW>((T*)a.d_stream + r * a.d_stream_stride + at.col[k], at.n, o);
                if (TOKEN && a.d_gate) put8<T, NARROW>((T*)a.d_gate + r * a.d_gate_stride + at.col[k], at.n, dg);
            }
        }
        m = sum(s1, s2);
        const float e1 = LAYER ? m.x / width : 0.f, e2 = m.y / width;
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = st.y * (dx[k][i] - e1 - uh[k][i] * e2);
            if (here && at.holds(k)) put8<T, NARROW>((T*)a.d_block + r * a.d_block_stride + at.col[k], at.n, o);
        }
    }
    // the parameters' gradients from the four sums, and the workgroup's: its row groups in order
#pragma unroll
    for (int q = 0; q < SUMS; q++) {
        if (sums.at[q] < 0) continue;
        float* to = part + (size_t(blockIdx.x) * sums.wanted + sums.at[q]) * a.width;
        float v[NV][8];
#pragma unroll
        for (int k = 0; k < NV; k++) {
            float gain[8], bias[8], gate[8];
            if (q < 3) {
                load_param<NARROW>(a.post_gain, a.param_dtype, at.col[k], at.n, 1.f, gain);
                load_param<NARROW>(a.post_bias, a.param_dtype, at.col[k], at.n, 0.f, bias);
                load_param<NARROW>(TOKEN ? nullptr : a.gate, a.param_dtype, at.col[k], at.n, 1.f, gate);
                if (!TOKEN && a.gate) gates(gate, a.gate_act);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (q < 2) v[k][i] = a.scale * gate[i] * acc[q][k][i];
                else if (q == 2)
                    v[k][i] = a.scale * gate_slope(gate[i], a.gate_act) * (gain[i] * acc[0][k][i] + bias[i] * acc[1][k][i]);
                else v[k][i] = acc[q - 1][k][i];
            }
        }
        if constexpr (G == 0) {
#pragma unroll
            for (int k = 0; k < NV; k++)
                if (at.holds(k)) put8<float, NARROW>(to + at.col[k], at.n, v[k]);
        } else {
            for (int g = 0; g < at.per; g++) {
                __syncthreads();
                if (at.group == g) {
#pragma unroll
                    for (int k = 0; k < NV; k++)
#pragma unroll
                        for (int i = 0; i < 8; i++)  // each column by one thread: the last chunk lies over the one before
                            if (at.counts(k, i)) cols[at.col[k] + i] = (g ? cols[at.col[k] + i] : 0.f) + v[k][i];
                }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < a.width; c += blockDim.x) to[c] = cols[c];
        }
    }
}

// Adds the workgroups' column sums: N columns a thread (the last ones moved back
// to end with the row), 8 threads side by side, every 32nd workgroup to each of
// 32 rows of threads, whose sums are added in order.
template <int N>
__global__ __launch_bounds__(256) void k_norm_cols(const float* part, int blocks, int64_t width, ColumnSums sums) {
    typedef float Some __attribute__((ext_vector_type(N), aligned(4)));
    __shared__ Some lds[32][8];
    const int x = threadIdx.x & 7, y = threadIdx.x >> 3;
    int q = 0;
    while (sums.at[q] != (int)blockIdx.y) q++;
    const int64_t c0 = (int64_t(blockIdx.x) * 8 + x) * N, c = min(c0, width - N), pitch = width * sums.wanted;
    const float* from = part + blockIdx.y * width + c;
    Some s = {};
    if (c0 < width) {
        int b = y;
        for (; b + 96 < blocks; b += 128) {
            Some v[4];
#pragma unroll
            for (int u = 0; u < 4; u++) v[u] = *(const Some*)(from + (b + 32 * u) * pitch);
            s += (v[0] + v[1]) + (v[2] + v[3]);
        }
        for (; b < blocks; b += 32) s += *(const Some*)(from + b * pitch);
    }
    lds[y][x] = s;
    __syncthreads();
    if (y || c0 >= width) return;
    for (int k = 1; k < 32; k++) s += lds[k][x];
    *(Some*)(sums.out[q] + c) = s;
}

// ------------------------------------------------------------------ launches

// Lanes per row (0: the workgroup) and threads of the workgroup: as many as the
// row has chunks of eight, by powers of two inside a wavefront and by whole
// wavefronts beyond; past 8,192 columns two chunks a thread. Forward over
// 4,099 x 1,153 f16: 18 us with 192 threads, 21 with the next power of two,
// 256; the backward takes 27 with either.
struct Threads {
    int g, block, nv;
};
Threads threads_of(int64_t width) {
    const int64_t chunks = (width + 7) / 8;
    if (chunks <= 64) {
        int g = 8;
        while (g < chunks) g *= 2;
        return {g, 256, 1};
    }
    if (chunks <= 1024) return {0, (int)((chunks + 63) / 64 * 64), 1};
    return {0, 1024, 2};
}

// Workgroups: as many as the device holds at once (its registers hold `waves`
// wavefronts a CU), and in the backward, whose column sums are written and read
// again for each, no more than leave each `turns` rows while every CU has one.
int blocks_of(int64_t rows, const Threads& t, int waves, int64_t turns, int cus) {
    const int64_t per = t.g ? t.block / t.g : 1, want = (rows + per - 1) / per;
    const int64_t full = int64_t(cus) * std::max(1, waves * 64 / t.block);
    return (int)std::max<int64_t>(1, std::min({want, full, std::max<int64_t>(cus, want / turns)}));
}

// Measured over 8 to 64 (forward) and 4 to 24 wavefronts a CU: 16,384 x 1,153
// with a gate a row 48 us at 16 against 56 at 12 and 60 at 20, its backward 86
// us at 8 against 88 at 12 and 96 at 16; 16,384 x 4,096 backward 123 us up to 12,
// 131 at 16. Rows for each workgroup: 4,099 x 1,153 31 us at 8, 42 at 16 (one
// workgroup a CU); 16,384 rows do not care.
constexpr int FORWARD_WAVES = 16, BACKWARD_WAVES = 12, BACKWARD_TOKEN_WAVES = 8;
constexpr int64_t FORWARD_TURNS = 1, BACKWARD_TURNS = 8;

template <class T, int G, int NV, bool NARROW = false>
void norm_at(const wc_norm_args& a, const Threads& t, int cus, hipStream_t s) {
    const dim3 grid(blocks_of(a.rows, t, FORWARD_WAVES, FORWARD_TURNS, cus));
    const bool layer = a.norm == WC_NORM_LAYER, token = a.gate && a.gate_stride;
    if (layer && token) k_norm<T, G, NV, true, true, NARROW><<<grid, t.block, 0, s>>>(a);
    else if (layer) k_norm<T, G, NV, true, false, NARROW><<<grid, t.block, 0, s>>>(a);
    else if (token) k_norm<T, G, NV, false, true, NARROW><<<grid, t.block, 0, s>>>(a);
    else k_norm<T, G, NV, false, false, NARROW><<<grid, t.block, 0, s>>>(a);
}

template <class T>
void norm(const wc_norm_args& a, int cus, hipStream_t s) {
    const Threads t = threads_of(a.width);
    if (a.width < 8) norm_at<T, 8, 1, true>(a, t, cus, s);
    else if (t.g == 8) norm_at<T, 8, 1>(a, t, cus, s);
    else if (t.g == 16) norm_at<T, 16, 1>(a, t, cus, s);
    else if (t.g == 32) norm_at<T, 32, 1>(a, t, cus, s);
    else if (t.g == 64) norm_at<T, 64, 1>(a, t, cus, s);
    else if (t.nv == 1) norm_at<T, 0, 1>(a, t, cus, s);
    else norm_at<T, 0, 2>(a, t, cus, s);
}

template <class T, int G, int NV, int MOST, bool NARROW = false>
void back_at(const wc_norm_back_args& a, const Threads& t, int blocks, const ColumnSums& c, hipStream_t s) {
    const bool layer = a.norm == WC_NORM_LAYER, token = a.gate && a.gate_stride;
    float* w = (float*)a.workspace;
    if (layer && token) k_norm_back<T, G, NV, true, true, NARROW, MOST><<<dim3(blocks), t.block, 0, s>>>(a, c, w);
    else if (layer) k_norm_back<T, G, NV, true, false, NARROW, MOST><<<dim3(blocks), t.block, 0, s>>>(a, c, w);
    else if (token) k_norm_back<T, G, NV, false, true, NARROW, MOST><<<dim3(blocks), t.block, 0, s>>>(a, c, w);
    else k_norm_back<T, G, NV, false, false, NARROW, MOST><<<dim3(blocks), t.block, 0, s>>>(a, c, w);
}

int back_blocks(const wc_norm_back_args& a, const Threads& t, int cus) {
    const int waves = a.gate && a.gate_stride ? BACKWARD_TOKEN_WAVES : BACKWARD_WAVES;
    return blocks_of(a.rows, t, waves, BACKWARD_TURNS, cus);
}

template <class T>
void norm_back(const wc_norm_back_args& a, int cus, hipStream_t s) {
    const Threads t = threads_of(a.width);
    const int blocks = back_blocks(a, t, cus);
    ColumnSums c = {{a.d_post_gain, a.d_post_bias, a.gate && !a.gate_stride ? (float*)a.d_gate : nullptr, a.d_pre_gain,
                     a.d_pre_bias}, {}, 0};
    for (int q = 0; q < SUMS; q++) c.at[q] = c.out[q] ? c.wanted++ : -1;
    if (a.width < 8) back_at<T, 8, 1, 256, true>(a, t, blocks, c, s);
    else if (t.g == 8) back_at<T, 8, 1, 256>(a, t, blocks, c, s);
    else if (t.g == 16) back_at<T, 16, 1, 256>(a, t, blocks, c, s);
    else if (t.g == 32) back_at<T, 32, 1, 256>(a, t, blocks, c, s);
    else if (t.g == 64) back_at<T, 64, 1, 256>(a, t, blocks, c, s);
    else if (t.block <= 512) back_at<T, 0, 1, 512>(a, t, blocks, c, s);
    else if (t.nv == 1) back_at<T, 0, 1, 1024>(a, t, blocks, c, s);
    else back_at<T, 0, 2, 1024>(a, t, blocks, c, s);
    if (!c.wanted) return;
    const int64_t n = a.width >= 4 ? 32 : 8;
    const dim3 grid((uint32_t)((a.width + n - 1) / n), c.wanted);
    if (n == 32) k_norm_cols<4><<<grid, 256, 0, s>>>((const float*)a.workspace, blocks, a.width, c);
    else k_norm_cols<1><<<grid, 256, 0, s>>>((const float*)a.workspace, blocks, a.width, c);
}

}  // namespace

size_t norm_back_scratch(const wc_norm_back_args& a, int cus) {
    // with or without a gate of the rows' own: the binding asks by shape
    const size_t blocks = blocks_of(a.rows, threads_of(a.width), BACKWARD_WAVES, BACKWARD_TURNS, cus);
    return pad256(blocks * SUMS * size_t(a.width) * 4);
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
