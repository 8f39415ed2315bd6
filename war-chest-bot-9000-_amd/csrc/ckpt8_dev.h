// The 8-bit checkpoint's values and the activation functions read from them.
#pragma once

#include "learn.h"
#include "learn_dev.h"

#pragma clang fp contract(fast)

namespace wc {
namespace learn {

// The power that an exponent byte stands for; 255, a group with an infinity or
// a NaN, gives NaN, which every product with it keeps.
__device__ __forceinline__ float step_of(uint32_t e) {
    return e == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(e << 23);
}

// The magnitude that values read into a type are held at: only a group near
// the end of the type's range can round beyond it (float32 and bf16: 2^128
// from 64 * 2^122; f16: 65536 from 64 * 2^10), told by its exponent byte. The
// comparisons keep a NaN.
template <class T>
__device__ __forceinline__ float held(float v) {
    constexpr float most = __is_same(T, f16) ? 65504.f : 3.4028234663852886e38f;
    return v > most ? most : v < -most ? -most : v;
}
template <class T>
__device__ __forceinline__ bool may_pass(uint32_t e) {
    return e >= (__is_same(T, f16) ? 137u : 249u);
}

// 1 / (1 + e^-x); the reciprocal is within an ulp.
__device__ __forceinline__ float sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-x)); }

constexpr float GELU_C = 0.7978845608028654f, GELU_K = 0.044715f;

// x/2 (1 + tanh u) = x sigma(2u), u = c (x + k x^3).
__device__ __forceinline__ float act_value(float x, int act) {
    if (act == WC_ACT_RELU) return x > 0.f ? x : x != x ? x : 0.f;
    if (act == WC_ACT_SILU) return x * sigmoid_fast(x);
    if (act == WC_ACT_GELU) return x * sigmoid_fast(2.f * GELU_C * (x + GELU_K * x * x * x));
    return x;
}

// The slopes: sigma (1 + x (1 - sigma)); s + 2 x s (1 - s) du/dx. Where the
// sigmoid is 0 or 1 its slope's term is 0 (x^2 may have overflowed there).
__device__ __forceinline__ float act_slope(float x, int act) {
    if (act == WC_ACT_RELU) return x > 0.f ? 1.f : x != x ? x : 0.f;
    if (act == WC_ACT_SILU) {
        const float s = sigmoid_fast(x);
        return s * (1.f + x * (1.f - s));
    }
    if (act == WC_ACT_GELU) {
        const float xx = x * x, s = sigmoid_fast(2.f * GELU_C * (x + GELU_K * xx * x)), t = s * (1.f - s);
        return t == 0.f ? s : s + 2.f * x * t * GELU_C * (1.f + 3.f * GELU_K * xx);
    }
    return x != x ? x : 1.f;
}

// Eight at a time: the choice once, not for each.
__device__ __forceinline__ void act_values(float (&v)[8], int act) {
    if (act == WC_ACT_NONE) return;
    if (act == WC_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_value(v[i], WC_ACT_RELU);
    } else if (act == WC_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_value(v[i], WC_ACT_GELU);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_value(v[i], WC_ACT_SILU);
    }
}
__device__ __forceinline__ void act_slopes(float (&v)[8], int act) {
    if (act == WC_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_slope(v[i], WC_ACT_NONE);
    } else if (act == WC_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_slope(v[i], WC_ACT_RELU);
    } else if (act == WC_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_slope(v[i], WC_ACT_GELU);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = act_slope(v[i], WC_ACT_SILU);
    }
}

}  // namespace learn
}  // namespace wc
