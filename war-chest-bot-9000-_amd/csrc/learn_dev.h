// Device helpers of the training operators: element types, eight-element
// loads and stores at any element alignment, and fixed-order reductions.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace wc {
namespace learn {

typedef _Float16 f16;
typedef __bf16 bf16;

// Consecutive elements. The type asks for the element's alignment only:
// the hardware takes wide accesses at any, and splits one that crosses a line.
template <class T, int N>
struct VecN {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <class T>
using Vec8 = VecN<T, 8>;

template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ p, float (&v)[8]) {
    const typename Vec8<T>::type x = *(const typename Vec8<T>::type*)p;
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (float)x[i];
}

// The first n (0 .. 8) of eight elements, `fill` in the place of the others.
template <class T>
__device__ __forceinline__ void load_n(const T* __restrict__ p, int n, float fill, float (&v)[8]) {
    if (n >= 8) {
        load8(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < n ? (float)p[i] : fill;
}

template <class T>
__device__ __forceinline__ void store_n(T* __restrict__ p, int n, const float (&v)[8]) {
    if (n >= 8) {
        typename Vec8<T>::type x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (T)v[i];
        *(typename Vec8<T>::type*)p = x;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < n) p[i] = (T)v[i];
}

// The first n (0 .. N) of N elements, zeros in the place of the others.
template <int N, class T>
__device__ __forceinline__ typename VecN<T, N>::type load_some(const T* p, int n) {
    if (n >= N) return *(const typename VecN<T, N>::type*)p;
    typename VecN<T, N>::type v = {};
#pragma unroll
    for (int i = 0; i < N - 1; i++)
        if (i < n) v[i] = p[i];
    return v;
}

// 2^x by the hardware (1 ulp; a result under 2^-126 is 0).
__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }

// e^x for the sigmoids: for the arguments that matter there x log2(e) is off by
// less than a millionth.
__device__ __forceinline__ float fast_exp(float x) { return power(x * 1.4426950408889634f); }

// Waits for a load: its value is asked for here. Used before a barrier after
// which another wavefront may write where it came from (outputs that may be
// their inputs).
__device__ __forceinline__ void settle(float& v) { asm volatile("" : "+v"(v)); }
template <class V>
__device__ __forceinline__ void settle(V& v) {
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(V) / 4)));
    Words w = __builtin_bit_cast(Words, v);
    if constexpr (sizeof(V) == 32) {  // as two operands of four registers
        typedef uint32_t Four __attribute__((ext_vector_type(4)));
        Four lo = __builtin_shufflevector(w, w, 0, 1, 2, 3), hi = __builtin_shufflevector(w, w, 4, 5, 6, 7);
        asm volatile("" : "+v"(lo), "+v"(hi));
        w = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
        asm volatile("" : "+v"(w));
    }
    v = __builtin_bit_cast(V, w);
}

__device__ __forceinline__ int64_t index_at(const void* p, int bits, int64_t i) {
    return bits == 64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

}  // namespace learn
}  // namespace wc
