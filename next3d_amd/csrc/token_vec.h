// Element types and row vectors of the token operators (layer_norm.hip, rotary.hip): float32, float16 and bfloat16 in memory, float32 in registers.
#pragma once
#include "common.h"

// N consecutive elements of T, aligned like ONE element: rows of odd length and strided views start anywhere, and gfx950 loads and stores up to
// 16 bytes at any element address in one instruction.
template <typename T, int N> struct TokenVec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T> struct TokenVec<T, 1> {
    typedef T type;
};

template <typename T, int N>
__device__ __forceinline__ void token_load(const T* __restrict__ p, float (&f)[N]) {
    if constexpr (N == 1) {
        f[0] = (float)p[0];
    } else {
        const typename TokenVec<T, N>::type v = *reinterpret_cast<const typename TokenVec<T, N>::type*>(p);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = (float)v[e];
    }
}

// (one rounding to nearest even where T has 16 bits)
template <typename T, int N>
__device__ __forceinline__ void token_store(T* __restrict__ p, const float (&f)[N]) {
    if constexpr (N == 1) {
        p[0] = (T)f[0];
    } else {
        typename TokenVec<T, N>::type v;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (T)f[e];
        *reinterpret_cast<typename TokenVec<T, N>::type*>(p) = v;
    }
}

// Calls f(T*) with a null pointer of the element type of an N3D_* dtype; false for another dtype.
template <typename F>
static inline bool token_dispatch(int dtype, F&& f) {
    switch (dtype) {
        case N3D_F32: f((float*)nullptr); return true;
        case N3D_F16: f((_Float16*)nullptr); return true;
        case N3D_BF16: f((__bf16*)nullptr); return true;
        default: return false;
    }
}
