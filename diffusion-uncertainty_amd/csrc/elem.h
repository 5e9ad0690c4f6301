// Element types of the token operators (rel_attention.hip, sandwich_norm.hip, token_logprobs.hip): fp32, bf16, fp16 in memory, fp32 in
// registers.  A vector access moves 16 bytes: 4 fp32 or 8 sixteen-bit elements.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

template <typename T> struct Elem;
template <> struct Elem<float> { static constexpr int VEC = 4; };
template <> struct Elem<bf16_t> { static constexpr int VEC = 8; };
template <> struct Elem<f16_t> { static constexpr int VEC = 8; };

template <typename T, int N> struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };

// N consecutive elements as floats; N > 1 needs an address aligned to N * sizeof(T)
template <typename T, int N>
__device__ __forceinline__ void ld_elems(const T* p, float* f) {
    if constexpr (N == 1) {
        f[0] = (float)p[0];
    } else {
        const auto v = *(const typename VecOf<T, N>::type*)p;
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = (float)v[j];
    }
}
// ... and back, rounded to nearest once
template <typename T, int N>
__device__ __forceinline__ void st_elems(T* p, const float* f) {
    if constexpr (N == 1) {
        p[0] = (T)f[0];
    } else {
        typename VecOf<T, N>::type v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (T)f[j];
        *(typename VecOf<T, N>::type*)p = v;
    }
}

static inline size_t dua_dtype_size(int dt) { return dt == DUA_DTYPE_F32 ? 4 : 2; }
static inline bool dua_dtype_ok(int dt) { return dt == DUA_DTYPE_F32 || dt == DUA_DTYPE_BF16 || dt == DUA_DTYPE_F16; }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
