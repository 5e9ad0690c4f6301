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
// ... in memory at any address aligned to its elements (gfx950 moves 16 bytes from any of them in one instruction)
template <typename T, int N> struct MemVec { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };

// N consecutive elements as floats
template <typename T, int N>
__device__ __forceinline__ void ld_elems(const T* p, float* f) {
    const typename VecOf<T, N>::type v = *(const typename MemVec<T, N>::type*)p;
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = (float)v[j];
}
// ... and back, rounded to nearest once
template <typename T, int N>
__device__ __forceinline__ void st_elems(T* p, const float* f) {
    typename VecOf<T, N>::type v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)f[j];
    *(typename MemVec<T, N>::type*)p = v;
}

static inline size_t dua_dtype_size(int dt) { return dt == DUA_DTYPE_F32 ? 4 : 2; }
static inline bool dua_dtype_ok(int dt) { return dt == DUA_DTYPE_F32 || dt == DUA_DTYPE_BF16 || dt == DUA_DTYPE_F16; }

// Sums over a wavefront (or its first 16 lanes) in the lanes' own order, on the data-parallel path of the vector unit: a handful of cycles a
// step where a shuffle through LDS takes some sixty.  EXEC must be full.
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL> __device__ __forceinline__ float dpp_move(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true)); }
__device__ __forceinline__ float lane_of(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ float row_scan(float v) {          // lane 15 of every 16: the sum of its row
    v = dpp_add<0x111, 0xF>(v);
    v = dpp_add<0x112, 0xF>(v);
    v = dpp_add<0x114, 0xF>(v);
    return dpp_add<0x118, 0xF>(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    v = row_scan(v);
    v = dpp_add<0x142, 0xA>(v);                                // lane 15 of rows 0, 2 into rows 1, 3
    v = dpp_add<0x143, 0xC>(v);                                // lane 31 into rows 2, 3
    return lane_of(v, 63);
}
__device__ __forceinline__ float row_sum16(float v) { return lane_of(row_scan(v), 15); }
