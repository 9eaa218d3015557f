// sp_dense_common.hpp — element types, 16-byte vectors and wave reductions of the dense operators (sp_dense.hip).
//
// Rows are read and written in vectors of 16 bytes that start at the row's first element, whatever its address: gfx950 takes
// vector accesses at any element address, so odd widths and padded rows need no other path than the row's last vector.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef long long i64;
typedef unsigned long long u64;

template <typename T> struct VecOf { static constexpr int N = 16 / sizeof(T); };

template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) RawVec {
    T v[N];
};
// N consecutive elements at any element address, as one access
template <typename T, int N> __device__ __forceinline__ RawVec<T, N> vec_load(const T *p) {
    RawVec<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int N> __device__ __forceinline__ void vec_store(T *p, const RawVec<T, N> &r) { __builtin_memcpy(p, &r, sizeof(r)); }

__device__ __forceinline__ float up(float x) { return x; }
__device__ __forceinline__ float up(__bf16 x) { return (float)x; }
__device__ __forceinline__ float up(_Float16 x) { return (float)x; }

// element i of an index array of either width
__device__ __forceinline__ i64 load_index(const void *p, int is64, i64 i) { return is64 ? ((const i64 *)p)[i] : (i64)((const int *)p)[i]; }
__device__ __forceinline__ float load_scalar(const void *p, int dtype, i64 i) {
    return dtype == 0 ? ((const float *)p)[i] : dtype == 1 ? (float)((const __bf16 *)p)[i] : (float)((const _Float16 *)p)[i];
}

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32: 1 ulp, results below 2^-126 become 0

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

constexpr float NEG_INF = -__builtin_inff();

}  // namespace
