// Element vectors of the decay block's kernels: V consecutive elements of a row
// (16 bytes, or one element where a row or a width is not made of whole vectors)
// as fp32 registers, rounded once (to nearest even) where they are stored.
#pragma once
#include "grk_common.h"

namespace grk {

typedef _Float16 f16_t;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ float to_f32(f16_t x) { return (float)x; }

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) { return f32_to_bf16(x); }
// The fp32 value is pinned first: else some uses become a mixed-precision fma that rounds
// once where others round twice, and the bits depend on the path taken.
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float x) {
  asm("" : "+v"(x));
  return (f16_t)x;
}

// Elements of a 16-byte vector.
template <typename T> constexpr int vec_elems() { return 16 / (int)sizeof(T); }

template <typename T, int V>
__device__ __forceinline__ void vload(const T* p, float* f) {
  if constexpr (V == 1) {
    f[0] = to_f32(*p);
  } else {
    static_assert(V * sizeof(T) == 16, "a vector is 16 bytes");
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    T t[V];
    __builtin_memcpy(t, &w, 16);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = to_f32(t[e]);
  }
}

// PAST: the store passes the caches by.
template <typename T, int V, bool PAST = false>
__device__ __forceinline__ void vstore(T* p, const float* f) {
  if constexpr (V == 1) {
    *p = from_f32<T>(f[0]);
  } else {
    static_assert(V * sizeof(T) == 16, "a vector is 16 bytes");
    T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = from_f32<T>(f[e]);
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 w;
    __builtin_memcpy(&w, t, 16);
    if constexpr (PAST) __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
    else *reinterpret_cast<u32x4*>(p) = w;
  }
}

// One element type of the three at run time (host): f(T{}).
template <typename F>
inline int for_dtype(int dtype, F f) {
  if (dtype == GRK_F32) return f(float{});
  if (dtype == GRK_BF16) return f(bf16_t{});
  return f(f16_t{});
}

inline bool known_dtype(int dtype) { return dtype == GRK_F32 || dtype == GRK_BF16 || dtype == GRK_F16; }

// Rows of `cols` columns start on, and the stride is made of, whole 16-byte vectors.
inline bool vec_rows(const void* p, int64_t ld, int dtype) {
  return (uintptr_t)p % 16 == 0 && ld * (int64_t)dtype_size(dtype) % 16 == 0;
}

}  // namespace grk
