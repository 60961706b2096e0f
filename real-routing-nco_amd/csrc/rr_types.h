// Element types of the operators that serve float32, float16 and bfloat16 alike (rr_norm.hip, rr_xattn.hip, rr_draw.hip).
// Every sum, maximum and statistic is held in 32 bits or more; a value is rounded to its type once, when it is stored.
#pragma once
#include "rr_common.h"
#include "../../include/rrnco_hip.h"      // the entry points and structs as callers see them

#define RR_F32 0
#define RR_F16 1
#define RR_BF16 2

typedef _Float16 rr_f16;
typedef __bf16 rr_bf16;

template <typename T> struct rr_vec_of;                     // 16 bytes of T
template <> struct rr_vec_of<float> { static constexpr int N = 4; };
template <> struct rr_vec_of<rr_f16> { static constexpr int N = 8; };
template <> struct rr_vec_of<rr_bf16> { static constexpr int N = 8; };

// N consecutive elements as floats by one access of N elements; the address needs the element's alignment only (global memory takes 16 bytes at any place:
// rows of odd widths and odd strides go the same way as others)
template <typename T, int N>
__device__ __forceinline__ void rr_load_n(const T* __restrict__ p, float (&x)[N]) {
  if constexpr (N == 1) {
    x[0] = (float)p[0];
  } else {
    static_assert(N * sizeof(T) == 16, "one 16-byte access");
    typedef T V __attribute__((ext_vector_type(N)));
    typedef V U __attribute__((aligned(sizeof(T))));
    const V v = *reinterpret_cast<const U*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
  }
}
template <typename T, int N>
__device__ __forceinline__ void rr_store_n(T* __restrict__ p, const float (&x)[N]) {
  static_assert(N * sizeof(T) == 16, "one 16-byte access");
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V U __attribute__((aligned(sizeof(T))));
  V v;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (T)x[i];
  *reinterpret_cast<U*>(p) = v;
}
// the first n of them (the others as zeros, unwritten)
template <typename T, int N>
__device__ __forceinline__ void rr_load_first(const T* __restrict__ p, int n, float (&x)[N]) {
  if (n >= N) rr_load_n<T, N>(p, x);
  else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < n ? (float)p[i] : 0.f;
  }
}
template <typename T, int N>
__device__ __forceinline__ void rr_store_first(T* __restrict__ p, int n, const float (&x)[N]) {
  if (n >= N) rr_store_n<T, N>(p, x);
  else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) p[i] = (T)x[i];
  }
}
__host__ __forceinline__ bool rr_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
