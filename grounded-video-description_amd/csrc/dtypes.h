// Element types of the kernels that take 32- and 16-bit tensors (GVD_F32 / GVD_BF16 / GVD_F16 of include/gvd_hip.h): all
// arithmetic is fp32 (or wider); a value is rounded once, to nearest even, where it is stored.
//
// Vectors are read and written at the alignment of ONE element: rows of odd width, views into flat buffers and offset columns
// go through the same 16-byte instructions as aligned ones (gfx950 global memory accesses need no more than that).
#pragma once
#include "gvd_common.h"

typedef __bf16 gvd_bf16;
typedef _Float16 gvd_f16;

template <typename T, int N> struct GvdVec {
  typedef T type __attribute__((ext_vector_type(N)));
  typedef type loose __attribute__((aligned(sizeof(T))));
};

// N elements at p (element-aligned) -> fp32
template <typename T, int N> __device__ __forceinline__ void gvd_load(const T* p, float (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = (float)p[0];
  } else {
    const typename GvdVec<T, N>::loose x = *reinterpret_cast<const typename GvdVec<T, N>::loose*>(p);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = (float)x[k];
  }
}

template <typename T, int N> __device__ __forceinline__ void gvd_store(T* p, const float (&v)[N]) {
  if constexpr (N == 1) {
    p[0] = (T)v[0];
  } else {
    typename GvdVec<T, N>::type x;
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = (T)v[k];
    *reinterpret_cast<typename GvdVec<T, N>::loose*>(p) = x;
  }
}

// the first `left` (< N) of N elements; the rest of v is 0
template <typename T, int N> __device__ __forceinline__ void gvd_load_part(const T* p, int left, float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = k < left ? (float)p[k] : 0.f;
}

template <typename T, int N> __device__ __forceinline__ void gvd_store_part(T* p, int left, const float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (k < left) p[k] = (T)v[k];
}

// LDS accesses of the lanes of one wave before it happen before those after it
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

static inline int gvd_dtype_bytes(int dtype) { return dtype == GVD_F32 ? 4 : (dtype == GVD_BF16 || dtype == GVD_F16) ? 2 : 0; }
