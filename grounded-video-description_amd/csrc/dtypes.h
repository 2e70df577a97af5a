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

// The same past the caches: for tensors that do not fit them, whose lines would only push others out.
template <typename T, int N> __device__ __forceinline__ void gvd_store_past(T* p, const float (&v)[N]) {
  typename GvdVec<T, N>::type x;
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = (T)v[k];
  __builtin_nontemporal_store(x, reinterpret_cast<typename GvdVec<T, N>::loose*>(p));
}

constexpr int64_t GVD_CACHE_BYTES = 256ll << 20;         // last-level cache

// LDS accesses of the lanes of one wave before it happen before those after it
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Reductions over a wave on the vector ALU: a lane takes its partner's value by DPP - within 4, 8, 16 lanes, then lane 15 of a
// row of 16 to the next row, lane 31 to the upper half - so that lane 63 ends with the result (a shuffle goes by way of the LDS
// unit and takes some ten times as long).  `none`: what lanes without a partner take.
template <int STEP> __device__ __forceinline__ unsigned gvd_dpp(unsigned x, unsigned none) {
  constexpr int ctrl[6] = {0xb1, 0x4e, 0x141, 0x140, 0x142, 0x143};      // quad 1032, quad 2301, half row and row mirrored, broadcasts
  constexpr int rows[6] = {0xf, 0xf, 0xf, 0xf, 0xa, 0xc};
  return (unsigned)__builtin_amdgcn_update_dpp((int)none, (int)x, ctrl[STEP], rows[STEP], 0xf, false);
}
template <int STEP> __device__ __forceinline__ double gvd_dpp(double x, double none) {
  const uint64_t a = __builtin_bit_cast(uint64_t, x), b = __builtin_bit_cast(uint64_t, none);
  const uint64_t lo = gvd_dpp<STEP>((unsigned)a, (unsigned)b), hi = gvd_dpp<STEP>((unsigned)(a >> 32), (unsigned)(b >> 32));
  return __builtin_bit_cast(double, lo | hi << 32);
}
__device__ __forceinline__ double gvd_lane63(double x) {
  const uint64_t a = __builtin_bit_cast(uint64_t, x);
  const uint64_t lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)a, 63);
  const uint64_t hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(a >> 32), 63);
  return __builtin_bit_cast(double, lo | hi << 32);
}
__device__ __forceinline__ double gvd_wave_sum_f64(double x) {
  x += gvd_dpp<0>(x, 0.0); x += gvd_dpp<1>(x, 0.0); x += gvd_dpp<2>(x, 0.0);
  x += gvd_dpp<3>(x, 0.0); x += gvd_dpp<4>(x, 0.0); x += gvd_dpp<5>(x, 0.0);
  return gvd_lane63(x);
}

static inline int gvd_dtype_bytes(int dtype) { return dtype == GVD_F32 ? 4 : (dtype == GVD_BF16 || dtype == GVD_F16) ? 2 : 0; }
