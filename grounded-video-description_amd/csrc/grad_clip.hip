// The global L2 norm of many gradient tensors, and clipping:
//
//   norm = inv_scale * sqrt(sum over all tensors and elements of g^2),   factor = min(1, max_norm / (norm + 1e-6)) * inv_scale
//   dst  = factor * g     (in place, or into other tensors: 16-bit gradients of a scaled loss into fp32 master gradients)
//
// Bound by memory: the norm has to be known before the first element is written, so the gradients are read twice and written
// once.  Squares and sums are fp64 - no gradient that fp32 holds, 1e-45 to 3e38, vanishes or overflows in them - and added in a
// fixed order (no atomics).  Two kinds of launch: gvd_grad_sumsq leaves one partial sum per workgroup; in gvd_grad_scale every
// workgroup adds up all the partials by itself, in the same order, so no launch is spent on joining them.
//
// Measured, 100 tensors of 2.5 M elements bf16 -> fp32: norm 84 us (6.0 TB/s), both 312 us; 10 tensors of 4 M fp32: 30 and 82
// us. What got it there from 128 + 294 us: a whole chunk in flight before its first use, stores and second reads past the cache
// (394 -> 330 us), eight workgroups of the second pass for each resident one (330 -> 312), destinations taken from their
// 128-byte lines on (views of a flat buffer at odd offsets: 368 -> 332).
//
// Up to GVD_GRAD_MAX_TENSORS tensors go into a launch by value (addresses and sizes in the kernel's arguments); a workgroup
// finds the tensor of its chunk by bisection in the chunk counts.
#include "dtypes.h"

namespace {

constexpr int CHUNK = GVD_GRAD_CHUNK;
constexpr int MAX_GRID = 1024;

// A chunk's tensor: the lanes hold the tensors' first chunks (two each) and count those at or before it.
struct FirstChunks {
  unsigned a, b;
  __device__ __forceinline__ FirstChunks(const gvd_grad_group& g) {
    const int lane = threadIdx.x & 63;
    a = lane < g.count ? g.chunk0[lane] : 0xffffffffu;
    b = lane + 64 < g.count ? g.chunk0[lane + 64] : 0xffffffffu;
  }
  __device__ __forceinline__ int tensor_of(unsigned chunk) const {
    return __popcll(__ballot(a <= chunk)) + __popcll(__ballot(b <= chunk)) - 1;
  }
};

__device__ __forceinline__ double block_sum_f64(double v, double* s_red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, GVD_WAVE);
  if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
}

// A full chunk is loaded as a whole, 16 bytes a lane and instruction, before its first element is used.
template <typename T> __device__ __forceinline__ double chunk_sumsq(const T* p, int64_t n) {
  constexpr int N = 16 / sizeof(T), VECS = CHUNK / (256 * N);
  typedef typename GvdVec<T, N>::loose Loose;
  double s = 0.0;
  if (n == CHUNK) {
    typename GvdVec<T, N>::type x[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) x[i] = *reinterpret_cast<const Loose*>(p + (i * 256 + threadIdx.x) * N);
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) { const double v = (float)x[i][k]; s = fma(v, v, s); }
    return s;
  }
  const int64_t nv = n / N * N;
  for (int64_t i = (int64_t)threadIdx.x * N; i < nv; i += 256 * N) {
    float v[N];
    gvd_load<T, N>(p + i, v);
#pragma unroll
    for (int k = 0; k < N; ++k) s = fma((double)v[k], (double)v[k], s);
  }
  for (int64_t i = nv + threadIdx.x; i < n; i += 256) { const double v = (float)p[i]; s = fma(v, v, s); }
  return s;
}

__global__ __launch_bounds__(256) void grad_sumsq_kernel(const gvd_grad_group g, double* __restrict__ partials) {
  __shared__ double s_red[4];
  double s = 0.0;
  const FirstChunks first(g);
  const unsigned chunks = g.chunk0[g.count];
  for (unsigned c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = first.tensor_of(c);
    const int64_t e0 = (int64_t)(c - g.chunk0[t]) * CHUNK;
    const int64_t n = g.n[t] - e0 < CHUNK ? g.n[t] - e0 : CHUNK;
    if (g.src_type[t] == GVD_F32) s += chunk_sumsq(reinterpret_cast<const float*>(g.src[t]) + e0, n);
    else if (g.src_type[t] == GVD_BF16) s += chunk_sumsq(reinterpret_cast<const gvd_bf16*>(g.src[t]) + e0, n);
    else s += chunk_sumsq(reinterpret_cast<const gvd_f16*>(g.src[t]) + e0, n);
  }
  s = block_sum_f64(s, s_red);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// the factor as f 2^e: f is a normal fp32 number (or 0), e is 0 but for factors under 2^-100 (large norms) and over 2^100 (tiny loss
// scales, where f is at least 2^63 and so no product of it is subnormal)
struct Factor { float f; int e; };
__device__ __forceinline__ Factor factor_of(double factor) {
  int e = 0;
  if (factor < 0x1p-100) factor = frexp(factor, &e);
  else if (factor > 0x1p100) { factor = frexp(factor, &e) * 0x1p64; e -= 64; }
  return {(float)factor, e};
}
__device__ __forceinline__ float operator*(float x, Factor f) { return ldexpf(x * f.f, f.e); }

template <bool PAST, typename TI, typename TO>
__device__ __forceinline__ void chunk_scale(const TI* src, TO* dst, int64_t n, Factor f) {
  constexpr int N = 16 / (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO)), VECS = CHUNK / (256 * N);
  if (n == CHUNK) {
    typename GvdVec<TI, N>::type x[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const auto* from = reinterpret_cast<const typename GvdVec<TI, N>::loose*>(src + (i * 256 + threadIdx.x) * N);
      if constexpr (PAST) x[i] = __builtin_nontemporal_load(from); else x[i] = *from;
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      float v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = (float)x[i][k] * f;
      if constexpr (PAST) gvd_store_past<TO, N>(dst + (i * 256 + threadIdx.x) * N, v);
      else gvd_store<TO, N>(dst + (i * 256 + threadIdx.x) * N, v);
    }
    return;
  }
  const int64_t nv = n / N * N;
  for (int64_t i = (int64_t)threadIdx.x * N; i < nv; i += 256 * N) {
    float v[N];
    gvd_load<TI, N>(src + i, v);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = v[k] * f;
    gvd_store<TO, N>(dst + i, v);
  }
  for (int64_t i = nv + threadIdx.x; i < n; i += 256) dst[i] = (TO)((float)src[i] * f);
}

// Chunk k of a tensor.  Its chunks begin where the destination begins a 128-byte line (the first one holds what lies before,
// too): results that are views of a flat buffer begin anywhere, and stores of parts of lines cost more than such loads.
template <bool PAST, typename TI, typename TO>
__device__ __forceinline__ void scale_chunk(const TI* src, TO* dst, int64_t k, int64_t n, Factor f) {
  const int64_t before = (int64_t)((128u - (unsigned)(reinterpret_cast<uintptr_t>(dst) & 127u)) % 128u / sizeof(TO));
  if (k == 0 && threadIdx.x < before && threadIdx.x < n) dst[threadIdx.x] = (TO)((float)src[threadIdx.x] * f);
  const int64_t e0 = k * CHUNK + before, e1 = e0 + CHUNK < n ? e0 + CHUNK : n;
  if (e0 < e1) chunk_scale<PAST>(src + e0, dst + e0, e1 - e0, f);
}

template <bool PAST, typename TI>
__device__ __forceinline__ void scale_to(const TI* src, void* dst, int type, int64_t k, int64_t n, Factor f) {
  if (type == GVD_F32) scale_chunk<PAST>(src, reinterpret_cast<float*>(dst), k, n, f);
  else if (type == GVD_BF16) scale_chunk<PAST>(src, reinterpret_cast<gvd_bf16*>(dst), k, n, f);
  else scale_chunk<PAST>(src, reinterpret_cast<gvd_f16*>(dst), k, n, f);
}

template <bool PAST>
__global__ __launch_bounds__(256) void grad_scale_kernel(const gvd_grad_group g, const gvd_grad_clip c,
                                                         const double* __restrict__ partials, int n_partials, float* norm_out) {
  __shared__ double s_red[4];
  double s = 0.0;
  for (int i = threadIdx.x; i < n_partials; i += 256) s += partials[i];
  const double norm = sqrt(block_sum_f64(s, s_red)) * c.inv_scale;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double clip = c.max_norm / (norm + 1e-6);
  const double factor = (clip > 1.0 ? 1.0 : clip) * c.inv_scale;           // (a NaN norm makes every gradient NaN)
  const Factor f = factor_of(factor);
  const unsigned chunks = g.count ? g.chunk0[g.count] : 0;
  const FirstChunks first(g);
  // from the last chunk to the first: what gvd_grad_sumsq read last is still in the 256 MB cache
  for (unsigned at = blockIdx.x; at < chunks; at += gridDim.x) {
    const unsigned k = chunks - 1 - at;
    const int t = first.tensor_of(k);
    if (factor == 1.0 && g.src[t] == g.dst[t]) continue;                       // in place and nothing to clip
    const int64_t at_t = k - g.chunk0[t], n = g.n[t];
    const int to = g.dst_type[t];
    if (g.src_type[t] == GVD_F32) scale_to<PAST>(reinterpret_cast<const float*>(g.src[t]), g.dst[t], to, at_t, n, f);
    else if (g.src_type[t] == GVD_BF16) scale_to<PAST>(reinterpret_cast<const gvd_bf16*>(g.src[t]), g.dst[t], to, at_t, n, f);
    else scale_to<PAST>(reinterpret_cast<const gvd_f16*>(g.src[t]), g.dst[t], to, at_t, n, f);
  }
}

bool bad_group(const gvd_grad_group* g, bool need_dst) {
  if (!g || g->count < 0 || g->count > GVD_GRAD_MAX_TENSORS || g->chunk0[0] != 0) return true;
  for (int t = 0; t < g->count; ++t) {
    const int is = gvd_dtype_bytes(g->src_type[t]), os = gvd_dtype_bytes(g->dst_type[t]);
    if (!g->src[t] || g->n[t] <= 0 || !is || reinterpret_cast<uintptr_t>(g->src[t]) % is) return true;
    if (need_dst && (!g->dst[t] || !os || reinterpret_cast<uintptr_t>(g->dst[t]) % os || (g->dst[t] == g->src[t] && is != os)))
      return true;
    const int64_t chunks = (g->n[t] + CHUNK - 1) / CHUNK;
    if ((int64_t)g->chunk0[t] + chunks != (int64_t)g->chunk0[t + 1]) return true;
  }
  return false;
}

unsigned grid_of(const gvd_grad_group* g, unsigned most) {
  const unsigned chunks = g->chunk0[g->count];
  return chunks < most ? chunks : most;
}

}  // namespace

extern "C" int gvd_grad_chunk(void) { return CHUNK; }

extern "C" int gvd_grad_parts(const gvd_grad_group* g) { return bad_group(g, false) ? GVD_EINVAL : (int)grid_of(g, MAX_GRID); }

extern "C" int gvd_grad_sumsq(const gvd_grad_group* g, void* partials, gvd_stream_t stream) {
  if (bad_group(g, false) || g->count == 0 || !partials || !gvd_aligned16(partials) && reinterpret_cast<uintptr_t>(partials) % 8)
    return GVD_EINVAL;
  hipLaunchKernelGGL(grad_sumsq_kernel, dim3(grid_of(g, MAX_GRID)), dim3(256), 0, gvd_s(stream), *g,
                     reinterpret_cast<double*>(partials));
  GVD_CHECK_LAUNCH();
  return 0;
}

extern "C" int gvd_grad_scale(const gvd_grad_group* g, const gvd_grad_clip* c, const void* partials, int n_partials,
                              float* norm_out, gvd_stream_t stream) {
  if (bad_group(g, true) || !c || !(c->max_norm >= 0.0) || !(c->inv_scale > 0.0) || !partials || n_partials <= 0 ||
      reinterpret_cast<uintptr_t>(partials) % 8 || (g->count == 0 && !norm_out))
    return GVD_EINVAL;
  int64_t bytes = 0;
  for (int t = 0; t < g->count; ++t) bytes += g->n[t] * (gvd_dtype_bytes(g->src_type[t]) + gvd_dtype_bytes(g->dst_type[t]));
  const unsigned grid = g->count ? grid_of(g, 8 * MAX_GRID) : 1;
  hipLaunchKernelGGL((bytes > GVD_CACHE_BYTES ? grad_scale_kernel<true> : grad_scale_kernel<false>), dim3(grid), dim3(256), 0,
                     gvd_s(stream), *g, *c, reinterpret_cast<const double*>(partials), n_partials, norm_out);
  GVD_CHECK_LAUNCH();
  return 0;
}
