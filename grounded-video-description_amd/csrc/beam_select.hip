// Beam search's selection over beams and vocabulary, and the reordering of the beams' states.
//
//   lp[q,v]   = x[q,v] - log sum_v exp(x[q,v])                       log-softmax of beam q's logits
//   cand[q,v] = score[q] + lp[q,v]     an ended beam: score[q] for the end word, -inf for the others
//                                      a beam whose score or log-sum-exp is not finite (all words banned, NaN or +inf logits,
//                                      a beam that is not in use yet): -inf for all words
//   the `width` largest of the K * V candidates of a sample, descending, equal ones by q * V + v ascending
//
// Bound by the logits, which are read once: one launch walks them with the running maximum and sum of the softmax and keeps the
// `width` best of each part of a row, a second one joins the parts and the beams of a sample.  The best words of a row are its
// largest logits, so the walk compares logits; only the join, a few candidates per beam, needs scores, and computes them in
// fp64: two beams' candidates may lie closer together than fp32 tells apart.
#include "dtypes.h"
#include <math.h>

namespace {

constexpr int MAX_BEAMS = GVD_BEAM_SELECT_MAX, MAX_WIDTH = GVD_BEAM_SELECT_MAX;
constexpr int MAX_PARTS = 64;             // parts of a row: one lane each in the join
constexpr int LIST = 512;                 // words at or over the threshold that one tile may have before it is ranked the slow way

typedef unsigned long long u64;

// order-preserving bits of a logit (no NaN) in the upper half, the word's complement below: larger = better, ties to the lower
// word.  -0 counts as +0.  0 = no word.
__device__ __forceinline__ unsigned order_bits(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order_bits(unsigned u) {
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ u64 make_key(unsigned bits, int word) { return ((u64)bits << 32) | (unsigned)~word; }
__device__ __forceinline__ int key_word(u64 k) { return (int)~(unsigned)k; }

struct SelectArgs {
  const void* logits; int64_t ld;
  const float* scores; const uint8_t* finished;
  int B, K, V, W, eos;
  int parts, tiles_per_part;
  double2* stat;                          // [rows][parts] (maximum, sum of exp(x - maximum))
  u64* best;                              // [rows][parts][W] descending
  float* out_scores; int64_t* parent; int64_t* word; uint8_t* out_finished;
};

__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const u64 o = __shfl_xor(v, off, GVD_WAVE);
    v = o > v ? o : v;
  }
  return v;
}

// One part of one row.  A thread holds IPT logits of a tile.  Threshold: among the 64 lanes' maxima of a wave, the W-th largest
// is at most the W-th largest logit of the tile, so only logits at or over (the largest such value of the four waves) can be among
// the best W: usually a few more than W.  They are put on a list and ranked against each other.
template <typename T, int IPT>
__global__ __launch_bounds__(256) void beam_part_kernel(const SelectArgs a) {
  constexpr int N = IPT < 16 / (int)sizeof(T) ? IPT : 16 / (int)sizeof(T);
  constexpr int TILE = 256 * IPT;
  __shared__ u64 s_list[LIST];
  __shared__ u64 s_best[MAX_WIDTH];
  __shared__ float s_max[4];
  __shared__ unsigned s_thr[4];
  __shared__ u64 s_top[4];
  __shared__ double s_sum[4];
  __shared__ int s_n;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row = blockIdx.y;
  if (a.finished && a.finished[row]) return;
  if (!(fabsf(a.scores[row]) < INFINITY)) return;
  const int W = a.W, V = a.V;
  const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  double sum = 0.0;
  float top = -INFINITY;
  if (tid < MAX_WIDTH) s_best[tid] = 0;
  if (tid == 0) s_n = 0;
  const int64_t first = (int64_t)blockIdx.x * a.tiles_per_part;
  for (int t = 0; t < a.tiles_per_part; ++t) {
    const int64_t v0 = (first + t) * TILE;
    if (v0 >= V) break;
    float v[IPT];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < IPT / N; ++i) {
      const int64_t at = v0 + (int64_t)(i * 256 + tid) * N;
      float y[N];
      if (at + N <= V) gvd_load<T, N>(x + at, y);
      else {
#pragma unroll
        for (int k = 0; k < N; ++k) y[k] = at + k < V ? (float)x[at + k] : -INFINITY;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) { v[i * N + k] = y[k]; mx = fmaxf(mx, y[k]); }
    }
    // W-th largest of the lanes' maxima, bit by bit
    const unsigned mine = order_bits(mx);
    unsigned thr = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned c = thr | (1u << bit);
      if (__popcll(__ballot(mine >= c)) >= W) thr = c;
    }
    mx = wave_max(mx);
    if ((tid & 63) == 0) { s_max[wave] = mx; s_thr[wave] = thr; }
    __syncthreads();
    mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    thr = max(max(s_thr[0], s_thr[1]), max(s_thr[2], s_thr[3]));
    thr = max(thr, (unsigned)(s_best[W - 1] >> 32));
    const float was = top;
    top = fmaxf(top, mx);
    const float ref = top > -INFINITY ? top : 0.f;           // (nothing but -inf so far: every term is exp(-inf) = 0)
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < IPT; ++i) part += expf(v[i] - ref);
    sum = sum * (double)expf(was - ref) + (double)part;
    // the list: the best of the tiles before, then this tile's words at or over the threshold
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int64_t at = v0 + (int64_t)((i / N) * 256 + tid) * N + i % N;
      const unsigned u = order_bits(v[i]);
      if (u >= thr && at < V) {
        const int k = atomicAdd(&s_n, 1);
        if (k < LIST - MAX_WIDTH) s_list[MAX_WIDTH + k] = make_key(u, (int)at);
      }
    }
    if (tid < MAX_WIDTH) s_list[tid] = s_best[tid];
    __syncthreads();
    const int n = s_n;
    if (n <= LIST - MAX_WIDTH) {
      for (int i = tid; i < MAX_WIDTH + n; i += 256) {
        const u64 k = s_list[i];
        int rank = 0;
        for (int j = 0; j < MAX_WIDTH + n; ++j) rank += s_list[j] > k;
        if (k && rank < W) s_best[rank] = k;
      }
    } else {
      // more words at the threshold than the list holds (equal logits): W times the best of what is left
      u64 last = ~0ull;
      for (int r = 0; r < W; ++r) {
        u64 k = 0;
        if (tid < MAX_WIDTH && s_list[tid] < last) k = s_list[tid];
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
          const int64_t at = v0 + (int64_t)((i / N) * 256 + tid) * N + i % N;
          const u64 c = at < V ? make_key(order_bits(v[i]), (int)at) : 0;
          if (c < last && c > k) k = c;
        }
        k = wave_max_u64(k);
        if ((tid & 63) == 0) s_top[wave] = k;
        __syncthreads();
        k = s_top[0];
#pragma unroll
        for (int w = 1; w < 4; ++w) k = s_top[w] > k ? s_top[w] : k;
        if (tid == 0) s_best[r] = k;
        last = k;
        __syncthreads();
      }
    }
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, GVD_WAVE);
  if ((tid & 63) == 0) s_sum[wave] = sum;
  __syncthreads();
  const int64_t rec = (int64_t)row * a.parts + blockIdx.x;
  if (tid == 0) a.stat[rec] = make_double2((double)top, (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]));
  if (tid < W) a.best[rec * W + tid] = s_best[tid];
}

// One workgroup per sample, one wave per beam (and the beams 16 further on): a lane holds the head of one part's list, the
// wave takes the best head W times.  Then the first wave does the same over the beams' lists.
__global__ __launch_bounds__(1024) void beam_join_kernel(const SelectArgs a) {
  __shared__ double s_score[MAX_BEAMS][MAX_WIDTH];
  __shared__ int s_word[MAX_BEAMS][MAX_WIDTH];
  const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int K = a.K, W = a.W, V = a.V;
  for (int q = wave; q < K; q += waves) {
    const int row = b * K + q;
    const float score = a.scores[row];
    const bool over = a.finished && a.finished[row];
    bool live = fabsf(score) < INFINITY;
    if (live && over) {
      if (lane < W) {
        const int w = lane == 0 ? a.eos : lane - 1 < a.eos ? lane - 1 : lane;
        s_score[q][lane] = lane == 0 ? (double)score : -INFINITY;
        s_word[q][lane] = w < V ? w : -1;
      }
      continue;
    }
    double lse = 0.0;
    if (live) {
      const int64_t rec = (int64_t)row * a.parts + lane;
      const double2 st = lane < a.parts ? a.stat[rec] : make_double2(-INFINITY, 0.0);
      double m = st.x;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) m = fmax(m, __shfl_xor(m, off, GVD_WAVE));
      double s = lane < a.parts && st.y != 0.0 ? st.y * exp(st.x - m) : 0.0;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, GVD_WAVE);
      lse = m + log(s);
      live = fabs(lse) < INFINITY;
    }
    if (!live) {
      if (lane < W) {
        s_score[q][lane] = -INFINITY;
        s_word[q][lane] = lane < V ? lane : -1;
      }
      continue;
    }
    const u64* list = a.best + ((int64_t)row * a.parts + lane) * W;
    int at = 0;
    u64 head = lane < a.parts ? list[0] : 0;
    for (int r = 0; r < W; ++r) {
      const u64 k = wave_max_u64(head);
      if (lane == 0) {
        s_score[q][r] = (double)score + ((double)from_order_bits((unsigned)(k >> 32)) - lse);
        s_word[q][r] = k ? key_word(k) : -1;
      }
      if (k && head == k) head = ++at < W ? list[at] : 0;
    }
  }
  __syncthreads();
  if (wave) return;
  int at = 0, my_beam = 0, my_word = 0;
  double my_score = 0.0;
  for (int r = 0; r < W; ++r) {
    const bool have = lane < K && at < W && s_word[lane][at] >= 0;
    double sc = have ? s_score[lane][at] : -INFINITY;
    int who = have ? lane : 64 + lane;                       // (no candidate left: after every lane that has one)
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const double os = __shfl_xor(sc, off, GVD_WAVE);
      const int ow = __shfl_xor(who, off, GVD_WAVE);
      if (os > sc || (os == sc && ow < who)) { sc = os; who = ow; }
    }
    const int beam = who & 63;
    const int w = s_word[beam][__shfl(at, beam, GVD_WAVE)];
    if (lane == r) { my_score = sc; my_beam = beam; my_word = w; }
    if (lane == beam) ++at;
  }
  if (lane < W) {
    const int64_t o = (int64_t)b * W + lane;
    a.out_scores[o] = (float)my_score;
    a.parent[o] = (int64_t)b * K + my_beam;
    a.word[o] = my_word;
    if (a.out_finished) a.out_finished[o] = my_word == a.eos || (a.finished && a.finished[b * K + my_beam]);
  }
}

// words of one workgroup's tile, parts of a row
struct SelectShape { int ipt, parts, tiles_per_part; };

SelectShape select_shape(int64_t rows, int V) {
  SelectShape s;
  s.ipt = 32;
  while (s.ipt > 4 && (rows * ((V + 256 * s.ipt - 1) / (256 * s.ipt)) < 512 || 128 * s.ipt >= V)) s.ipt /= 2;
  const int tiles = (V + 256 * s.ipt - 1) / (256 * s.ipt);
  s.tiles_per_part = (tiles + MAX_PARTS - 1) / MAX_PARTS;
  s.parts = (tiles + s.tiles_per_part - 1) / s.tiles_per_part;
  return s;
}

template <typename T> void launch_parts(const SelectArgs& a, int ipt, hipStream_t st) {
  const dim3 grid((unsigned)a.parts, (unsigned)(a.B * a.K));
  if (ipt == 32) hipLaunchKernelGGL((beam_part_kernel<T, 32>), grid, dim3(256), 0, st, a);
  else if (ipt == 16) hipLaunchKernelGGL((beam_part_kernel<T, 16>), grid, dim3(256), 0, st, a);
  else if (ipt == 8) hipLaunchKernelGGL((beam_part_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((beam_part_kernel<T, 4>), grid, dim3(256), 0, st, a);
}

bool bad_select_shape(int B, int K, int V, int W) {
  return B <= 0 || K <= 0 || K > MAX_BEAMS || V <= 0 || W <= 0 || W > MAX_WIDTH || (int64_t)K * V < W || (int64_t)B * K > 65535 ||
         V > (1 << 28);
}

// ------------------------------------------------------------------------------------------------------------- reorder
// dst[o, r, :] = src[o, index[r], :], up to GVD_REORDER_MAX_TENSORS tensors in a launch.  A copy: bound by reading and writing
// the rows once.  A thread copies four units of 16 bytes; the last unit of a row is moved back so that it ends with the row
// (rows under 16 bytes: units of the largest power of two that divides them).
constexpr int UNITS = 1024;               // units of one workgroup

template <int BYTES> struct Unit;
template <> struct Unit<16> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(1))); };
template <> struct Unit<8> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(1))); };
template <> struct Unit<4> { typedef unsigned type __attribute__((aligned(1))); };
template <> struct Unit<2> { typedef uint16_t type __attribute__((aligned(1))); };
template <> struct Unit<1> { typedef uint8_t type; };

template <int BYTES>
__device__ void reorder_tile(const gvd_reorder_tensor& t, const int64_t* __restrict__ index, int64_t rows_in, int64_t rows_out,
                             int64_t tile) {
  typedef typename Unit<BYTES>::type U;
  const int64_t per_row = (t.row_bytes + BYTES - 1) / BYTES, total = t.outer * rows_out * per_row;
  const char* src[4];
  char* dst[4];
  int live = 0;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = tile * UNITS + u * 256 + threadIdx.x;
    src[u] = nullptr; dst[u] = nullptr;
    if (i < total) {
      const int64_t row = i / per_row, o = row / rows_out, r = row - o * rows_out;
      int64_t off = (i - row * per_row) * BYTES;
      if (off + BYTES > t.row_bytes) off = t.row_bytes - BYTES;
      const int64_t from = index[r];
      dst[u] = reinterpret_cast<char*>(t.dst) + o * t.dst_outer + r * t.dst_row + off;
      if (from >= 0 && from < rows_in) src[u] = reinterpret_cast<const char*>(t.src) + o * t.src_outer + from * t.src_row + off;
      live = u + 1;
    }
  }
  U x[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (src[u]) x[u] = *reinterpret_cast<const U*>(src[u]);
    else x[u] = (U)~(U)0;                                     // an index outside the rows: nothing is read, all bits set
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (u < live) *reinterpret_cast<U*>(dst[u]) = x[u];
}

__global__ __launch_bounds__(256) void reorder_rows_kernel(const gvd_reorder_group g, const int64_t* __restrict__ index,
                                                           int64_t rows_in, int64_t rows_out) {
  int t = 0;
  while (t + 1 < g.count && (int64_t)blockIdx.x >= g.tile0[t + 1]) ++t;
  const gvd_reorder_tensor& x = g.t[t];
  const int64_t tile = (int64_t)blockIdx.x - g.tile0[t];
  switch (x.unit) {
    case 16: reorder_tile<16>(x, index, rows_in, rows_out, tile); break;
    case 8: reorder_tile<8>(x, index, rows_in, rows_out, tile); break;
    case 4: reorder_tile<4>(x, index, rows_in, rows_out, tile); break;
    case 2: reorder_tile<2>(x, index, rows_in, rows_out, tile); break;
    default: reorder_tile<1>(x, index, rows_in, rows_out, tile); break;
  }
}

}  // namespace

extern "C" size_t gvd_beam_select_workspace_bytes(int B, int K, int V, int W) {
  if (bad_select_shape(B, K, V, W)) return 0;
  const int64_t rows = (int64_t)B * K;
  const SelectShape s = select_shape(rows, V);
  return (size_t)(rows * s.parts * (16 + 8 * (int64_t)W));
}

extern "C" int gvd_beam_select(const gvd_beam_select_args* g, gvd_stream_t stream) {
  if (!g || bad_select_shape(g->B, g->K, g->V, g->W) || !gvd_dtype_bytes(g->dtype) || !g->logits || g->ld < g->V || !g->scores ||
      !g->out_scores || !g->parent || !g->word || !g->workspace || !gvd_aligned16(g->workspace) || g->eos < -1 || g->eos >= g->V ||
      (g->finished && g->eos < 0) || g->workspace_bytes < gvd_beam_select_workspace_bytes(g->B, g->K, g->V, g->W))
    return GVD_EINVAL;
  const int64_t rows = (int64_t)g->B * g->K;
  const SelectShape s = select_shape(rows, g->V);
  SelectArgs a = {};
  a.logits = g->logits; a.ld = g->ld;
  a.scores = g->scores; a.finished = g->finished;
  a.B = g->B; a.K = g->K; a.V = g->V; a.W = g->W; a.eos = g->eos;
  a.parts = s.parts; a.tiles_per_part = s.tiles_per_part;
  a.stat = reinterpret_cast<double2*>(g->workspace);
  a.best = reinterpret_cast<u64*>(a.stat + rows * s.parts);
  a.out_scores = g->out_scores; a.parent = g->parent; a.word = g->word; a.out_finished = g->out_finished;
  const hipStream_t st = gvd_s(stream);
  if (g->dtype == GVD_F32) launch_parts<float>(a, s.ipt, st);
  else if (g->dtype == GVD_BF16) launch_parts<gvd_bf16>(a, s.ipt, st);
  else launch_parts<gvd_f16>(a, s.ipt, st);
  GVD_CHECK_LAUNCH();
  const int waves = g->K < 16 ? g->K : 16;
  hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)g->B), dim3((unsigned)(64 * waves)), 0, st, a);
  GVD_CHECK_LAUNCH();
  return 0;
}

extern "C" int gvd_reorder_rows(const gvd_reorder_group* group, const int64_t* index, int64_t rows_in, int64_t rows_out,
                                gvd_stream_t stream) {
  if (!group || group->count <= 0 || group->count > GVD_REORDER_MAX_TENSORS || !index || rows_in <= 0 || rows_out <= 0 ||
      rows_out > 0x7fffffffll)
    return GVD_EINVAL;
  gvd_reorder_group g = *group;
  int64_t tiles = 0;
  for (int i = 0; i < g.count; ++i) {
    gvd_reorder_tensor& t = g.t[i];
    if (!t.src || !t.dst || t.outer <= 0 || t.outer > 0x7fffffffll || t.row_bytes <= 0) return GVD_EINVAL;
    t.unit = 16;
    while (t.unit > 1 && (t.row_bytes < t.unit || (t.row_bytes < 16 && t.row_bytes % t.unit))) t.unit /= 2;
    g.tile0[i] = tiles;
    const int64_t per_row = (t.row_bytes + t.unit - 1) / t.unit;
    if (per_row > (1ll << 33) / (t.outer * rows_out)) return GVD_EINVAL;     // (a launch holds fewer than 2^32 threads)
    tiles += (t.outer * rows_out * per_row + UNITS - 1) / UNITS;
  }
  g.tile0[g.count] = tiles;
  if (tiles > (1ll << 23)) return GVD_EINVAL;
  hipLaunchKernelGGL(reorder_rows_kernel, dim3((unsigned)tiles), dim3(256), 0, gvd_s(stream), g, index, rows_in, rows_out);
  GVD_CHECK_LAUNCH();
  return 0;
}
