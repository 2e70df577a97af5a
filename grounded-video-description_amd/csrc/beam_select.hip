// Beam search's selection over beams and vocabulary, and the reordering of the beams' states.
//
//   lp[q,v]   = x[q,v] - log sum_v exp(x[q,v])                       log-softmax of beam q's logits
//   cand[q,v] = score[q] + lp[q,v]     an ended beam: score[q] for the end word, -inf for the others
//                                      a beam whose score or log-sum-exp is not finite (all words banned, NaN or +inf logits,
//                                      a beam that is not in use yet): -inf for all words
//   the `width` largest of the K * V candidates of a sample, descending, equal ones by q * V + v ascending
//
// One launch walks the logits, once, with the running maximum and sum of the softmax and keeps the `width` best of each part of a
// row, a second one joins the parts and the beams of a sample.  The best words of a row are its largest logits, so the walk
// compares logits.  Two beams' candidates may lie closer together than fp32 tells apart, and their order hangs on the beams'
// log-sum-exps: exponentials, sums, logarithm and candidates are fp64 throughout (good to some 1e-14; with fp32 exponentials, 1e-7,
// beams closer than that came out in either order).
#include "dtypes.h"
#include <math.h>

namespace {

constexpr int MAX_BEAMS = GVD_BEAM_SELECT_MAX, MAX_WIDTH = GVD_BEAM_SELECT_MAX;
constexpr int MAX_PARTS = 64;             // parts of a row: one lane each in the join
constexpr int JOIN_LIST = 256;            // words of all parts of a row
constexpr int LIST = 192;                 // words a wave collects before it ranks them

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

template <int STEP> __device__ __forceinline__ u64 dpp_u64(u64 x) {
  return (u64)gvd_dpp<STEP>((unsigned)x, 0u) | (u64)gvd_dpp<STEP>((unsigned)(x >> 32), 0u) << 32;
}
template <int STEP> __device__ __forceinline__ u64 max_step(u64 x) {
  const u64 o = dpp_u64<STEP>(x);
  return o > x ? o : x;
}
__device__ __forceinline__ u64 lane63(u64 x) {
  const u64 hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), 63);
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, 63) | hi << 32;
}
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
  v = max_step<0>(v); v = max_step<1>(v); v = max_step<2>(v);
  v = max_step<3>(v); v = max_step<4>(v); v = max_step<5>(v);
  return lane63(v);
}

template <int STEP> __device__ __forceinline__ unsigned max_step(unsigned x) { return max(x, gvd_dpp<STEP>(x, 0u)); }
__device__ __forceinline__ float wave_max_f32(float f) {
  unsigned x = order_bits(f);
  x = max_step<0>(x); x = max_step<1>(x); x = max_step<2>(x);
  x = max_step<3>(x); x = max_step<4>(x); x = max_step<5>(x);
  return from_order_bits((unsigned)__builtin_amdgcn_readlane((int)x, 63));
}
// a value that W lanes or more reach, and next to no more than W: its upper half exactly, bit by bit (0: fewer lanes have any)
__device__ __forceinline__ unsigned wave_bound(unsigned x, int W) {
  unsigned t = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const unsigned c = t | 1u << bit;
    if (__popcll(__ballot(x >= c)) >= W) t = c;
  }
  return t;
}

__device__ __forceinline__ float least_of(u64 floor) {
  const unsigned bits = (unsigned)(floor >> 32);
  return bits > 0x007fffffu ? from_order_bits(bits) : -INFINITY;
}

__device__ __forceinline__ int lanes_below(u64 mask, int lane) { return __popcll(mask & ((1ull << lane) - 1ull)); }

// the best W of the n words on a wave's list, in order, to its front: every word counts those before it
__device__ __forceinline__ void rank_list(u64* list, int n, int W, int lane) {
  u64 k[LIST / 64];
  int r[LIST / 64];
#pragma unroll
  for (int i = 0; i < LIST / 64; ++i) { k[i] = lane + 64 * i < n ? list[lane + 64 * i] : 0; r[i] = 0; }
  if (n <= 64) {
#pragma unroll 8
    for (int j = 0; j < n; ++j) r[0] += list[j] > k[0];
  } else {
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const u64 o = list[j];
#pragma unroll
      for (int i = 0; i < LIST / 64; ++i) r[i] += o > k[i];
    }
  }
  wave_lds_fence();
  if (lane < W) list[lane] = 0;
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < LIST / 64; ++i)
    if (k[i] && r[i] < W) list[r[i]] = k[i];
  wave_lds_fence();
}

// One wave per part of a row: 64 * IPT logits at a time, the next ones on their way meanwhile.  Every lane has a running
// maximum and sum of its own.  A word goes on the list if it beats the W-th best so far (key `floor`); at the start that is a
// value that the maxima of W lanes reach.  The list is ranked, and the floor raised, behind a tile and when it is full; logits
// of any order and equality only make that more frequent.  A wave works by itself, without a barrier.  Bound by the fp64
// exponentials, some 25 full-rate instructions each: 256 rows of 131072 bf16 logits take 52 us (2^x in fp32: 29 us, and the order
// of close beams wrong), 320 rows of 5000 fp32 8.2 us (5.9), 5 rows 4.7 us (4.4).  A series written out here instead of exp()
// is 3 % faster.  A workgroup per part, with barriers and a list of its own, took twice the time of the waves.  Code is kept small
// (a lane finds its next word by selecting, not by 32 copies of the append): at one tile a wave, fetching 50 KB of instructions
// was most of the time.
template <typename T, int IPT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(IPT == 32 && sizeof(T) == 2 ? 4 : 3)))
void beam_part_kernel(const SelectArgs a) {
  constexpr int N = 16 / (int)sizeof(T), VECS = IPT / N, TILE = 64 * IPT;
  typedef typename GvdVec<T, N>::type Vec;
  typedef typename GvdVec<T, N>::loose Loose;
  __shared__ u64 s_list[4][LIST];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int part = blockIdx.x * 4 + wave, row = blockIdx.y;
  if (part >= a.parts) return;
  const float score = a.scores[row];
  const bool over = a.finished ? a.finished[row] != 0 : false;
  const int W = a.W, V = a.V;
  const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ld;
  u64* list = s_list[wave];
  if (lane < W) list[lane] = 0;
  int n = W;                               // words on the list, the best W of before in front
  u64 floor = 0;
  double sum = 0.0;
  float top = -INFINITY;
  const int64_t first = (int64_t)part * a.tiles_per_part * TILE;
  const int64_t end = first + (int64_t)a.tiles_per_part * TILE < V ? first + (int64_t)a.tiles_per_part * TILE : V;
  Vec next[VECS];
  const auto fetch = [&](int64_t v0) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int64_t at = v0 + (i * 64 + lane) * N;
      if (at + N <= V) next[i] = *reinterpret_cast<const Loose*>(x + at);
      else {
#pragma unroll
        for (int k = 0; k < N; ++k) next[i][k] = at + k < V ? x[at + k] : (T)-INFINITY;
      }
    }
  };
  fetch(first);                            // (on its way while the beam's score is)
  if (over || !(fabsf(score) < INFINITY)) return;
  for (int64_t v0 = first; v0 < end; v0 += TILE) {
    float v[IPT];
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < IPT; ++i) { v[i] = (float)next[i / N][i % N]; mx = fmaxf(mx, v[i]); }
    if (v0 + TILE < end) fetch(v0 + TILE);
    // softmax in fp64, as the candidates are compared; nothing but -inf so far: every term is 0
    const float was = top;
    top = fmaxf(top, mx);
    const double ref = top > -INFINITY ? (double)top : 0.0;
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < IPT; ++i) s[i & 1] += exp((double)v[i] - ref);
    sum = sum * exp((double)was - ref) + (s[0] + s[1]);
    // no word under `least` is among the best (bits under those of -inf are no number).  Where W lanes or more have one over it -
    // the first tile, rising logits - what W lanes reach in this tile raises it
    float least = least_of(floor);
    const u64 lanes = __ballot(mx >= least);
    if (!lanes) continue;
    if (__popcll(lanes) >= W) {
      const u64 reached = (u64)wave_bound(order_bits(mx), W) << 32;
      floor = reached > floor ? reached : floor;
      least = least_of(floor);
    }
    unsigned todo = 0;                     // the lane's words at or over it
#pragma unroll
    for (int i = 0; i < IPT; ++i) todo |= v[i] >= least ? 1u << i : 0u;
    while (true) {
      const u64 any = __ballot(todo != 0);
      if (!any || n + __popcll(any) > LIST) {
        wave_lds_fence();
        if (n > W) rank_list(list, n, W, lane);
        n = W;
        floor = list[W - 1] > floor ? list[W - 1] : floor;
        if (!any) break;
      }
      const int i = __ffs(todo) - 1;       // the lane's next one (-1: none)
      float mine = 0.f;
#pragma unroll
      for (int k = 0; k < IPT; ++k) mine = i == k ? v[k] : mine;
      const int64_t at = v0 + ((i / N) * 64 + lane) * N + i % N;
      const u64 key = make_key(order_bits(mine), (int)at);
      const bool hit = todo && key >= floor && at < V;
      const u64 hits = __ballot(hit);
      if (hit) list[n + lanes_below(hits, lane)] = key;
      n += __popcll(hits);
      todo &= todo - 1;
    }
  }
  // the lanes' sums, each to its own maximum, into one (NaN and +inf go through to the join, which drops the beam)
  const float all = wave_max_f32(top);
  sum = gvd_wave_sum_f64(sum != 0.0 ? sum * exp((double)top - (double)all) : 0.0);
  const int64_t rec = (int64_t)row * a.parts + part;
  if (lane == 0) a.stat[rec] = make_double2((double)all, sum);
  if (lane < W) a.best[rec * W + lane] = list[lane];
}

// One workgroup per sample, one wave per beam (and the beams 16 further on): the words of the row's parts at or over the best
// W-th word of a part, and over what the best words of W lanes reach, are put on a list and ranked.  Then all waves do the same
// with the candidates of the beams.  A chain of dependent steps: 5 us for 5 beams, 10 us for 15 samples of 12 beams (23 us when
// every listed word was ranked against every other).
__global__ __launch_bounds__(1024) void beam_join_kernel(const SelectArgs a) {
  __shared__ double s_score[MAX_BEAMS * MAX_WIDTH];
  __shared__ int s_word[MAX_BEAMS * MAX_WIDTH];
  __shared__ u64 s_list[16][JOIN_LIST];
  __shared__ int s_n;
  const int b = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  const int K = a.K, W = a.W, V = a.V;
  if (threadIdx.x == 0) s_n = 0;
  for (int q = wave; q < K; q += waves) {
    const int row = b * K + q;
    double* score_q = s_score + q * W;
    int* word_q = s_word + q * W;
    const float score = a.scores[row];
    const bool over = a.finished ? a.finished[row] != 0 : false;
    // (loaded before they are known to be there: the lists of a beam that was passed over hold anything, and are not used)
    const int64_t rec = (int64_t)row * a.parts;
    const int total = a.parts * W;
    const u64* words = a.best + rec * W;
    const double2 st = lane < a.parts ? a.stat[rec + lane] : make_double2(-INFINITY, 0.0);
    u64 floor = lane < a.parts ? words[lane * W + W - 1] : 0;
    u64 mine[JOIN_LIST / 64];
#pragma unroll
    for (int i = 0; i < JOIN_LIST / 64; ++i) mine[i] = lane + 64 * i < total ? words[lane + 64 * i] : 0;
    bool live = fabsf(score) < INFINITY;
    if (live && over) {
      if (lane < W) {
        const int w = lane == 0 ? a.eos : lane - 1 < a.eos ? lane - 1 : lane;
        score_q[lane] = lane == 0 ? (double)score : -INFINITY;
        word_q[lane] = w < V ? w : -1;
      }
      continue;
    }
    double lse = 0.0;
    if (live) {
      const double m = wave_max_f32((float)st.x);
      lse = m + log(gvd_wave_sum_f64(lane < a.parts && st.y != 0.0 ? st.y * exp(st.x - m) : 0.0));
      live = fabs(lse) < INFINITY;
    }
    if (!live) {
      if (lane < W) {
        score_q[lane] = -INFINITY;
        word_q[lane] = lane < V ? lane : -1;
      }
      continue;
    }
    u64 most = mine[0];
#pragma unroll
    for (int i = 1; i < JOIN_LIST / 64; ++i) most = mine[i] > most ? mine[i] : most;
    const u64 reached = (u64)wave_bound((unsigned)(most >> 32), W) << 32;          // (by the best words of W lanes)
    floor = wave_max_u64(floor);
    floor = reached > floor ? reached : floor;
    u64* list = s_list[wave];
    int n = 0;
#pragma unroll
    for (int i = 0; i < JOIN_LIST / 64; ++i) {
      if (64 * i >= total) break;
      const bool keep = mine[i] && mine[i] >= floor;
      const u64 hits = __ballot(keep);
      if (keep) list[n + lanes_below(hits, lane)] = mine[i];
      n += __popcll(hits);
    }
    if (lane < W) { score_q[lane] = -INFINITY; word_q[lane] = -1; }
    wave_lds_fence();
    for (int i = lane; i < n; i += 64) {
      const u64 k = list[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) r += list[j] > k;
      if (r < W) {
        score_q[r] = (double)score + ((double)from_order_bits((unsigned)(k >> 32)) - lse);
        word_q[r] = key_word(k);
      }
    }
    wave_lds_fence();
  }
  __syncthreads();
  // candidates by (score descending, place in the lists ascending): a beam's list is in order already, and beams go up
  double floor = -INFINITY;
  for (int q = 0; q < K; ++q)
    if (s_word[q * W + W - 1] >= 0) floor = fmax(floor, s_score[q * W + W - 1]);
  double* kept_score = reinterpret_cast<double*>(&s_list[0][0]);
  int* kept = reinterpret_cast<int*>(kept_score + MAX_BEAMS * MAX_WIDTH);
  for (int e = threadIdx.x; e < K * W; e += blockDim.x)
    if (s_word[e] >= 0 && s_score[e] >= floor) {
      const int at = atomicAdd(&s_n, 1);
      kept[at] = e;
      kept_score[at] = s_score[e];
    }
  __syncthreads();
  const int n = s_n;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int e = kept[i];
    const double sc = kept_score[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += kept_score[j] > sc || (kept_score[j] == sc && kept[j] < e);
    if (r < W) {
      const int64_t to = (int64_t)b * W + r;
      const int q = e / W, w = s_word[e];
      a.out_scores[to] = (float)sc;
      a.parent[to] = (int64_t)b * K + q;
      a.word[to] = w;
      if (a.out_finished) a.out_finished[to] = w == a.eos || (a.finished && a.finished[b * K + q]);
    }
  }
}

// logits of one lane and tile, parts (waves) of a row, tiles of a part
struct SelectShape { int ipt, parts, tiles_per_part; };

SelectShape select_shape(int64_t rows, int V, int W, int dtype) {
  // parts that fill the device (16 waves a CU), and the tile that a wave gets through its part with soonest: a tile of i logits a
  // lane costs some 24 + i (its bound and its ranking as much as 24 logits).  Both launches, with events: 15 x 12 beams, 32003 words
  // fp16: one tile of 32 a wave 30 us, two of 16 31.5, three of 8 35; 64 x 5 beams, 5000 words fp32: one of 8 19.2 us, of 16 20, two
  // of 4 20.4.
  const int least = dtype == GVD_F32 ? 4 : 8;
  int64_t most = MAX_PARTS < JOIN_LIST / W ? MAX_PARTS : JOIN_LIST / W;
  if (most > 4096 / rows) most = 4096 / rows > 1 ? 4096 / rows : 1;
  SelectShape s = {0, 0, 0};
  int64_t cost = 0;
  for (int ipt = 32; ipt >= least; ipt /= 2) {
    if (ipt > least && 32 * ipt >= V) continue;              // (half of the tile would do)
    const int tiles = (V + 64 * ipt - 1) / (64 * ipt), per_part = (int)((tiles + most - 1) / most);
    if (s.ipt && (int64_t)per_part * (24 + ipt) >= cost) continue;
    cost = (int64_t)per_part * (24 + ipt);
    s = {ipt, (tiles + per_part - 1) / per_part, per_part};
  }
  return s;
}

template <typename T> void launch_parts(const SelectArgs& a, int ipt, hipStream_t st) {
  const dim3 grid((unsigned)((a.parts + 3) / 4), (unsigned)(a.B * a.K));
  if (ipt == 32) hipLaunchKernelGGL((beam_part_kernel<T, 32>), grid, dim3(256), 0, st, a);
  else if (ipt == 16) hipLaunchKernelGGL((beam_part_kernel<T, 16>), grid, dim3(256), 0, st, a);
  else if (ipt == 8 || sizeof(T) == 2) hipLaunchKernelGGL((beam_part_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((beam_part_kernel<T, 4>), grid, dim3(256), 0, st, a);
}

bool bad_select_shape(int B, int K, int V, int W) {
  return B <= 0 || K <= 0 || K > MAX_BEAMS || V <= 0 || W <= 0 || W > MAX_WIDTH || (int64_t)K * V < W || (int64_t)B * K > 65535 ||
         V > (1 << 28);
}

// ------------------------------------------------------------------------------------------------------------- reorder
// dst[o, r, :] = src[o, index[r], :], up to GVD_REORDER_MAX_TENSORS tensors in a launch.  A copy: bound by reading and writing
// the rows once (2 caches of 256 x 1 MB: 129 us, 8.3 TB/s of rows read and written: parents repeat, and come from the cache).
// A thread copies four units of 16 bytes; the last unit of a row is moved back so that it ends with the row (rows under 16
// bytes: units of 8, 4 or 1 bytes).
constexpr int UNITS = 1024;               // units of one workgroup

template <int BYTES> struct Unit;
template <> struct Unit<16> { typedef unsigned type __attribute__((ext_vector_type(4), aligned(1))); };
template <> struct Unit<8> { typedef unsigned type __attribute__((ext_vector_type(2), aligned(1))); };
template <> struct Unit<4> { typedef unsigned type __attribute__((aligned(1))); };
template <> struct Unit<1> { typedef uint8_t type; };

template <int BYTES>
__device__ void reorder_tile(const gvd_reorder_tensor& t, const int64_t* __restrict__ index, int64_t rows_in, int64_t rows_out,
                             int64_t tile) {
  typedef typename Unit<BYTES>::type U;
  const int64_t per_row = (t.row_bytes + BYTES - 1) / BYTES;
  const char* src[4];
  char* dst[4];
  const auto place = [&](int u, int64_t o, int64_t r, int64_t unit) {
    int64_t off = unit * BYTES;
    if (off + BYTES > t.row_bytes) off = t.row_bytes - BYTES;
    const int64_t from = index[r];
    dst[u] = reinterpret_cast<char*>(t.dst) + o * t.dst_outer + r * t.dst_row + off;
    src[u] = from >= 0 && from < rows_in ? reinterpret_cast<const char*>(t.src) + o * t.src_outer + from * t.src_row + off : nullptr;
  };
  if (per_row >= UNITS) {                 // a tile lies in one row (the host counts tiles the same way)
    const unsigned tiles = (unsigned)((per_row + UNITS - 1) / UNITS), row = (unsigned)tile / tiles, o = row / (unsigned)rows_out;
    const int64_t unit0 = (int64_t)((unsigned)tile - row * tiles) * UNITS + threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      dst[u] = nullptr; src[u] = nullptr;
      if (unit0 + 256 * u < per_row) place(u, o, row - o * (unsigned)rows_out, unit0 + 256 * u);
    }
  } else {                                // (fewer than 2^31 units: 32-bit divisions)
    const unsigned total = (unsigned)(t.outer * rows_out * per_row), pr = (unsigned)per_row, ro = (unsigned)rows_out;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const unsigned i = (unsigned)tile * UNITS + u * 256 + threadIdx.x;
      dst[u] = nullptr; src[u] = nullptr;
      if (i < total) {
        const unsigned row = i / pr, o = row / ro;
        place(u, o, row - o * ro, i - row * pr);
      }
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
    if (dst[u]) *reinterpret_cast<U*>(dst[u]) = x[u];
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
    default: reorder_tile<1>(x, index, rows_in, rows_out, tile); break;
  }
}

}  // namespace

extern "C" size_t gvd_beam_select_workspace_bytes(int B, int K, int V, int W) {
  if (bad_select_shape(B, K, V, W)) return 0;
  const int64_t rows = (int64_t)B * K;
  int64_t most = 0;                        // (of the two shapes: the type is not among the arguments)
  for (int dtype : {GVD_F32, GVD_BF16}) {
    const int64_t parts = select_shape(rows, V, W, dtype).parts;
    most = parts > most ? parts : most;
  }
  return (size_t)(rows * most * (16 + 8 * (int64_t)W));
}

extern "C" int gvd_beam_select(const gvd_beam_select_args* g, gvd_stream_t stream) {
  if (!g || bad_select_shape(g->B, g->K, g->V, g->W) || !gvd_dtype_bytes(g->dtype) || !g->logits || g->ld < g->V || !g->scores ||
      !g->out_scores || !g->parent || !g->word || !g->workspace || !gvd_aligned16(g->workspace) || g->eos < -1 || g->eos >= g->V ||
      (g->finished && g->eos < 0) || g->workspace_bytes < gvd_beam_select_workspace_bytes(g->B, g->K, g->V, g->W))
    return GVD_EINVAL;
  const int64_t rows = (int64_t)g->B * g->K;
  const SelectShape s = select_shape(rows, g->V, g->W, g->dtype);
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
    t.unit = t.row_bytes >= 16 ? 16 : t.row_bytes % 8 == 0 ? 8 : t.row_bytes % 4 == 0 ? 4 : 1;
    g.tile0[i] = tiles;
    const int64_t per_row = (t.row_bytes + t.unit - 1) / t.unit;
    if (t.outer > (1ll << 33) / rows_out || per_row > (1ll << 33) / (t.outer * rows_out)) return GVD_EINVAL;
    if (per_row >= UNITS) tiles += t.outer * rows_out * ((per_row + UNITS - 1) / UNITS);
    else if (t.outer * rows_out * per_row >= 0x7fffffffll) return GVD_EINVAL;
    else tiles += (t.outer * rows_out * per_row + UNITS - 1) / UNITS;
  }
  g.tile0[g.count] = tiles;
  if (tiles > (1ll << 23)) return GVD_EINVAL;                   // (a launch holds fewer than 2^32 threads)
  hipLaunchKernelGGL(reorder_rows_kernel, dim3((unsigned)tiles), dim3(256), 0, gvd_s(stream), g, index, rows_in, rows_out);
  GVD_CHECK_LAUNCH();
  return 0;
}
