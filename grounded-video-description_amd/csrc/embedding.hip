// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward    out[n,:] = act(scale * W[tok[n],:])
//   backward   dW[v,:]  = scale * act'(scale * W[v,:]) * sum over n with tok[n] = v, n ascending, of dy[n,:]
//
// (act' depends on the table row alone, so it multiplies the finished sum once.)  Both directions are bound by the rows they
// move: out / dy once, the table's rows once.  The backward never adds with atomics: the positions are sorted by token (stable),
// every row of dW is summed by one owner in a fixed order and written once, rows without a token as zeros.  Sums are fp32.
#include "dtypes.h"

namespace {

__device__ __forceinline__ float act_relu(float x) { return x > 0.f ? x : (x == x ? 0.f : x); }      // (NaN stays NaN)

// token n as a key in [0, vocab]; vocab = "no row": out of range, or the padding row in the backward
__device__ __forceinline__ unsigned token_key(const void* tok, int tok64, int64_t n, unsigned vocab, int64_t pad) {
  const int64_t t = tok64 ? reinterpret_cast<const int64_t*>(tok)[n] : (int64_t)reinterpret_cast<const int*>(tok)[n];
  return t < 0 || t >= (int64_t)vocab || t == pad ? vocab : (unsigned)t;
}

// ------------------------------------------------------------------------------------------------------------- forward
// One wave per row and 64 * N columns.
template <typename T, int N>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* tok, int tok64, int64_t n, const T* __restrict__ table,
                                                            int64_t ld, unsigned vocab, int width, float scale, int act,
                                                            T* __restrict__ out, int64_t ldo) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= n) return;
  const int col = (blockIdx.y * 64 + (threadIdx.x & 63)) * N;
  if (col >= width) return;
  const unsigned v = token_key(tok, tok64, row, vocab, -1);
  const int left = width - col;
  float x[N];
  if (v == vocab) {                       // a token outside the table: nothing is read, the row is NaN
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = __builtin_nanf("");
  } else {
    const T* w = table + (int64_t)v * ld + col;
    if (left >= N) gvd_load<T, N>(w, x); else gvd_load_part<T, N>(w, left, x);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      x[k] *= scale;
      if (act) x[k] = act_relu(x[k]);
    }
  }
  T* o = out + row * ldo + col;
  if (left >= N) gvd_store<T, N>(o, x); else gvd_store_part<T, N>(o, left, x);
}

// ------------------------------------------------------------------------------------------- positions sorted by token
// n <= RANK_MAX: the place of position i is the number of positions that go before it, counted directly: keys smaller, or
// equal and earlier.  n^2 comparisons (2 instructions each) spread over n / 64 workgroups of 16 waves.
constexpr int RANK_MAX = 8192;
constexpr int RANK_THREADS = 1024;

__global__ __launch_bounds__(RANK_THREADS) void token_rank_kernel(const void* tok, int tok64, int n, unsigned vocab, int64_t pad,
                                                                  unsigned* __restrict__ skey, unsigned* __restrict__ spos) {
  __shared__ unsigned s_key[RANK_MAX];
  __shared__ int s_cnt[16][64];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int i = tid; i < n; i += RANK_THREADS) s_key[i] = token_key(tok, tok64, i, vocab, pad);
  __syncthreads();
  const int i = blockIdx.x * 64 + lane;
  const unsigned key = i < n ? s_key[i] : 0;
  int c = 0;
  for (int j = wave; j < n; j += 16) c += s_key[j] < key || (s_key[j] == key && j < i);
  s_cnt[wave][lane] = c;
  __syncthreads();
  if (wave == 0 && i < n) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) place += s_cnt[w][lane];
    skey[place] = key;
    spos[place] = (unsigned)i;
  }
}

// Larger n: stable counting sorts by digits of up to 9 bits, least significant first.  The positions are cut into at most
// SORT_BLOCKS contiguous parts, one workgroup each: a launch counts every part's digits, the next one places them - each
// workgroup adds up the counts before its own by itself.  A wave takes 64 consecutive positions at a time; lanes of equal digit
// find each other by ballots, so equal digits keep their order.
constexpr int SORT_BLOCKS = 128;
constexpr int SORT_BITS = 9;
constexpr int SORT_DIGITS = 1 << SORT_BITS;
constexpr int SORT_TILE = 2048;

struct SortPass {
  const void* tok; int tok64; unsigned vocab; int64_t pad;       // first pass: keys from the tokens, positions 0, 1, ...
  const unsigned* key_in; const unsigned* pos_in;                // later passes
  unsigned* key_out; unsigned* pos_out;
  unsigned* hist;                                                // [blocks][SORT_DIGITS]
  int64_t n, per;                                                // positions; positions of one workgroup
  int shift, bits;
};

// LDS accesses of the lanes of one wave before it happen before those after it
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ unsigned sort_key(const SortPass& p, int64_t i) {
  return p.tok ? token_key(p.tok, p.tok64, i, p.vocab, p.pad) : p.key_in[i];
}

__global__ __launch_bounds__(256) void sort_count_kernel(const SortPass p) {
  __shared__ unsigned s_hist[SORT_DIGITS];
  for (int d = threadIdx.x; d < SORT_DIGITS; d += 256) s_hist[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * p.per, i1 = i0 + p.per < p.n ? i0 + p.per : p.n;
  const unsigned mask = (1u << p.bits) - 1;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += 256) atomicAdd(&s_hist[(sort_key(p, i) >> p.shift) & mask], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < SORT_DIGITS; d += 256) p.hist[(int64_t)blockIdx.x * SORT_DIGITS + d] = s_hist[d];
}

__global__ __launch_bounds__(256) void sort_place_kernel(const SortPass p) {
  __shared__ unsigned s_next[SORT_DIGITS];                   // where the next position of this digit goes
  __shared__ unsigned s_wave[4][SORT_DIGITS];
  __shared__ unsigned s_sum[256];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const unsigned mask = (1u << p.bits) - 1;
  // digits 2 tid, 2 tid + 1: their counts before this part, and in all
  unsigned before[2] = {0, 0}, all[2] = {0, 0};
  for (unsigned b = 0; b < gridDim.x; ++b) {
    const uint2 h = *reinterpret_cast<const uint2*>(p.hist + (int64_t)b * SORT_DIGITS + 2 * tid);
    all[0] += h.x; all[1] += h.y;
    if (b < blockIdx.x) { before[0] += h.x; before[1] += h.y; }
  }
  s_sum[tid] = all[0] + all[1];
  __syncthreads();
  for (int off = 1; off < 256; off <<= 1) {
    const unsigned add = tid >= off ? s_sum[tid - off] : 0;
    __syncthreads();
    s_sum[tid] += add;
    __syncthreads();
  }
  const unsigned base = s_sum[tid] - (all[0] + all[1]);
  s_next[2 * tid] = base + before[0];
  s_next[2 * tid + 1] = base + all[0] + before[1];
  const int64_t i0 = (int64_t)blockIdx.x * p.per, i1 = i0 + p.per < p.n ? i0 + p.per : p.n;
  constexpr int ROUNDS = SORT_TILE / 256;
  for (int64_t t0 = i0; t0 < i1; t0 += SORT_TILE) {
    for (int d = tid; d < 4 * SORT_DIGITS; d += 256) (&s_wave[0][0])[d] = 0;
    __syncthreads();
    unsigned key[ROUNDS], place[ROUNDS];
    const int64_t w0 = t0 + wave * (SORT_TILE / 4) + lane;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) key[r] = w0 + 64 * r < i1 ? sort_key(p, w0 + 64 * r) : 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const bool in = w0 + 64 * r < i1;
      const unsigned d = (key[r] >> p.shift) & mask;
      unsigned long long same = __ballot(in);
      for (int b = 0; b < p.bits; ++b) {
        const unsigned long long set = __ballot((d >> b) & 1u);
        same &= (d >> b) & 1u ? set : ~set;
      }
      const unsigned seen = in ? s_wave[wave][d] : 0;
      const int rank = __popcll(same & ((1ull << lane) - 1ull));
      place[r] = seen + rank;
      wave_lds_fence();
      if (in && rank == 0) s_wave[wave][d] = seen + (unsigned)__popcll(same);
      wave_lds_fence();
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int64_t i = w0 + 64 * r;
      if (i < i1) {
        const unsigned d = (key[r] >> p.shift) & mask;
        unsigned to = s_next[d] + place[r];
        for (int w = 0; w < wave; ++w) to += s_wave[w][d];
        p.key_out[to] = key[r];
        p.pos_out[to] = p.tok ? (unsigned)i : p.pos_in[i];
      }
    }
    __syncthreads();
    for (int d = tid; d < SORT_DIGITS; d += 256) s_next[d] += s_wave[0][d] + s_wave[1][d] + s_wave[2][d] + s_wave[3][d];
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------------- sums by token
// A token that fills whole groups of GROUP sorted positions (64; and 64 of those groups) has them summed beforehand, one
// workgroup per group, so that no owner of a row adds up more than a few hundred rows whatever the tokens are.
constexpr int GROUP = 64;

struct SumArgs {
  const unsigned* skey; const unsigned* spos; int64_t n;
  const void* dy; int64_t ld;
  float* part1; float* part2;             // fp32 [n / 64][width], [n / 4096][width]
  const void* table; int64_t ldt;         // for act'
  void* dw;
  unsigned vocab; int width; float scale; int act;
};

template <typename T, int N> __device__ __forceinline__ void add_row(const T* p, int left, float (&s)[N]) {
  float x[N];
  if (left >= N) gvd_load<T, N>(p, x); else gvd_load_part<T, N>(p, left, x);
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] += x[k];
}

// s += dy rows of sorted positions [i, e), in order
template <typename T, int N> __device__ __forceinline__ void add_rows(const SumArgs& a, int64_t i, int64_t e, int col, float (&s)[N]) {
  const T* dy = reinterpret_cast<const T*>(a.dy) + col;
  const int left = a.width - col;
  for (; i < e; ++i) add_row<T, N>(dy + (int64_t)a.spos[i] * a.ld, left, s);
}

// level 1: groups of 64 positions of one token; level 2: groups of 64 such groups
template <typename T, int N, int LEVEL>
__global__ __launch_bounds__(256) void token_group_kernel(const SumArgs a) {
  const int64_t g = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  constexpr int64_t LEN = LEVEL == 1 ? GROUP : GROUP * GROUP;
  if ((g + 1) * LEN > a.n) return;
  const unsigned v = a.skey[g * LEN];
  if (v >= a.vocab || a.skey[g * LEN + LEN - 1] != v) return;
  const int col = (blockIdx.y * 64 + (threadIdx.x & 63)) * N;
  if (col >= a.width) return;
  const int left = a.width - col;
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
  if constexpr (LEVEL == 1) {
    add_rows<T, N>(a, g * LEN, (g + 1) * LEN, col, s);
  } else {
    for (int64_t c = g * GROUP; c < (g + 1) * GROUP; ++c) add_row<float, N>(a.part1 + c * a.width + col, left, s);
  }
  float* o = (LEVEL == 1 ? a.part1 : a.part2) + g * a.width + col;
  if (left >= N) gvd_store<float, N>(o, s); else gvd_store_part<float, N>(o, left, s);
}

// first sorted position whose key is >= v: 64 lanes look at 64 places at a time
__device__ __forceinline__ int64_t wave_lower_bound(const unsigned* skey, int64_t n, unsigned v, int lane) {
  int64_t lo = 0, len = n;                       // the answer is in [lo, lo + len]
  while (len > 0) {
    const int64_t step = (len + 63) >> 6;
    const int64_t at = lo + (int64_t)lane * step;
    const bool less = at < lo + len && skey[at] < v;
    const int c = __popcll(__ballot(less));      // (sorted: the first c lanes)
    if (c == 0) return lo;
    const int64_t from = lo + (int64_t)(c - 1) * step + 1;
    const int64_t to = c < 64 && lo + (int64_t)c * step < lo + len ? lo + (int64_t)c * step : lo + len;
    lo = from;
    len = to - from;
  }
  return lo;
}

// one wave per row of the table and 64 * N columns
template <typename T, int N>
__global__ __launch_bounds__(256) void token_rows_kernel(const SumArgs a) {
  const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v >= (int64_t)a.vocab) return;
  const int lane = threadIdx.x & 63;
  const int64_t b = wave_lower_bound(a.skey, a.n, (unsigned)v, lane);
  const int64_t e = b + wave_lower_bound(a.skey + b, a.n - b, (unsigned)v + 1, lane);
  const int col = (blockIdx.y * 64 + lane) * N;
  if (col >= a.width) return;
  const int left = a.width - col;
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
  const int64_t g1 = (b + GROUP - 1) / GROUP, g2 = e / GROUP;               // whole groups [g1, g2)
  if (e > b) {
    if (g1 >= g2) {
      add_rows<T, N>(a, b, e, col, s);
    } else {
      add_rows<T, N>(a, b, g1 * GROUP, col, s);
      const int64_t h1 = (g1 + GROUP - 1) / GROUP, h2 = g2 / GROUP;         // whole groups of groups
      const int64_t c1 = h1 < h2 ? h1 * GROUP : g2, c2 = h1 < h2 ? h2 * GROUP : g2;
      for (int64_t c = g1; c < c1; ++c) add_row<float, N>(a.part1 + c * a.width + col, left, s);
      for (int64_t c = h1; c < h2; ++c) add_row<float, N>(a.part2 + c * a.width + col, left, s);
      for (int64_t c = c2; c < g2; ++c) add_row<float, N>(a.part1 + c * a.width + col, left, s);
      add_rows<T, N>(a, g2 * GROUP, e, col, s);
    }
    if (a.act) {
      float w[N];
      const T* t = reinterpret_cast<const T*>(a.table) + v * a.ldt + col;
      if (left >= N) gvd_load<T, N>(t, w); else gvd_load_part<T, N>(t, left, w);
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] = w[k] * a.scale > 0.f ? s[k] * a.scale : 0.f;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) s[k] *= a.scale;
    }
  }
  T* o = reinterpret_cast<T*>(a.dw) + v * (int64_t)a.width + col;
  if (left >= N) gvd_store<T, N>(o, s); else gvd_store_part<T, N>(o, left, s);
}

// ---------------------------------------------------------------------------------------------------------------- host
// columns of one lane: 16 bytes where the width fills a wave with them, else the smallest power of two that covers the width
int lane_columns(int width, int dtype) {
  const int most = dtype == GVD_F32 ? 4 : 8;
  int n = 1;
  while (n < most && 64 * n < width) n *= 2;
  return n;
}

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

struct BwdSpace {
  int64_t skey, spos, key2, pos2, hist, part1, part2, bytes;
  bool rank;
  int passes, bits, blocks;
  int64_t per;
};

BwdSpace bwd_space(int64_t n, int64_t vocab, int width) {
  BwdSpace s = {};
  s.rank = n <= RANK_MAX;
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;                  // keys 0 ... vocab
  s.passes = (bits + SORT_BITS - 1) / SORT_BITS;
  s.bits = (bits + s.passes - 1) / s.passes;
  const int64_t tiles = (n + SORT_TILE - 1) / SORT_TILE;
  s.per = (tiles + SORT_BLOCKS - 1) / SORT_BLOCKS * SORT_TILE;
  s.blocks = (int)((n + s.per - 1) / s.per);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) { const int64_t o = at; at += align256(bytes); return o; };
  s.skey = take(4 * n);
  s.spos = take(4 * n);
  if (!s.rank) {
    s.key2 = take(4 * n);
    s.pos2 = take(4 * n);
    s.hist = take((int64_t)s.blocks * SORT_DIGITS * 4);
  }
  s.part1 = take(n / GROUP * width * 4);
  s.part2 = take(n / (GROUP * GROUP) * width * 4);
  s.bytes = at;
  return s;
}

bool bad_shape(int64_t n, int64_t vocab, int width, int dtype) {
  return n <= 0 || n > GVD_EMBEDDING_MAX || vocab <= 0 || vocab > GVD_EMBEDDING_MAX || width <= 0 || width > (1 << 20) ||
         !gvd_dtype_bytes(dtype);
}

template <typename T, int N>
int launch_fwd(const void* tok, int tok64, int64_t n, const void* table, int64_t ld, int64_t vocab, int width, float scale,
               int act, void* out, int64_t ldo, hipStream_t st) {
  const dim3 grid((unsigned)((n + 3) / 4), (unsigned)((width + 64 * N - 1) / (64 * N)));
  hipLaunchKernelGGL((embedding_fwd_kernel<T, N>), grid, dim3(256), 0, st, tok, tok64, n, reinterpret_cast<const T*>(table), ld,
                     (unsigned)vocab, width, scale, act, reinterpret_cast<T*>(out), ldo);
  GVD_CHECK_LAUNCH();
  return 0;
}

template <typename T, int N> int launch_sums(const SumArgs& a, hipStream_t st) {
  const unsigned slices = (unsigned)((a.width + 64 * N - 1) / (64 * N));
  const int64_t g1 = a.n / GROUP, g2 = a.n / (GROUP * GROUP);
  if (g1) {
    hipLaunchKernelGGL((token_group_kernel<T, N, 1>), dim3((unsigned)((g1 + 3) / 4), slices), dim3(256), 0, st, a);
    GVD_CHECK_LAUNCH();
  }
  if (g2) {
    hipLaunchKernelGGL((token_group_kernel<T, N, 2>), dim3((unsigned)((g2 + 3) / 4), slices), dim3(256), 0, st, a);
    GVD_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL((token_rows_kernel<T, N>), dim3((unsigned)((a.vocab + 3) / 4), slices), dim3(256), 0, st, a);
  GVD_CHECK_LAUNCH();
  return 0;
}

#define GVD_BY_TYPE(CALL)                                                       \
  const int cols = lane_columns(width, dtype);                                  \
  if (dtype == GVD_F32) {                                                       \
    if (cols == 4) return CALL(float, 4);                                       \
    if (cols == 2) return CALL(float, 2);                                       \
    return CALL(float, 1);                                                      \
  }                                                                             \
  if (dtype == GVD_BF16) {                                                      \
    if (cols == 8) return CALL(gvd_bf16, 8);                                    \
    if (cols == 4) return CALL(gvd_bf16, 4);                                    \
    if (cols == 2) return CALL(gvd_bf16, 2);                                    \
    return CALL(gvd_bf16, 1);                                                   \
  }                                                                             \
  if (cols == 8) return CALL(gvd_f16, 8);                                       \
  if (cols == 4) return CALL(gvd_f16, 4);                                       \
  if (cols == 2) return CALL(gvd_f16, 2);                                       \
  return CALL(gvd_f16, 1);

}  // namespace

extern "C" int gvd_embedding_fwd(const void* tokens, int tok64, int64_t n, const void* table, int64_t ld, int64_t vocab, int width,
                                 int dtype, float scale, int act, void* out, int64_t ldo, gvd_stream_t stream) {
  if (!tokens || !table || !out || bad_shape(n, vocab, width, dtype) || ld < width || ldo < width) return GVD_EINVAL;
  const hipStream_t st = gvd_s(stream);
#define GVD_FWD(T, N) launch_fwd<T, N>(tokens, tok64, n, table, ld, vocab, width, scale, act, out, ldo, st)
  GVD_BY_TYPE(GVD_FWD)
#undef GVD_FWD
}

extern "C" size_t gvd_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int width) {
  if (bad_shape(n, vocab, width, GVD_F32)) return 0;
  return (size_t)bwd_space(n, vocab, width).bytes;
}

extern "C" int gvd_embedding_bwd(const void* tokens, int tok64, int64_t n, const void* dy, int64_t ld_dy, const void* table, int64_t ld,
                                 int64_t vocab, int width, int dtype, float scale, int act, int64_t padding_idx, void* dw,
                                 void* workspace, size_t workspace_bytes, gvd_stream_t stream) {
  if (!tokens || !dy || !dw || !workspace || bad_shape(n, vocab, width, dtype) || ld_dy < 0 || (act && (!table || ld < width)))
    return GVD_EINVAL;
  const BwdSpace s = bwd_space(n, vocab, width);
  if (workspace_bytes < (size_t)s.bytes || !gvd_aligned16(workspace)) return GVD_EINVAL;
  const hipStream_t st = gvd_s(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  const auto at = [&](int64_t o) { return reinterpret_cast<unsigned*>(ws + o); };
  const int64_t pad = padding_idx < 0 ? -1 : padding_idx;
  if (s.rank) {
    hipLaunchKernelGGL(token_rank_kernel, dim3((unsigned)((n + 63) / 64)), dim3(RANK_THREADS), 0, st, tokens, tok64, (int)n,
                       (unsigned)vocab, pad, at(s.skey), at(s.spos));
    GVD_CHECK_LAUNCH();
  } else {
    for (int i = 0; i < s.passes; ++i) {
      const bool to_first = ((s.passes - 1 - i) & 1) == 0;              // the last pass writes skey / spos
      SortPass p = {};
      if (i == 0) { p.tok = tokens; p.tok64 = tok64; p.vocab = (unsigned)vocab; p.pad = pad; }
      p.key_in = at(to_first ? s.key2 : s.skey); p.pos_in = at(to_first ? s.pos2 : s.spos);
      p.key_out = at(to_first ? s.skey : s.key2); p.pos_out = at(to_first ? s.spos : s.pos2);
      p.hist = at(s.hist);
      p.n = n; p.per = s.per;
      p.shift = i * s.bits; p.bits = s.bits;
      hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)s.blocks), dim3(256), 0, st, p);
      GVD_CHECK_LAUNCH();
      hipLaunchKernelGGL(sort_place_kernel, dim3((unsigned)s.blocks), dim3(256), 0, st, p);
      GVD_CHECK_LAUNCH();
    }
  }
  SumArgs a = {};
  a.skey = at(s.skey); a.spos = at(s.spos); a.n = n;
  a.dy = dy; a.ld = ld_dy;
  a.part1 = reinterpret_cast<float*>(ws + s.part1); a.part2 = reinterpret_cast<float*>(ws + s.part2);
  a.table = table; a.ldt = ld;
  a.dw = dw;
  a.vocab = (unsigned)vocab; a.width = width; a.scale = scale; a.act = act;
#define GVD_SUMS(T, N) launch_sums<T, N>(a, st)
  GVD_BY_TYPE(GVD_SUMS)
#undef GVD_SUMS
}
