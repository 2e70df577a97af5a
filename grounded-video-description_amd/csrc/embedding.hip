// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward    out[n,:] = act(scale * W[tok[n],:])
//   backward   dW[v,:]  = scale * act'(scale * W[v,:]) * sum over n with tok[n] = v of dy[n,:]
//
// (act' depends on the table row alone, so it multiplies the finished sum once.)  Both directions are bound by the rows they
// move: out / dy once, the table's rows once.  The backward never adds with atomics: the positions are sorted by token (stable;
// few, of a small table, are listed by token instead), every row of dW is summed by one owner in a fixed order and written once,
// rows without a token as zeros.  The order is that of the positions, but for frequent words, whose groups of positions are
// summed first (64 positions or more; in the form for few tokens more than 128): it depends on n and the table's size, not
// on the run.  Sums are fp32.
#include "dtypes.h"

namespace {

__device__ __forceinline__ float act_relu(float x) { return x > 0.f ? x : (x == x ? 0.f : x); }      // (NaN stays NaN)

// token n as a key in [0, vocab]; vocab = "no row": out of range, or the padding row in the backward
__device__ __forceinline__ unsigned token_key(const void* tok, int tok64, int64_t n, unsigned vocab, int64_t pad) {
  const int64_t t = tok64 ? reinterpret_cast<const int64_t*>(tok)[n] : (int64_t)reinterpret_cast<const int*>(tok)[n];
  return t < 0 || t >= (int64_t)vocab || t == pad ? vocab : (unsigned)t;
}

__device__ __forceinline__ unsigned wave_id() {
  return __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));          // (workgroups of four waves)
}

// A lane's first column in slice `slice` of 64 * N columns; -1: none.  The last lane of a row is moved back so that it ends
// with the row: it does some of its neighbour's columns again, the same sums in the same order, instead of a part of a vector
// (host: the width is N at least).
template <int N> __device__ __forceinline__ int lane_column(unsigned slice, int width) {
  const int col = (int)(slice * 64 + (threadIdx.x & 63)) * N;
  return col >= width ? -1 : col <= width - N ? col : width - N;
}

// ------------------------------------------------------------------------------------------------------------- forward
// One wave per R rows and 64 * N columns (a slice); the R tokens, then the R rows, are on their way together.  Waves next to
// each other take the slices of the same rows, so that a row is one stretch of memory traffic.  Bound by the rows: 131072 x
// 2048 bf16 take 121 us (5.5 TB/s of rows read once and written) with stores past the cache, 146 us without; R = 2 and 8 take
// 132. One decode step (5 x 512 fp32): 1.8 us, the launch.
template <typename T, int N, int R, bool PAST>
__global__ __launch_bounds__(256) void embedding_fwd_kernel(const void* tok, int tok64, int64_t n, const T* __restrict__ table,
                                                            int64_t ld, unsigned vocab, int width, float scale, int act,
                                                            T* __restrict__ out, int64_t ldo, unsigned slices) {
  const unsigned id = wave_id(), unit = id / slices;
  const int64_t row0 = (int64_t)unit * R;
  const int col = lane_column<N>(id - unit * slices, width);
  if (row0 >= n || col < 0) return;
  unsigned v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = row0 + r < n ? token_key(tok, tok64, row0 + r, vocab, -1) : vocab;
  float x[R][N];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (v[r] == vocab) {                  // a token outside the table: nothing is read, the row is NaN
#pragma unroll
      for (int k = 0; k < N; ++k) x[r][k] = __builtin_nanf("");
    } else {
      gvd_load<T, N>(table + (int64_t)v[r] * ld + col, x[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (row0 + r >= n) break;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      x[r][k] *= scale;
      if (act) x[r][k] = act_relu(x[r][k]);
    }
    T* o = out + (row0 + r) * ldo + col;
    if constexpr (PAST) gvd_store_past<T, N>(o, x[r]);
    else gvd_store<T, N>(o, x[r]);
  }
}

// ------------------------------------------------------------------------------------------- positions sorted by token
// n <= RANK_MAX: the place of position i is the number of positions that go before it, counted directly: keys smaller, or
// equal and earlier.  n^2 comparisons (2 instructions each) spread over n / 64 workgroups of 16 waves.  The whole backward with
// it and with the counting sort, us with events: 8192 words, 5000 x 512 fp32, 38 and 44.5; 16384, 50000 x 512 bf16, 57 and 53.
constexpr int RANK_MAX = 8192;
constexpr int RANK_THREADS = 1024;

__global__ __launch_bounds__(RANK_THREADS) void token_rank_kernel(const void* tok, int tok64, int n, unsigned vocab, int64_t pad,
                                                                  unsigned* __restrict__ skey, unsigned* __restrict__ spos) {
  __shared__ __attribute__((aligned(16))) unsigned s_key[RANK_MAX];
  __shared__ int s_cnt[16][64];
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int blocks = (n + 63) >> 6;                            // blocks of 64 keys
  for (int i = tid; i < 64 * blocks; i += RANK_THREADS) s_key[i] = i < n ? token_key(tok, tok64, i, vocab, pad) : 0xffffffffu;
  __syncthreads();
  const int mine = blockIdx.x, i = mine * 64 + lane;
  const unsigned key = s_key[i];
  // blocks before this one count equal keys too (key < mine + 1), blocks behind it only smaller ones
  int c = 0;
  for (int b = wave; b < blocks; b += 16) {
    const u32x4* k4 = reinterpret_cast<const u32x4*>(s_key + 64 * b);
    if (b != mine) {
      const unsigned than = b < mine ? key + 1 : key;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const u32x4 k = k4[j];
        c += (k[0] < than) + (k[1] < than) + (k[2] < than) + (k[3] < than);
      }
    } else {
      for (int j = 0; j < 64; ++j) c += s_key[64 * b + j] < (j < lane ? key + 1 : key);
    }
  }
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
// SORT_BLOCKS contiguous parts, one workgroup each: a launch counts every part's digits, the next one places them, each
// workgroup adding up the counts before its own by itself (32768 positions: 3.5 + 7.6 us a pass; 131072: 4.8 + 11.1.  Counting
// the next pass's digits by atomics while placing took as long as the launch it saves).  A wave takes 64 consecutive positions
// at a time; lanes of equal digit find each other by ballots, so equal digits keep their order.
constexpr int SORT_BLOCKS = 128;
constexpr int SORT_BITS = 9;
constexpr int SORT_DIGITS = 1 << SORT_BITS;
constexpr int SORT_TILE = 1024;

struct SortPass {
  const void* tok; int tok64; unsigned vocab; int64_t pad;       // first pass: keys from the tokens, positions 0, 1, ...
  const unsigned* key_in; const unsigned* pos_in;                // later passes
  unsigned* key_out; unsigned* pos_out;
  unsigned* hist;                                                // [parts][SORT_DIGITS]
  int64_t n, per;                                                // positions; positions of one workgroup
  int shift, bits;
};

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
  __shared__ __attribute__((aligned(16))) unsigned s_wave[4][SORT_DIGITS];
  __shared__ __attribute__((aligned(16))) unsigned s_all[4][SORT_DIGITS];
  __shared__ unsigned s_sum[4];
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const unsigned mask = (1u << p.bits) - 1;
  const int64_t i0 = (int64_t)blockIdx.x * p.per, i1 = i0 + p.per < p.n ? i0 + p.per : p.n;
  // counts of every digit before this part, and in all: a wave adds up every fourth part, a lane 8 digits
  {
    u32x4 before[2] = {}, all[2] = {};
#pragma unroll 8
    for (unsigned b = wave; b < gridDim.x; b += 4) {
      const u32x4* h = reinterpret_cast<const u32x4*>(p.hist + (int64_t)b * SORT_DIGITS + 8 * lane);
      const u32x4 x = h[0], y = h[1];
      all[0] += x; all[1] += y;
      if (b < blockIdx.x) { before[0] += x; before[1] += y; }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      *reinterpret_cast<u32x4*>(&s_wave[wave][8 * lane + 4 * k]) = before[k];
      *reinterpret_cast<u32x4*>(&s_all[wave][8 * lane + 4 * k]) = all[k];
    }
  }
  __syncthreads();
  unsigned before[2], all[2];                                // digits 2 tid, 2 tid + 1
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = 2 * tid + k;
    before[k] = s_wave[0][d] + s_wave[1][d] + s_wave[2][d] + s_wave[3][d];
    all[k] = s_all[0][d] + s_all[1][d] + s_all[2][d] + s_all[3][d];
  }
  unsigned upto = all[0] + all[1];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const unsigned add = __shfl_up(upto, off, GVD_WAVE);
    if (lane >= off) upto += add;
  }
  if (lane == 63) s_sum[wave] = upto;
  __syncthreads();
  unsigned base = upto - (all[0] + all[1]);
  for (int w = 0; w < wave; ++w) base += s_sum[w];
  s_next[2 * tid] = base + before[0];
  s_next[2 * tid + 1] = base + all[0] + before[1];
  constexpr int ROUNDS = SORT_TILE / 256;
  for (int64_t t0 = i0; t0 < i1; t0 += SORT_TILE) {
    for (int d = tid; d < 4 * SORT_DIGITS; d += 256) (&s_wave[0][0])[d] = 0;
    unsigned key[ROUNDS], pos[ROUNDS], place[ROUNDS];
    const int64_t w0 = t0 + wave * (SORT_TILE / 4) + lane;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
      const int64_t i = w0 + 64 * r;
      key[r] = i < i1 ? sort_key(p, i) : 0;
      pos[r] = i < i1 && !p.tok ? p.pos_in[i] : (unsigned)i;
    }
    __syncthreads();
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
      if (w0 + 64 * r < i1) {
        const unsigned d = (key[r] >> p.shift) & mask;
        unsigned to = s_next[d] + place[r];
        for (int w = 0; w < wave; ++w) to += s_wave[w][d];
        p.key_out[to] = key[r];
        p.pos_out[to] = pos[r];
      }
    }
    if (t0 + SORT_TILE < i1) {
      __syncthreads();
      for (int d = tid; d < SORT_DIGITS; d += 256) s_next[d] += s_wave[0][d] + s_wave[1][d] + s_wave[2][d] + s_wave[3][d];
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------------------------------------------- sums by token
// A token of 64 positions or more has its whole groups of GROUP sorted positions (and of GROUP groups) summed beforehand, one
// wave per group with 16 rows on their way, so that the owner of a row adds up m / 1024 + some 124 rows of a token of m positions
// - a few hundred for the largest batches of texts; all of 2^25 tokens the same: 32768 + 124 (131072 positions of 2048 bf16, half of
// them in such tokens: 50 us, 5.2 TB/s).
constexpr int GROUP = 32;
constexpr int STRETCH = 32;               // 8, 16 and 32 take the same time, 64 up to a fifth more

struct SumArgs {
  const unsigned* skey; const unsigned* spos; int64_t n;
  const void* dy; int64_t ld;
  float* part1; float* part2;             // fp32 [n / GROUP][width], [n / GROUP^2][width]
  const void* table; int64_t ldt;         // for act'
  void* dw;
  unsigned vocab; int width; float scale; int act;
  unsigned slices;
};

// a lane's N columns of a row, as loaded (rows in flight cost half the registers in 16-bit types)
template <typename T, int N> __device__ __forceinline__ typename GvdVec<T, N>::type fetch(const T* row, int col) {
  if (col < 0) return {};
  return *reinterpret_cast<const typename GvdVec<T, N>::loose*>(row + col);
}

// s += `count` (<= 64) rows of x, in order: row i is the one that lane i names (`which`); FLIGHT bytes of a lane on their way
// at a time, 16 rows at most
template <typename T, int N, int FLIGHT>
__device__ __forceinline__ void add_rows(const T* x, int64_t ld, unsigned which, int count, int col, float (&s)[N]) {
  constexpr int BATCH = FLIGHT / (int)(sizeof(T) * N) < 16 ? FLIGHT / (int)(sizeof(T) * N) : 16;
  for (int i = 0; i < count; i += BATCH) {
    typename GvdVec<T, N>::type r[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (i + k < count) r[k] = fetch<T, N>(x + (int64_t)(unsigned)__builtin_amdgcn_readlane(which, i + k) * ld, col);
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (i + k < count) {
#pragma unroll
        for (int e = 0; e < N; ++e) s[e] += (float)r[k][e];
      }
  }
}

// s += rows [i, e) of partial sums
template <int N>
__device__ __forceinline__ void add_partials(const float* part, int width, int64_t i, int64_t e, int col, float (&s)[N]) {
  for (; i < e; i += 64)
    add_rows<float, N, 128>(part + i * width, width, threadIdx.x & 63, e - i < 64 ? (int)(e - i) : 64, col, s);
}

// level 1: whole groups of 32 positions of a token with 64 positions or more; level 2: whole groups of 32 such groups
template <typename T, int N, int LEVEL>
__global__ __launch_bounds__(256) void token_group_kernel(const SumArgs a) {
  const unsigned id = wave_id(), g = id / a.slices;
  const int lane = threadIdx.x & 63;
  constexpr int64_t LEN = LEVEL == 1 ? GROUP : GROUP * GROUP;
  const int64_t i0 = (int64_t)g * LEN;
  if (i0 + LEN > a.n) return;
  const int col = lane_column<N>(id - g * a.slices, a.width);
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
  if constexpr (LEVEL == 1) {
    // keys of [i0 - 32, i0 + 64): the group, and 32 more of the same on its two sides together - else the token has fewer than 64
    const int64_t b = i0 - 32 + lane, e = i0 + 32 + lane;
    const unsigned before = b >= 0 ? a.skey[b] : 0xffffffffu, after = lane < 32 && e < a.n ? a.skey[e] : 0xffffffffu;
    const unsigned which = a.spos[i0 + (lane & 31)];
    const unsigned v = __builtin_amdgcn_readlane(before, 32);
    if (v >= a.vocab || __builtin_amdgcn_readlane(before, 63) != v) return;
    if (__popcll(__ballot(before == v)) + __popcll(__ballot(after == v)) < 64) return;
    add_rows<T, N, 256>(reinterpret_cast<const T*>(a.dy), a.ld, which, GROUP, col, s);
  } else {
    const unsigned v = a.skey[i0], last = a.skey[i0 + LEN - 1];
    if (v >= a.vocab || last != v) return;
    add_rows<float, N, 256>(a.part1 + (int64_t)g * GROUP * a.width, a.width, (unsigned)lane, GROUP, col, s);
  }
  if (col >= 0) gvd_store<float, N>((LEVEL == 1 ? a.part1 : a.part2) + (int64_t)g * a.width + col, s);
}

// ---------------------------------------------------------------------------------------------- few tokens: one launch
// n <= SMALL_MAX: a workgroup owns `rows` consecutive rows of the table and 64 * N columns.  It looks at all tokens and lists
// the positions of its rows, in order; a wave sums and writes one row at a time, and rows of more than SMALL_ALONE positions
// are left for all sixteen waves: each sums its sixteenth of the list, and the sums are added in order.  One launch instead of
// a sort, groups and rows: at these sizes a launch costs the host (4 us) as much as the work takes.  Every workgroup looks at all
// tokens, so it is for tables of at most SMALL_GROUPS workgroups of SMALL_ROWS rows and 256 columns, or a narrower table's width:
// two for every CU, which run side by side.  Measured with events (some 5 us of them the events'), words of falling frequency,
// this launch and the sort's several: 5000 x 512 fp32, 5 words 11.1 and 11.8 us, 256 12.0 and 16.0, 1280 17.0 and 20.6, 4096 28.0 and
// 26.8, and 8 us less of the host; 432 x 301 fp16, 2049 words, 16.6 and 26.0.  At the limit: 32768 x 64 fp32, 5 words 12.8 and 11.6,
// 1280 17.8 and 21.6, 4096 27.4 and 24.8.  Above it the other way round: 65536 x 32 fp32 (1024 workgroups) 20.0 and 11.7, 24.2 and
// 21.3, 37.9 and 25.0; 2^20 x 8 (16384) 217 and 33, 225 and 43, 241 and 47; 50000 x 1024 bf16, 256 words, 48.3 and 27.4.
constexpr int SMALL_MAX = 4096;
constexpr int SMALL_ROWS = 64;
constexpr int64_t SMALL_GROUPS = 512;
constexpr int SMALL_WAVES = 16;
constexpr int SMALL_ALONE = 128;            // positions that a wave adds up by itself: eight times 16 on their way

// row v = s, scaled
template <typename T, int N>
__device__ __forceinline__ void put_row(const SumArgs& a, int64_t v, int col, const float (&s)[N]) {
  if (col < 0) return;
  float x[N];
  if (a.act) {
    const typename GvdVec<T, N>::type w = fetch<T, N>(reinterpret_cast<const T*>(a.table) + v * a.ldt, col);
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = (float)w[k] * a.scale > 0.f ? s[k] * a.scale : 0.f;
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = s[k] * a.scale;
  }
  gvd_store<T, N>(reinterpret_cast<T*>(a.dw) + v * a.width + col, x);
}

template <typename T, int N>
__global__ __launch_bounds__(64 * SMALL_WAVES) void token_small_kernel(const SumArgs a, const void* tok, int tok64, int64_t pad,
                                                                       int rows) {
  __shared__ unsigned s_list[SMALL_MAX];                     // row of the workgroup << 16 | position
  __shared__ unsigned s_pos[SMALL_WAVES][128];
  __shared__ float s_sum[SMALL_WAVES][64 * N];
  __shared__ int s_count[SMALL_ROWS];
  __shared__ int s_found[SMALL_WAVES];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const unsigned unit = blockIdx.x / a.slices;
  const int col = lane_column<N>(blockIdx.x - unit * a.slices, a.width);
  const unsigned v0 = unit * (unsigned)rows, mine = a.vocab - v0 < (unsigned)rows ? a.vocab - v0 : (unsigned)rows;
  const T* dy = reinterpret_cast<const T*>(a.dy);
  const int n = (int)a.n;
  const int each = (n + 64 * SMALL_WAVES - 1) / (64 * SMALL_WAVES) * 64;      // a wave looks at `each` tokens, 64 at a time
  if (threadIdx.x < SMALL_ROWS) s_count[threadIdx.x] = 0;
  unsigned row[SMALL_MAX / (64 * SMALL_WAVES)];
#pragma unroll
  for (int i = 0; i < SMALL_MAX / (64 * SMALL_WAVES); ++i) {
    const int at = wave * each + 64 * i + lane;
    row[i] = 64 * i < each && at < n ? token_key(tok, tok64, at, a.vocab, pad) - v0 : 0xffffffffu;
  }
  int found = 0;
#pragma unroll
  for (int i = 0; i < SMALL_MAX / (64 * SMALL_WAVES); ++i) found += __popcll(__ballot(row[i] < mine));
  if (lane == 0) s_found[wave] = found;
  __syncthreads();
  int at = 0, total = 0;
#pragma unroll
  for (int w = 0; w < SMALL_WAVES; ++w) { at += w < wave ? s_found[w] : 0; total += s_found[w]; }
#pragma unroll
  for (int i = 0; i < SMALL_MAX / (64 * SMALL_WAVES); ++i) {
    const unsigned long long in = __ballot(row[i] < mine);
    if (row[i] < mine) {
      s_list[at + __popcll(in & ((1ull << lane) - 1ull))] = row[i] << 16 | (unsigned)(wave * each + 64 * i + lane);
      atomicAdd(&s_count[row[i]], 1);
    }
    at += __popcll(in);
  }
  __syncthreads();
  // s += the positions of row r in list entries [from, to): collected first, so that 64 of them are added in one go
  const auto add_listed = [&](unsigned r, int from, int to, float (&s)[N]) {
    unsigned* pos = s_pos[wave];
    int have = 0;
    for (int i = from; i < to; i += 64) {
      const unsigned e = i + lane < to ? s_list[i + lane] : 0xffffffffu;
      const unsigned long long all = __ballot(e >> 16 == r);
      if (e >> 16 == r) pos[have + __popcll(all & ((1ull << lane) - 1ull))] = e & 0xffffu;
      have += __popcll(all);
      if (have < 64 && i + 64 < to) continue;
      wave_lds_fence();
      const unsigned which = pos[lane], rest = pos[64 + lane];
      wave_lds_fence();
      pos[lane] = rest;
      const int now = have < 64 ? have : 64;
      add_rows<T, N, 256>(dy, a.ld, which, now, col, s);
      have -= now;
    }
    wave_lds_fence();
    if (have) add_rows<T, N, 256>(dy, a.ld, pos[lane], have, col, s);
    wave_lds_fence();
  };
  for (unsigned r = wave; r < mine; r += SMALL_WAVES) {
    if (s_count[r] > SMALL_ALONE) continue;
    float s[N];
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = 0.f;
    if (s_count[r]) add_listed(r, 0, total, s);
    put_row<T, N>(a, v0 + r, col, s);
  }
  for (unsigned r = 0; r < mine; ++r) {
    if (s_count[r] <= SMALL_ALONE) continue;
    float s[N];
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = 0.f;
    add_listed(r, total * wave / SMALL_WAVES, total * (wave + 1) / SMALL_WAVES, s);
#pragma unroll
    for (int k = 0; k < N; ++k) s_sum[wave][k * 64 + lane] = s[k];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < SMALL_WAVES; ++w)
#pragma unroll
        for (int k = 0; k < N; ++k) s[k] += s_sum[w][k * 64 + lane];
      put_row<T, N>(a, v0 + r, col, s);
    }
    __syncthreads();
  }
}

// first sorted position i in [lo, n) with skey[i] >= v (RISE = 0), or skey[i] + i >= v (RISE = 1): 64 lanes look at 64 places
// at a time
template <int RISE>
__device__ __forceinline__ int64_t wave_lower_bound(const unsigned* skey, int64_t lo, int64_t n, unsigned v, int lane) {
  int64_t len = n - lo;                          // the answer is in [lo, lo + len]
  while (len > 0) {
    const int64_t step = (len + 63) >> 6;
    const int64_t at = lo + (int64_t)lane * step;
    const bool less = at < lo + len && skey[at] + RISE * (unsigned)at < v;
    const int c = __popcll(__ballot(less));      // (ascending: the first c lanes)
    if (c == 0) return lo;
    const int64_t from = lo + (int64_t)(c - 1) * step + 1;
    const int64_t to = c < 64 && lo + (int64_t)c * step < lo + len ? lo + (int64_t)c * step : lo + len;
    lo = from;
    len = to - from;
  }
  return lo;
}

// The rows of the table, each followed by its sorted positions, are one sequence of vocab + n entries: row v is entry v +
// (positions of smaller keys).  It is cut into stretches of STRETCH entries, and a wave owns the rows that lie in its stretch
// (and 64 * N columns): it adds up their positions - fewer than 64 behind the stretch's end - and writes them, rows without a
// position as zeros.  So no wave has much more to do than another, whatever the tokens are (equal numbers of rows a wave took
// 394 us instead of 33 for 32768 words of falling frequency: the frequent ones lie side by side).  It walks 64 sorted positions
// at a time; the dy rows of several tokens are on their way together.  Bound by dy and dw: 131072 x 2048 bf16 of each, 176 us,
// 4.6 TB/s of what is left of dy and dw.
template <typename T, int N, bool PAST>
__global__ __launch_bounds__(256) void token_rows_kernel(const SumArgs a) {
  const unsigned id = wave_id(), unit = id / a.slices;
  const int lane = threadIdx.x & 63;
  const int64_t d0 = (int64_t)unit * STRETCH, d1 = d0 + STRETCH;
  if (d0 >= (int64_t)a.vocab + a.n) return;
  const int col = lane_column<N>(id - unit * a.slices, a.width);
  const T* dy = reinterpret_cast<const T*>(a.dy);
  T* dw = reinterpret_cast<T*>(a.dw);
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) s[k] = 0.f;
  // the first row of the stretch, `cur`, and its first position, `i`: behind i positions and d0 - i rows, or, if row d0 - i began
  // before the stretch, behind the rest of its positions
  int64_t i = wave_lower_bound<1>(a.skey, 0, a.n, (unsigned)d0, lane);
  unsigned cur = (unsigned)(d0 - i);
  if (i > 0 && i < a.n && a.skey[i - 1] == cur) {
    const unsigned long long same = __ballot(i + lane < a.n && a.skey[i + lane] == cur);
    i = ~same ? i + __popcll(same) : wave_lower_bound<0>(a.skey, i + 64, a.n, cur + 1, lane);
    ++cur;
  } else if (i > 0 && i == a.n && a.skey[i - 1] == cur) {
    ++cur;
  }
  const auto put = [&](unsigned v, const float (&x)[N]) {
    if (col < 0) return;
    T* o = dw + (int64_t)v * a.width + col;
    if constexpr (PAST) gvd_store_past<T, N>(o, x); else gvd_store<T, N>(o, x);
  };
  // rows cur ... v - 1 have no positions; row v, where there is a sum for it, is s
  const auto finish = [&](int64_t v, bool sum) {
    float x[N];
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = 0.f;
    for (; (int64_t)cur < v; ++cur) put(cur, x);
    if (!sum) return;
    if (a.act) {
      const typename GvdVec<T, N>::type w = fetch<T, N>(reinterpret_cast<const T*>(a.table) + v * a.ldt, col);
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = (float)w[k] * a.scale > 0.f ? s[k] * a.scale : 0.f;
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = s[k] * a.scale;
    }
    put((unsigned)v, x);
    cur = (unsigned)v + 1;
#pragma unroll
    for (int k = 0; k < N; ++k) s[k] = 0.f;
  };
  while (true) {
    const unsigned key = i + lane < a.n ? a.skey[i + lane] : a.vocab;
    const unsigned which = i + lane < a.n ? a.spos[i + lane] : 0;
    const unsigned first = __builtin_amdgcn_readfirstlane(key), last = __builtin_amdgcn_readlane(key, 63);
    finish((int64_t)first < d1 - i ? (int64_t)first : d1 - i, false);
    if (first >= a.vocab || (int64_t)first >= d1 - i) break;
    if (first == last) {                         // 64 positions or more of one token
      const int64_t e = wave_lower_bound<0>(a.skey, i + 64, a.n, first + 1, lane);
      const int64_t g1 = (i + GROUP - 1) / GROUP, g2 = e / GROUP;                 // whole groups (there is one at least)
      const int head = (int)(g1 * GROUP - i), ends = head + (int)(e - g2 * GROUP);  // positions before and behind them
      const int64_t at = lane < head ? i + lane : g2 * GROUP + lane - head;
      add_rows<T, N, 128>(dy, a.ld, lane < ends ? a.spos[at] : 0, ends, col, s);
      const int64_t h1 = (g1 + GROUP - 1) / GROUP, h2 = g2 / GROUP;               // whole groups of groups
      const bool two = h1 < h2;
      for (int k = 0; k < 3; ++k) {              // groups before, groups of groups, groups behind them
        const int64_t from = k == 0 ? g1 : k == 1 ? h1 : two ? h2 * GROUP : g2;
        const int64_t to = k == 0 ? (two ? h1 * GROUP : g2) : k == 1 ? (two ? h2 : h1) : g2;
        add_partials<N>(k == 1 ? a.part2 : a.part1, a.width, from, to, col, s);
      }
      finish(first, true);
      i = e;
      continue;
    }
    // the tokens that end within these 64 positions, up to the first one whose row lies behind the stretch
    const unsigned left = __shfl_up(key, 1, GVD_WAVE);
    const unsigned long long behind = __ballot((lane == 0 || key != left) && (key >= a.vocab || (int64_t)key + i + lane >= d1));
    int count = __popcll(__ballot(key != last));
    if (behind) count = count < __ffsll(behind) - 1 ? count : __ffsll(behind) - 1;
    constexpr int BATCH = 4;
    for (int j0 = 0; j0 < count; j0 += BATCH) {
      typename GvdVec<T, N>::type x[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (j0 + k < count) x[k] = fetch<T, N>(dy + (int64_t)(unsigned)__builtin_amdgcn_readlane(which, j0 + k) * a.ld, col);
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        if (j0 + k < count) {
          const unsigned v = __builtin_amdgcn_readlane(key, j0 + k);
#pragma unroll
          for (int e = 0; e < N; ++e) s[e] += (float)x[k][e];
          if (__builtin_amdgcn_readlane(key, j0 + k + 1) != v) finish(v, true);   // (count <= 63: lane 63 belongs to a later token)
        }
      }
    }
    i += count;
  }
}

// ---------------------------------------------------------------------------------------------------------------- host
// columns of one lane: 16 bytes where the width fills a wave with them, else the smallest power of two that covers the width
int lane_columns(int width, int dtype) {
  const int most = dtype == GVD_F32 ? 4 : 8;
  int n = 1;
  while (n < most && 64 * n < width) n *= 2;
  return n;
}

constexpr int64_t MAX_WAVES = (1ll << 26) - 4;      // (a launch holds fewer than 2^32 threads)

int64_t align256(int64_t x) { return (x + 255) & ~(int64_t)255; }

struct BwdSpace {
  int64_t skey, spos, key2, pos2, hist, part1, part2, bytes;
  bool small, rank;
  int passes, bits, blocks;
  int64_t per;
};

BwdSpace bwd_space(int64_t n, int64_t vocab, int width) {
  BwdSpace s = {};
  s.small = n <= SMALL_MAX && (vocab + SMALL_ROWS - 1) / SMALL_ROWS * ((width + 255) / 256) <= SMALL_GROUPS;
  if (s.small) return s;                                // (no workspace)
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
  const unsigned slices = (unsigned)((width + 64 * N - 1) / (64 * N));
  const bool many = n * slices >= 16384;   // (four rows a wave still leave four waves to every SIMD)
  const int64_t waves = (many ? (n + 3) / 4 : n) * slices;
  if (waves > MAX_WAVES) return GVD_EINVAL;
  const bool past = n * width * (int64_t)sizeof(T) > GVD_CACHE_BYTES;
  const auto kernel = !many ? embedding_fwd_kernel<T, N, 1, false>
                      : past ? embedding_fwd_kernel<T, N, 4, true> : embedding_fwd_kernel<T, N, 4, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, tok, tok64, n, reinterpret_cast<const T*>(table),
                     ld, (unsigned)vocab, width, scale, act, reinterpret_cast<T*>(out), ldo, slices);
  GVD_CHECK_LAUNCH();
  return 0;
}

template <typename T, int N> int launch_small(SumArgs a, const void* tok, int tok64, int64_t pad, hipStream_t st) {
  a.slices = (unsigned)((a.width + 64 * N - 1) / (64 * N));
  // rows a workgroup, up to 64, for two workgroups to every CU, or four: fewer frequent words in one workgroup, but all tokens
  // looked at twice as often (5000 x 512 fp32, us with events: 5 words 11.1 and 14.3, 1280 18.6 and 16.8, 4096 39 and 31.5)
  const int64_t groups_wanted = a.n <= 512 ? 512 : 1024;
  int rows = 1;
  while (rows < SMALL_ROWS && (int64_t)a.vocab * a.slices > rows * groups_wanted) ++rows;
  const int64_t groups = ((int64_t)a.vocab + rows - 1) / rows * a.slices;
  if (groups > MAX_WAVES / SMALL_WAVES) return GVD_EINVAL;
  hipLaunchKernelGGL((token_small_kernel<T, N>), dim3((unsigned)groups), dim3(64 * SMALL_WAVES), 0, st, a, tok, tok64, pad, rows);
  GVD_CHECK_LAUNCH();
  return 0;
}

template <typename T, int N> int launch_sums(SumArgs a, hipStream_t st) {
  a.slices = (unsigned)((a.width + 64 * N - 1) / (64 * N));
  const int64_t g1 = a.n / GROUP * a.slices, g2 = a.n / (GROUP * GROUP) * a.slices;
  const int64_t owners = ((int64_t)a.vocab + a.n + STRETCH - 1) / STRETCH * a.slices;
  if (g1 > MAX_WAVES || owners > MAX_WAVES) return GVD_EINVAL;
  if (a.n >= 64) {
    hipLaunchKernelGGL((token_group_kernel<T, N, 1>), dim3((unsigned)((g1 + 3) / 4)), dim3(256), 0, st, a);
    GVD_CHECK_LAUNCH();
  }
  if (g2) {
    hipLaunchKernelGGL((token_group_kernel<T, N, 2>), dim3((unsigned)((g2 + 3) / 4)), dim3(256), 0, st, a);
    GVD_CHECK_LAUNCH();
  }
  const bool past = (int64_t)a.vocab * a.width * (int64_t)sizeof(T) > GVD_CACHE_BYTES;
  hipLaunchKernelGGL((past ? token_rows_kernel<T, N, true> : token_rows_kernel<T, N, false>), dim3((unsigned)((owners + 3) / 4)),
                     dim3(256), 0, st, a);
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

extern "C" int gvd_embedding_bwd(const void* tokens, int tok64, int64_t n, const void* dy, int64_t ld_dy, const void* table,
                                 int64_t ld, int64_t vocab, int width, int dtype, float scale, int act, int64_t padding_idx, void* dw,
                                 void* workspace, size_t workspace_bytes, gvd_stream_t stream) {
  if (!tokens || !dy || !dw || bad_shape(n, vocab, width, dtype) || ld_dy < 0 || (act && (!table || ld < width)))
    return GVD_EINVAL;
  const BwdSpace s = bwd_space(n, vocab, width);
  if (s.bytes && (!workspace || workspace_bytes < (size_t)s.bytes || !gvd_aligned16(workspace))) return GVD_EINVAL;
  const hipStream_t st = gvd_s(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  const auto at = [&](int64_t o) { return reinterpret_cast<unsigned*>(ws + o); };
  const int64_t pad = padding_idx < 0 ? -1 : padding_idx;
  SumArgs a = {};
  a.n = n;
  a.dy = dy; a.ld = ld_dy;
  a.table = table; a.ldt = ld;
  a.dw = dw;
  a.vocab = (unsigned)vocab; a.width = width; a.scale = scale; a.act = act;
  if (s.small) {
#define GVD_SMALL(T, N) launch_small<T, N>(a, tokens, tok64, pad, st)
    GVD_BY_TYPE(GVD_SMALL)
#undef GVD_SMALL
  }
  a.skey = at(s.skey); a.spos = at(s.spos);
  a.part1 = reinterpret_cast<float*>(ws + s.part1); a.part2 = reinterpret_cast<float*>(ws + s.part2);
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
#define GVD_SUMS(T, N) launch_sums<T, N>(a, st)
  GVD_BY_TYPE(GVD_SUMS)
#undef GVD_SUMS
}
