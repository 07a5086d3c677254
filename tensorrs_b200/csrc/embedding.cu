// embedding.cu -- the rows of a table that belong to a sequence of tokens, and
// the gradient of the table.
//
//   trs_embedding           out[t] = scale table[id_t]
//   trs_embedding_backward  grad[v] = sum over the t with id_t = v, in the order
//                           of t, of scale grad_out[t] (or that added to grad[v])
//
// An id outside [0, V) (padding, or a row that another part of a split table
// holds) gives a row of zeros and no gradient.
//
// What bounds both: HBM.  The lookup reads N rows and writes N rows.  The
// gradient reads N rows and writes the V rows of the table, most of them zeros.
// Few tokens make up most of a text, so that one row of the table can collect
// thousands of rows; adding them with atomics would serialise there and change
// its result from run to run.  Instead:
//
//   emb_keys_kernel     the ids as 32-bit keys (V for those outside), and the
//                       counts of their lowest digit per tile of 4096 tokens
//   emb_sort_kernel     one digit (up to 9 bits) of a stable radix sort of
//                       (key, token): two launches below V = 2^18.  Every CTA
//                       finds its places from all tiles' counts (no CTA waits on
//                       another), and counts the next digit as it writes.
//   emb_sort_one_kernel the keys and all digits in one launch, for up to 4096 tokens
//   emb_sum_kernel      up to 32 sorted positions per group of lanes: rows of one key
//                       are added in f64 in registers and written at the end of
//                       the run; a run that crosses into other positions leaves
//                       partial sums
//   emb_join_kernel     adds the partial sums of such a run in order
//
// The zeros of the other rows are written by additional CTAs of the first
// kernels, which leave nearly all of HBM's bandwidth free.
//
// Measured: 16384 tokens of 2048 f32 looked up 37 us (33.7 the kernel: 5.6 TB/s,
// 0.87 of the copy rate); gradient of 16384 tokens of 1024 into 50000 rows 76 us:
// zeros and sorting 40 (205 MB, 5.1 TB/s; the sort alone 19), sums 24, joins 10.
// Bulk copies of zeros from shared memory (94 us in all), 32-byte stores (80) and
// zeros next to the sums for the rows that no token looked up (101) were slower.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>

#include "../../include/trs.h"
#include "kernels.cuh"
#include "tokens.h"

namespace trs {
namespace {

constexpr int kEmbThreads = 256;

template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// How a CTA's threads share rows of D elements: groups of 2^lg lanes, a lane
// taking V elements at a time.
struct Lanes {
  int lg;
  int chunks;  // D / V
};

struct EmbDev {
  const char* table;
  int64_t tv, td;        // strides of the table (backward: of its gradient)
  char* grad;            // backward: the table's gradient
  RowsDev ids, rows;     // rows: the output, or its gradient
  int ids64;
  uint32_t N, V;
  int D;
  Lanes l;
  FastDiv f_T;
  double scale;
  int wide;              // lookup: the scale is no normal number of the table's type
  int accumulate;
  // backward
  uint32_t *key[2], *tok[2];
  uint32_t* hist[4];     // [tile][bin] of every digit
  uint32_t* crossing;    // count, then the positions' groups in which a crossing run begins
  double* part;          // [group of positions][2][D]
  uint32_t tiles, groups;
  int digits, bits;
  int positions;         // sorted positions per group of lanes, a power of two up to 32
};

__device__ __forceinline__ uint32_t emb_key(const EmbDev& d, uint32_t r) {
  const uint32_t b = fdiv(r, d.f_T), t = r - b * d.f_T.d;
  const int64_t at = b * d.ids.sb + t * d.ids.st;
  const int64_t id = d.ids64 ? static_cast<const int64_t*>(d.ids.p)[at] : static_cast<const int32_t*>(d.ids.p)[at];
  return id < 0 || id >= (int64_t)d.V ? d.V : (uint32_t)id;
}
template <class T>
__device__ __forceinline__ T* row_at(const EmbDev& d, uint32_t r) {
  const uint32_t b = fdiv(r, d.f_T), t = r - b * d.f_T.d;
  return static_cast<T*>(d.rows.p) + b * d.rows.sb + t * d.rows.st;
}
template <class T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p, int64_t c, int64_t sd) {
  if constexpr (V > 1) return *reinterpret_cast<const Vec<T, V>*>(p + c * V);
  else return Vec<T, V>{{p[c * sd]}};
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, int64_t c, int64_t sd, const Vec<T, V>& x) {
  if constexpr (V > 1) *reinterpret_cast<Vec<T, V>*>(p + c * V) = x;
  else p[c * sd] = x.v[0];
}

// ---- lookup ------------------------------------------------------------------

template <class T, int V>
__global__ void __launch_bounds__(kEmbThreads) emb_lookup_kernel(const EmbDev d) {
  constexpr int U = 4;  // rows of a group in flight
  const int L = 1 << d.l.lg, per = kEmbThreads >> d.l.lg, c0 = threadIdx.x & (L - 1);
  // A scale that f32 holds as a normal number is rounded to it, as the table's own values are;
  // any other would lose its digits or all of itself, and is applied in f64 (16384 tokens of
  // 2048 from random rows: 45.0 and 45.3 us).
  const T scale = (T)d.scale;
  const bool wide = d.wide;
  for (uint64_t base = (uint64_t)blockIdx.x * per * U + (threadIdx.x >> d.l.lg); base < d.N;
       base += (uint64_t)gridDim.x * per * U) {
    uint32_t id[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const uint64_t r = base + (uint64_t)j * per;
      id[j] = r < d.N ? emb_key(d, (uint32_t)r) : d.V;
    }
    for (int c = c0; c < d.l.chunks; c += L) {
      Vec<T, V> x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[j].v[i] = (T)0;
        if (id[j] < d.V) x[j] = load<T, V>(reinterpret_cast<const T*>(d.table) + (int64_t)id[j] * d.tv, c, d.td);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const uint64_t r = base + (uint64_t)j * per;
        if (r >= d.N) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) x[j].v[i] = id[j] >= d.V ? (T)0 : wide ? (T)((double)x[j].v[i] * d.scale) : x[j].v[i] * scale;
        store<T, V>(row_at<T>(d, (uint32_t)r), c, d.rows.sd, x[j]);
      }
    }
  }
}

// ---- gradient: sorting the tokens ----------------------------------------------

constexpr int kSortThreads = 512;
constexpr int kSortTile = 4096;              // tokens per CTA
constexpr int kBins = 512;
constexpr int kWarps = kSortThreads / 32;
constexpr int kRounds = kSortTile / kSortThreads;  // a warp's share: rounds of 32 consecutive tokens

// The part `share` of `shares` of the zeros, by the CTAs behind the tiles'.
template <class T, int V>
__device__ __forceinline__ void emb_zeros(const EmbDev& d, int share, int shares) {
  const uint32_t cta = blockIdx.x - d.tiles, ctas = gridDim.x - d.tiles;
  const int L = 1 << d.l.lg, per = kSortThreads >> d.l.lg, c0 = threadIdx.x & (L - 1);
  const uint64_t r0 = (uint64_t)d.V * share / shares, r1 = (uint64_t)d.V * (share + 1) / shares;
  Vec<T, V> z;
#pragma unroll
  for (int i = 0; i < V; ++i) z.v[i] = (T)0;
  for (uint64_t r = r0 + (uint64_t)cta * per + (threadIdx.x >> d.l.lg); r < r1; r += (uint64_t)ctas * per)
    for (int c = c0; c < d.l.chunks; c += L)
      store<T, V>(reinterpret_cast<T*>(d.grad) + (int64_t)r * d.tv, c, d.td, z);
}

template <class T, int V>
__global__ void __launch_bounds__(kSortThreads) emb_keys_kernel(const EmbDev d) {
  __shared__ uint32_t count[kBins];
  pdl_launch_dependents();
  if (blockIdx.x >= d.tiles) {
    emb_zeros<T, V>(d, 0, d.digits + 1);
    return;
  }
  count[threadIdx.x] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) d.crossing[0] = 0;
  for (int p = 1; p < d.digits; ++p) d.hist[p][blockIdx.x * kBins + threadIdx.x] = 0;
  __syncthreads();
  const uint32_t mask = (1u << d.bits) - 1;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const uint64_t r = (uint64_t)blockIdx.x * kSortTile + i * kSortThreads + threadIdx.x;
    if (r < d.N) {
      const uint32_t k = emb_key(d, (uint32_t)r);
      d.key[0][r] = k;
      atomicAdd(&count[k & mask], 1u);
    }
  }
  __syncthreads();
  d.hist[0][blockIdx.x * kBins + threadIdx.x] = count[threadIdx.x];
}

// The lanes whose bin (of `bits` bits) is this lane's, among those that are `there`
// (a ballot per bit: several times as fast as match.any).
__device__ __forceinline__ uint32_t emb_peers(uint32_t bin, bool there, int bits) {
  uint32_t peers = __ballot_sync(0xffffffffu, there);
  for (int i = 0; i < bits; ++i) {
    const uint32_t set = __ballot_sync(0xffffffffu, (bin >> i) & 1u);
    peers &= (bin >> i) & 1u ? set : ~set;
  }
  return peers;
}

// What a CTA's stable sort by one digit shares: a warp's tokens of every bin, then
// where they go.
struct SortShared {
  uint32_t at[kWarps][kBins];
  uint32_t sums[kWarps];
};

// rank[i]: the place of this thread's token of round i among its warp's tokens of the
// bin; at: how many each warp has.
__device__ __forceinline__ void emb_rank(SortShared& sh, const uint32_t (&bin)[kRounds], const bool (&there)[kRounds], int bits,
                                         uint32_t (&rank)[kRounds]) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sh.at[w][threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const uint32_t peers = emb_peers(bin[i], there[i], bits);
    uint32_t have = 0;
    if (there[i]) have = sh.at[warp][bin[i]];
    __syncwarp();
    rank[i] = have + __popc(peers & ((1u << lane) - 1));
    if (there[i] && lane == __ffs(peers) - 1) sh.at[warp][bin[i]] = have + __popc(peers);
    __syncwarp();
  }
  __syncthreads();
}

// at: the first place of each warp's tokens of this thread's bin, given how many of
// the bin there are in all and before this tile.
__device__ __forceinline__ void emb_places(SortShared& sh, uint32_t total, uint32_t before) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint32_t scan = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, scan, o);
    if (lane >= o) scan += y;
  }
  if (lane == 31) sh.sums[warp] = scan;
  __syncthreads();
  uint32_t place = scan - total + before;
  for (int w = 0; w < warp; ++w) place += sh.sums[w];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t n = sh.at[w][threadIdx.x];
    sh.at[w][threadIdx.x] = place;
    place += n;
  }
  __syncthreads();
}

// Sorts by digit p, stable; from buffer p % 2 into the other one.
template <class T, int V>
__global__ void __launch_bounds__(kSortThreads) emb_sort_kernel(const EmbDev d, int p) {
  __shared__ SortShared sh;
  pdl_launch_dependents();
  if (blockIdx.x >= d.tiles) {
    emb_zeros<T, V>(d, p + 1, d.digits + 1);
    pdl_wait();
    return;
  }
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  pdl_wait();
  const uint32_t mask = (1u << d.bits) - 1, shift = p * d.bits;
  const uint64_t first = (uint64_t)blockIdx.x * kSortTile + warp * (32 * kRounds);
  uint32_t key[kRounds], tok[kRounds], bin[kRounds], rank[kRounds];
  bool there[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const uint64_t r = first + i * 32 + lane;
    there[i] = r < d.N;
    key[i] = there[i] ? d.key[p & 1][r] : 0;
    tok[i] = p == 0 ? (uint32_t)r : there[i] ? d.tok[p & 1][r] : 0;
    bin[i] = (key[i] >> shift) & mask;
  }
  // this thread's bin: all tiles' tokens, and those of the earlier tiles
  uint32_t total = 0, before = 0;
  for (uint32_t t = 0; t < d.tiles; ++t) {
    const uint32_t n = d.hist[p][t * kBins + threadIdx.x];
    total += n;
    before += t < blockIdx.x ? n : 0;
  }
  emb_rank(sh, bin, there, d.bits, rank);
  emb_places(sh, total, before);
  const bool last = p + 1 == d.digits;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    if (!there[i]) continue;
    const uint32_t to = sh.at[warp][bin[i]] + rank[i];
    d.key[(p + 1) & 1][to] = key[i];
    d.tok[(p + 1) & 1][to] = tok[i];
    if (!last) atomicAdd(&d.hist[p + 1][to / kSortTile * kBins + ((key[i] >> (shift + d.bits)) & mask)], 1u);
  }
}

// All of it in one launch for tokens of one tile; the zeros by the other CTAs.
template <class T, int V>
__global__ void __launch_bounds__(kSortThreads) emb_sort_one_kernel(const EmbDev d) {
  extern __shared__ uint32_t s_raw[];
  pdl_launch_dependents();
  if (blockIdx.x >= 1) {
    emb_zeros<T, V>(d, 0, 1);
    return;
  }
  SortShared& sh = *reinterpret_cast<SortShared*>(s_raw);
  uint32_t* s_key = s_raw + sizeof(SortShared) / 4;
  uint32_t* s_tok = s_key + kSortTile;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t mask = (1u << d.bits) - 1, first = warp * (32 * kRounds) + lane;
  uint32_t key[kRounds], tok[kRounds], bin[kRounds], rank[kRounds];
  bool there[kRounds];
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    tok[i] = first + i * 32;
    there[i] = tok[i] < d.N;
    key[i] = there[i] ? emb_key(d, tok[i]) : 0;
  }
  if (threadIdx.x == 0) d.crossing[0] = 0;
  for (int p = 0; p < d.digits; ++p) {
#pragma unroll
    for (int i = 0; i < kRounds; ++i) bin[i] = (key[i] >> (p * d.bits)) & mask;
    emb_rank(sh, bin, there, d.bits, rank);
    uint32_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) total += sh.at[w][threadIdx.x];
    emb_places(sh, total, 0);
    const bool last = p + 1 == d.digits;
    uint32_t* keys = last ? d.key[d.digits & 1] : s_key;
    uint32_t* toks = last ? d.tok[d.digits & 1] : s_tok;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      if (!there[i]) continue;
      const uint32_t to = sh.at[warp][bin[i]] + rank[i];
      keys[to] = key[i];
      toks[to] = tok[i];
    }
    __syncthreads();
    if (last) break;
#pragma unroll
    for (int i = 0; i < kRounds; ++i)
      if (there[i]) {
        key[i] = s_key[first + i * 32];
        tok[i] = s_tok[first + i * 32];
      }
    __syncthreads();
  }
}

// ---- gradient: adding the rows --------------------------------------------------

template <class T>
__device__ __forceinline__ T emb_result(const EmbDev& d, double sum, T before) {
  const double x = d.accumulate ? __fma_rn(sum, d.scale, (double)before) : sum * d.scale;
  return (T)x;
}

template <class T, int V>
__global__ void __launch_bounds__(kEmbThreads) emb_sum_kernel(const EmbDev d) {
  constexpr int U = 4;  // rows in flight (8: 82 us against 77, 16 81: the registers cost CTAs)
  __shared__ uint32_t s_key[kEmbThreads], s_tok[kEmbThreads];
  pdl_launch_dependents();
  pdl_wait();
  const int L = 1 << d.l.lg, per = kEmbThreads >> d.l.lg, c0 = threadIdx.x & (L - 1), P = d.positions;
  const uint32_t* key = d.key[d.digits & 1];
  const uint32_t* tok = d.tok[d.digits & 1];
  // the CTA's positions, at most one per thread: groups of few lanes take fewer positions
  const uint64_t first = (uint64_t)blockIdx.x * per * P;
  for (int i = threadIdx.x; i < per * P; i += kEmbThreads) {
    const bool there = first + i < d.N;
    s_key[i] = there ? key[first + i] : ~0u;
    s_tok[i] = there ? tok[first + i] : 0;
  }
  __syncthreads();
  const int lg = threadIdx.x >> d.l.lg;  // group in the CTA
  const uint32_t g = blockIdx.x * per + lg;
  if (g >= d.groups) return;
  const uint32_t p0 = g * P, n = min((uint32_t)P, d.N - p0);
  const uint32_t *keys = s_key + lg * P, *toks = s_tok + lg * P;
  const uint32_t prev = p0 > 0 ? key[p0 - 1] : ~0u, next = p0 + n < d.N ? key[p0 + n] : ~0u;
  const uint32_t head = keys[0], tail = keys[n - 1];
  if (head == d.V) return;
  // a run that begins here and goes on
  if (c0 == 0 && tail == next && tail != d.V && !(head == tail && prev == head))
    d.crossing[1 + atomicAdd(d.crossing, 1u)] = g;
  for (int c = c0; c < d.l.chunks; c += L) {
    double acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.0;
    uint32_t cur = head;
    bool from_before = prev == head;
    auto flush = [&](bool goes_on) {
      if (from_before || goes_on) {
        double* to = d.part + ((uint64_t)g * 2 + (from_before ? 0 : 1)) * d.D + (int64_t)c * V;
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = acc[i];
      } else {
        T* row = reinterpret_cast<T*>(d.grad) + (int64_t)cur * d.tv;
        Vec<T, V> x;
        if (d.accumulate) x = load<T, V>(row, c, d.td);
#pragma unroll
        for (int i = 0; i < V; ++i) x.v[i] = emb_result<T>(d, acc[i], d.accumulate ? x.v[i] : (T)0);
        store<T, V>(row, c, d.td, x);
      }
    };
    for (uint32_t p = 0; p < n; p += U) {
      uint32_t k[U];
      Vec<T, V> x[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        k[j] = p + j < n ? keys[p + j] : d.V;
        if (k[j] < d.V) x[j] = load<T, V>(row_at<T>(d, toks[p + j]), c, d.rows.sd);
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (k[j] >= d.V) continue;  // sorted last: nothing follows
        if (k[j] != cur) {
          flush(false);
          cur = k[j];
          from_before = false;
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i] = 0.0;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = __dadd_rn(acc[i], (double)x[j].v[i]);
      }
    }
    flush(cur == next);
  }
}

// Runs that cross from one group of positions into others: 32 lanes times C columns
// times 8 parts of the run, folded in order.
template <class T>
__global__ void __launch_bounds__(256) emb_join_kernel(const EmbDev d) {
  constexpr int C = 2;
  __shared__ double s[8][32 * C];
  pdl_wait();
  const uint32_t* key = d.key[d.digits & 1];
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32, blocks = (d.D + 32 * C - 1) / (32 * C), P = d.positions;
  const uint32_t n = d.crossing[0];
  for (uint64_t item = blockIdx.x; item < (uint64_t)n * blocks; item += gridDim.x) {
    const uint32_t g = d.crossing[1 + item / blocks];
    const int c = (int)(item % blocks) * 32 * C + lane;
    const uint32_t k = key[(uint64_t)g * P + P - 1];
    // the groups behind g that begin with the key, 32 at a time
    uint32_t end = g + 1;
    for (;; end += 32) {
      const uint32_t at = end + lane;
      const uint32_t same = __ballot_sync(0xffffffffu, at < d.groups && key[(uint64_t)at * P] == k);
      if (same != ~0u) {
        end += __ffs(~same) - 1;
        break;
      }
    }
    const uint32_t cnt = end - g;  // parts: group g's second slot, then the first slots
    const uint32_t a = (uint32_t)((uint64_t)cnt * w / 8), b = (uint32_t)((uint64_t)cnt * (w + 1) / 8);
    double sum[C];
#pragma unroll
    for (int e = 0; e < C; ++e) sum[e] = 0.0;
    for (uint32_t i = a; i < b; i += 4) {
      double x[4][C];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < C; ++e)
          x[j][e] = i + j < b && c + 32 * e < d.D ? d.part[((uint64_t)(g + i + j) * 2 + (i + j == 0 ? 1 : 0)) * d.D + c + 32 * e] : 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < C; ++e) sum[e] = __dadd_rn(sum[e], x[j][e]);
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < C; ++e) s[w][32 * e + lane] = sum[e];
    __syncthreads();
    if (threadIdx.x < 32 * C) {
      const int col = (int)(item % blocks) * 32 * C + threadIdx.x;
      if (col < d.D) {
        double all = s[0][threadIdx.x];
        for (int i = 1; i < 8; ++i) all = __dadd_rn(all, s[i][threadIdx.x]);
        T* to = reinterpret_cast<T*>(d.grad) + (int64_t)k * d.tv + (int64_t)col * d.td;
        *to = emb_result<T>(d, all, d.accumulate ? *to : (T)0);
      }
    }
  }
}

// ---- host side -------------------------------------------------------------------

Lanes lanes_for(int chunks) {
  Lanes l;
  l.chunks = chunks;
  l.lg = 0;
  while (l.lg < 8 && (1 << l.lg) < chunks) ++l.lg;
  return l;
}

struct EmbCall {
  const char* fn;
  const trs_view *table, *ids, *rows;  // table: or its gradient; rows: the output, or its gradient
  double scale;
  int accumulate;
};

template <class T, int V>
Error launch_lookup(EmbDev& d, cudaStream_t s) {
  d.l = lanes_for(d.D / V);
  const int64_t per = (kEmbThreads >> d.l.lg) * 4, blocks = ((int64_t)d.N + per - 1) / per;
  emb_lookup_kernel<T, V><<<(unsigned)std::min<int64_t>(blocks, 1 << 20), kEmbThreads, 0, s>>>(d);
  return check_launch("embedding lookup kernel");
}

template <class T, int V>
Error launch_backward(EmbDev& d, cudaStream_t s) {
  d.l = lanes_for(d.D / V);
  int vbits = 1;
  while (vbits < 32 && (d.V >> vbits) != 0) ++vbits;  // keys 0 .. V
  d.digits = (vbits + 8) / 9;
  d.bits = (vbits + d.digits - 1) / d.digits;
  d.tiles = (uint32_t)(((uint64_t)d.N + kSortTile - 1) / kSortTile);
  const int sms = current_device_info().sm_count;
  // as many positions per group as still leave two CTAs of groups per SM, and as fit a CTA's threads
  // (rows below 128 bytes get fewer than 8, so that a frequent token's run comes in many parts, which one
  // CTA finds and adds per 64 columns: 65536 tokens into 50000 rows, a few making up most of them, 64 us
  // for rows of 16 and 127 of 4; all of them one token 420 and 1360)
  d.positions = 32;
  while (d.positions > 8 && (uint64_t)d.N / d.positions < ((uint64_t)2 * sms << 8 >> d.l.lg)) d.positions /= 2;
  while ((d.positions << 8 >> d.l.lg) > kEmbThreads) d.positions /= 2;
  d.groups = (uint32_t)(((uint64_t)d.N + d.positions - 1) / d.positions);
  const size_t n = ((size_t)d.N + 3) / 4 * 4, h = (size_t)d.tiles * kBins;
  Scratch mem, part;
  Error e = mem.alloc(sizeof(uint32_t) * (4 * n + d.digits * h + d.groups + 4), s);
  if (e.ok() && d.N) e = part.alloc(sizeof(double) * 2 * (size_t)d.groups * d.D, s);
  if (!e.ok()) return e;
  uint32_t* at = mem.as<uint32_t>();
  for (int i = 0; i < 2; ++i, at += n) d.key[i] = at;
  for (int i = 0; i < 2; ++i, at += n) d.tok[i] = at;
  for (int i = 0; i < d.digits; ++i, at += h) d.hist[i] = at;
  d.crossing = at;
  d.part = part.as<double>();
  const unsigned zeros = d.accumulate || d.V == 0 ? 0u : 2u * sms;
  if (d.tiles + zeros == 0) return Error{};
  if (d.tiles == 1) {
    auto k = emb_sort_one_kernel<T, V>;
    const int smem = (int)sizeof(SortShared) + 2 * kSortTile * 4;
    allow_smem((const void*)k, smem);
    k<<<1 + zeros, kSortThreads, smem, s>>>(d);
    e = check_launch("embedding sort kernel");
  } else {
    emb_keys_kernel<T, V><<<d.tiles + zeros, kSortThreads, 0, s>>>(d);
    e = check_launch("embedding keys kernel");
    for (int p = 0; e.ok() && p < d.digits; ++p)
      e = launch_after(emb_sort_kernel<T, V>, dim3(d.tiles + zeros), kSortThreads, 0, s, "embedding sort kernel", d, p);
  }
  if (!e.ok() || d.N == 0) return e;
  const unsigned per = kEmbThreads >> d.l.lg;
  e = launch_after(emb_sum_kernel<T, V>, dim3((d.groups + per - 1) / per), kEmbThreads, 0, s, "embedding sum kernel", d);
  if (!e.ok() || d.groups < 2) return e;
  const uint64_t most = (uint64_t)d.groups * ((d.D + 63) / 64);
  return launch_after(emb_join_kernel<T>, dim3((unsigned)std::min<uint64_t>(most, 8u * sms)), 256, 0, s,
                      "embedding join kernel", d);
}

Error run_embedding(const EmbCall& c, bool backward, cudaStream_t stream) {
  const std::string fn = c.fn;
  if (!c.table || !c.ids || !c.rows) return make_error(TRS_ERR_ARG, fn + ": null view");
  Error e = validate_view(c.table, backward ? "the table's gradient" : "the table");
  if (!e.ok()) return e;
  e = validate_view(c.ids, "ids");
  if (!e.ok()) return e;
  if (c.ids->ndim < 1 || c.ids->ndim > 2)
    return make_error(TRS_ERR_SHAPE, fn + ": ids must be [tokens] or [batch, tokens]");
  const Tokens t = tokens_of(c.ids, c.ids->ndim);
  e = check_tokens(fn, c.rows, t, 1, backward ? "the output gradient" : "the output");
  if (!e.ok()) return e;
  if (c.table->ndim != 2) return make_error(TRS_ERR_SHAPE, fn + ": the table must be [vocabulary, width]");
  if (c.rows->shape[t.lead] != c.table->shape[1])
    return make_error(TRS_ERR_SHAPE, fn + ": rows and table must agree in width");
  if (c.ids->dtype != TRS_I32 && c.ids->dtype != TRS_I64)
    return make_error(TRS_ERR_DTYPE, fn + ": ids must be i32 or i64");
  const int dt = c.table->dtype;
  if (dt != TRS_F32 && dt != TRS_F64) return make_error(TRS_ERR_DTYPE, fn + ": the table must be f32 or f64");
  if (c.rows->dtype != dt) return make_error(TRS_ERR_DTYPE, fn + ": rows and table must agree in dtype");
  const int64_t lim = (1ll << 31) - 8192;
  const int64_t V = c.table->shape[0], D = c.table->shape[1];
  if (t.B >= lim || t.T >= lim || t.n() >= lim || V >= lim || D >= lim)
    return make_error(TRS_ERR_SHAPE, fn + ": 2^31 or more tokens, rows or elements of a row");
  e = backward ? check_outputs(fn, {c.table}, {c.rows, c.ids}) : check_outputs(fn, {c.rows}, {c.table, c.ids});
  if (!e.ok()) return e;
  if (D == 0 || (backward ? V == 0 : t.n() == 0)) return Error{};
  EmbDev d;
  std::memset(static_cast<void*>(&d), 0, sizeof(d));
  const int es = dtype_size(dt);
  d.table = static_cast<char*>(c.table->data) + c.table->offset * es;
  d.grad = const_cast<char*>(d.table);
  d.tv = c.table->strides[0];
  d.td = c.table->strides[1];
  d.ids = rows_dev(c.ids, t);
  d.rows = rows_dev(c.rows, t);
  d.ids64 = c.ids->dtype == TRS_I64;
  d.N = (uint32_t)t.n();
  d.V = (uint32_t)V;
  d.D = (int)D;
  d.f_T = make_fastdiv((uint32_t)std::max<int64_t>(t.T, 1));
  d.scale = c.scale;
  const double size = std::fabs(c.scale);
  d.wide = dt == TRS_F32 && ((size > 0.0 && size < FLT_MIN) || (size > FLT_MAX && size <= DBL_MAX));
  d.accumulate = c.accumulate != 0;
  const bool vec = (V == 0 || rows_vectors(c.table)) && (d.N == 0 || rows_vectors(c.rows));
  if (backward) {
    if (dt == TRS_F32) return vec ? launch_backward<float, 4>(d, stream) : launch_backward<float, 1>(d, stream);
    return vec ? launch_backward<double, 2>(d, stream) : launch_backward<double, 1>(d, stream);
  }
  if (dt == TRS_F32) return vec ? launch_lookup<float, 4>(d, stream) : launch_lookup<float, 1>(d, stream);
  return vec ? launch_lookup<double, 2>(d, stream) : launch_lookup<double, 1>(d, stream);
}

trs_status finish(const Error& e) {
  if (!e.ok()) set_last_error(e.msg);
  return e.status;
}

// Nothing thrown leaves a C entry.
template <class F>
trs_status guarded(F f) {
  try {
    return finish(f());
  } catch (...) {
    try {
      set_last_error("out of host memory");
    } catch (...) {
    }
    return TRS_ERR_OOM;
  }
}

}  // namespace
}  // namespace trs

using namespace trs;

extern "C" {

trs_status trs_embedding(const trs_view* table, const trs_view* ids, double scale, trs_view* out, trs_stream stream) {
  return guarded([&] {
    return run_embedding(EmbCall{"embedding", table, ids, out, scale, 0}, false, static_cast<cudaStream_t>(stream));
  });
}

trs_status trs_embedding_backward(const trs_view* grad_out, const trs_view* ids, double scale, int32_t accumulate,
                                  trs_view* grad_table, trs_stream stream) {
  return guarded([&] {
    return run_embedding(EmbCall{"embedding_backward", grad_table, ids, grad_out, scale, accumulate}, true,
                         static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
