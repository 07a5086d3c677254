// head_tc.cu -- a model's last layer with its loss on the 5th-generation tensor
// cores, for more or wider rows than head_few.cu takes.
//
// Products.  f32 operands are written 2^e (hi + lo) with hi and lo in fp16, 11
// bits each, e placing the largest magnitude in [2^14, 2^15): of a hidden row,
// of 256 rows of the weight, of 256 rows of g h.  A product is hi hi + (hi lo + lo
// hi), three tcgen05.mma with f32 accumulation.  The gradient of the scores
// without the row's own factor, softmax(x) - t, lies in [-1, 1] and is split under
// the fixed 2^15, off by 2^-40 at most: a tile's largest is known only when the tile
// is, and is near 1 wherever a target lies in it.  dh, whose terms sum up to softmax
// - t near 1, does not notice; rows of dw whose tokens are all improbable do (p of
// 2^-21: 2e-5 of the row, 2^-29: 1e-3, 2^-40: nothing left).  The factor g temperature
// goes into g h for dw and onto the rows of dh, so that rows with very different
// gradients keep their digits.
// The tensor core cuts its sums instead of rounding them, so a sum leaves the
// accumulator for f32 registers every 256 elements.
//
//   head_pack_kernel  the planes [hi, lo] of hidden rows (those with a target,
//                     gathered), of a piece of the weight and of g h
//   head_gemm_kernel  persistent CTA pairs, 256 x 256 tiles: a warp streams
//                     64-element slabs of both operands by TMA, one warp issues
//                     the MMAs of the pair (tcgen05 cta_group::2: each CTA holds
//                     half of A and half of B, and its 128 rows of the result),
//                     two warpgroups add what leaves the accumulator and finish
//                     the tile:
//       kScores       statistics of each row over the tile (HeadPart)
//       kScoreGrad    softmax(x) - t, split, into planes
//       kProducts     dw = dx^T h and dh = dx w from those planes, the contraction
//                     along the rows of both (MN-major operands)
//
// The vocabulary is taken in pieces, so that the planes of the weight and of dx
// stay small; dh collects the pieces in their order.  No atomics add values.
//
// Measured (B200, cold caches, f32 products a second): scores of 2048 rows on 32000
// x 1024 249 us, 540 TFLOP/s, the tensor pipe busy 89 % of the time at 1.5 GHz: power
// bounds it; with the gradient's planes 272 us (81 %); dw and dh 596 us, 450 TFLOP/s
// (74 %).  In a step of 8192 rows on 50000 x 2048 at the power limit 427 TFLOP/s in
// all, 1.28 PFLOP/s of fp16 products (0.91 of the sustained rate of plain ones).
//
// Every wait is bounded; a CTA whose wait runs out sets the async-error word,
// lets its copies and MMAs end, frees its tensor memory and returns.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <string>

#include "head.h"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace trs {
namespace {

// a b c, in an order in which no step leaves the range when the product does not
__device__ __forceinline__ float mul3(float a, float b, float c) {
  const float x = fabsf(a), y = fabsf(b), z = fabsf(c);
  if (x > y) return y > z ? a * c * b : x > z ? a * b * c : b * c * a;
  return x > z ? b * c * a : y > z ? a * b * c : a * c * b;
}

// ---- planes ---------------------------------------------------------------------

struct PlanesDev {
  HeadDev d;
  __half* to;            // [2][rows][Dp]
  __half* gto;           // hidden rows with a gradient: the planes of g temperature h, alike
  int64_t plane;         // elements of a plane
  int Dp;                // the width rounded up to whole slabs of 64
  float* down;           // 2^e: hidden rows: of every row; weight: of every 256 rows
  float* gdown;          // g h: of every 256 rows
  int v0, n;             // weight: the piece's first row and its rows
  int along_v;           // weight: tokens are the denser dimension
};

// 2^k and 2^-k that bring a largest magnitude (its bits) into [2^14, 2^15),
// within what an f32 holds.
__device__ __forceinline__ void plane_scale(uint32_t top, float* up, float* down) {
  int k = 14 - ((int)(top >> 23) - 127);
  k = k > 126 ? 126 : k < -126 ? -126 : k;
  *up = __uint_as_float((uint32_t)(k + 127) << 23);
  *down = __uint_as_float((uint32_t)(127 - k) << 23);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t magnitude(const float4& x) {
  return max(max(magnitude(x.x), magnitude(x.y)), max(magnitude(x.z), magnitude(x.w)));
}

__device__ __forceinline__ void split_store(__half* to, int64_t plane, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 back = __half22float2(h);
  *reinterpret_cast<__half2*>(to) = h;
  *reinterpret_cast<__half2*>(to + plane) = __floats2half2_rn(a - back.x, b - back.y);
}
__device__ __forceinline__ void split_store(__half* to, int64_t plane, float a, float b, float c, float e) {
  const float v[4] = {a, b, c, e};
  __half h[4], l[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    h[j] = __float2half_rn(v[j]);
    l[j] = __float2half_rn(v[j] - __half2float(h[j]));
  }
  *reinterpret_cast<uint2*>(to) = *reinterpret_cast<uint2*>(h);
  *reinterpret_cast<uint2*>(to + plane) = *reinterpret_cast<uint2*>(l);
}

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address, in the cluster's shared memory, of `p` of CTA `rank`
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}

// Planes of 256 rows by a cluster of 8 CTAs, 32 rows each: the largest
// magnitudes first, which the cluster shares, then the same rows again out of L2.
// Hidden rows (those with a target, gathered; zeros behind the last one up to a
// whole tile) have a power of two each, g h and the weight one per 256 rows: as
// much as the products that contract along the rows keep in the accumulator.
// Bound by HBM: 131 MB of weight in 50 us (262 MB read and written; 98 MB in 42 us).
enum PackKind { kPackWeight, kPackHidden, kPackHiddenGrad };

constexpr int kPackWarps = 16;

template <int KIND>
__device__ __forceinline__ void pack_rows(const PlanesDev& a, int block) {
  constexpr int W = kPackWarps, R = 32 / W;  // R: rows of a warp
  __shared__ uint32_t warp_top[W], tops[8];
  __shared__ float tile[32][33];
  const HeadDev& d = a.d;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t rank = cta_rank();
  const int t256 = block / 8, r0 = block * 32 + warp * R;  // this warp's rows
  if (KIND == kPackHiddenGrad && d.dh.p) {  // rows without a target have no gradient
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (r0 + j >= d.N || d.eid[(int64_t)(r0 + j) * d.K] != kNoToken) continue;
      float* to = head_row<float>(d, d.dh, r0 + j);
      for (int64_t c = lane; c < d.D; c += 32) to[c * d.dh.sd] = 0.f;
    }
  }
  int rows = a.n;
  if (KIND != kPackWeight) {
    rows = *d.live;
    if (t256 * 256 >= rows) {  // the whole cluster
      if (KIND == kPackHiddenGrad && t256 == 0 && threadIdx.x == 0) a.gdown[0] = 1.f;
      return;
    }
  }
  if (KIND != kPackHidden) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const bool along_v = KIND == kPackWeight && a.along_v;
  const int64_t sd = KIND == kPackWeight ? d.wd : d.hid.sd;
  const bool vec = KIND == kPackWeight ? d.vec_w : d.vec_h;
  const float* p[R];
  float g[R];
  uint32_t top[R], all = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    p[j] = nullptr;
    g[j] = 0.f;
    top[j] = 0;
    if (r0 + j >= rows) continue;
    if (KIND == kPackWeight) {
      p[j] = d.w + (int64_t)(a.v0 + r0 + j) * d.wv;
    } else {
      const int row = d.rows[r0 + j];
      p[j] = head_row<const float>(d, d.hid, row);
      if (KIND == kPackHiddenGrad) g[j] = *head_row<const float>(d, d.gl, row) * d.temp;
    }
  }
  constexpr int B = 4;  // 16-byte loads of each row in flight
  auto load = [&](int j, int c) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (p[j] && c < d.D)
      asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(p[j] + c));
    return x;
  };
  if (along_v) {
    const int v = block * 32 + lane;
    const float* w = d.w + (int64_t)(a.v0 + v) * d.wv;
    if (v < rows)
#pragma unroll 4
      for (int c = warp; c < d.D; c += W) all = max(all, magnitude(w[c * d.wd]));
  } else {
    if (!vec) {  // element by element, the lanes side by side
#pragma unroll 8
      for (int c = lane; c < d.D; c += 32)
#pragma unroll
        for (int j = 0; j < R; ++j) top[j] = max(top[j], p[j] ? magnitude(p[j][c * sd]) : 0u);
    }
    for (int c = lane * 4; vec && c < d.D; c += 128 * B) {
      float4 x[B][R];
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int j = 0; j < R; ++j) x[b][j] = load(j, c + 128 * b);
#pragma unroll
      for (int b = 0; b < B; ++b)
#pragma unroll
        for (int j = 0; j < R; ++j) top[j] = max(top[j], magnitude(x[b][j]));
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      top[j] = __reduce_max_sync(0xffffffffu, top[j]);
      all = max(all, KIND == kPackHiddenGrad ? magnitude(g[j] * __uint_as_float(top[j])) : top[j]);
    }
  }
  float up = 1.f, down = 1.f;  // of the 256 rows
  if (KIND != kPackHidden) {
    all = __reduce_max_sync(0xffffffffu, all);
    if (lane == 0) warp_top[warp] = all;
    __syncthreads();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all eight CTAs run
    if (threadIdx.x < 8) {
      uint32_t x = warp_top[0];
      for (int i = 1; i < W; ++i) x = max(x, warp_top[i]);
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr(&tops[rank], threadIdx.x)), "r"(x) : "memory");
    }
    cluster_sync();
    all = tops[0];
    for (int i = 1; i < 8; ++i) all = max(all, tops[i]);
    plane_scale(all, &up, &down);
    if (rank == 0 && threadIdx.x == 0) (KIND == kPackWeight ? a.down : a.gdown)[t256] = down;
  }
  if (along_v) {  // 32 x 32 tiles through shared memory
    const int v = block * 32;
    for (int c0 = 0; c0 < a.Dp; c0 += 32) {
      __syncthreads();
      for (int i = warp; i < 32; i += W)
        tile[i][lane] = v + lane < rows && c0 + i < d.D ? d.w[(int64_t)(a.v0 + v + lane) * d.wv + (c0 + i) * d.wd] : 0.f;
      __syncthreads();
      const int r = threadIdx.x / 8, c = threadIdx.x % 8 * 4;
      if (threadIdx.x < 256 && v + r < rows)
        split_store(a.to + (int64_t)(v + r) * a.Dp + c0 + c, a.plane, tile[c][r] * up, tile[c + 1][r] * up, tile[c + 2][r] * up,
                    tile[c + 3][r] * up);
    }
    return;
  }
  float ups[R];
#pragma unroll
  for (int j = 0; j < R; ++j) ups[j] = up;
  if (KIND != kPackWeight) {
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float dn;
      plane_scale(top[j], &ups[j], &dn);
      if (lane == 0) a.down[r0 + j] = dn;
    }
  }
  if (!vec) {  // pairs of elements
#pragma unroll 8
    for (int c = lane * 2; c < a.Dp; c += 64) {
      float2 x[R];
#pragma unroll
      for (int j = 0; j < R; ++j) x[j] = make_float2(p[j] && c < d.D ? p[j][c * sd] : 0.f, p[j] && c + 1 < d.D ? p[j][(c + 1) * sd] : 0.f);
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (KIND == kPackWeight && !p[j]) continue;
        const int64_t at = (int64_t)(r0 + j) * a.Dp + c;
        split_store(a.to + at, a.plane, x[j].x * ups[j], x[j].y * ups[j]);
        if (KIND == kPackHiddenGrad && a.gto) split_store(a.gto + at, a.plane, mul3(x[j].x, g[j], up), mul3(x[j].y, g[j], up));
      }
    }
    return;
  }
  for (int c0 = lane * 4; c0 < a.Dp; c0 += 128 * B) {
    float4 x[B][R];
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int j = 0; j < R; ++j) x[b][j] = load(j, c0 + 128 * b);
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const int c = c0 + 128 * b;
        if (c >= a.Dp || (KIND == kPackWeight && !p[j])) continue;
        const int64_t at = (int64_t)(r0 + j) * a.Dp + c;
        const float4 y = x[b][j];
        split_store(a.to + at, a.plane, y.x * ups[j], y.y * ups[j], y.z * ups[j], y.w * ups[j]);
        if (KIND == kPackHiddenGrad && a.gto)
          split_store(a.gto + at, a.plane, mul3(y.x, g[j], up), mul3(y.y, g[j], up), mul3(y.z, g[j], up), mul3(y.w, g[j], up));
      }
  }
}

// The hidden rows (clusters below `hidden`, HKIND; none: a later piece) next to a
// piece of the weight.
template <int HKIND>
__global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(kPackWarps * 32)
head_pack_kernel(const __grid_constant__ PlanesDev h, const __grid_constant__ PlanesDev w, int hidden) {
  pdl_launch_dependents();
  // next to the hidden rows the weight does not need the call's kernels before it, the first of which lets others begin
  // only when all that came before the call has ended (kernels of another thread's call may lie between; the memory
  // written here was taken before either)
  if ((int)blockIdx.x < hidden || hidden == 0) pdl_wait();
  if ((int)blockIdx.x < hidden) pack_rows<HKIND>(h, blockIdx.x);
  else pack_rows<kPackWeight>(w, blockIdx.x - hidden);
}

// ---- pieces of the pair's plumbing ---------------------------------------------------

constexpr int CG = 2;                        // CTAs of a pair
constexpr int BM = 128 * CG, BN = 256;       // a tile of the pair
constexpr int BR = BN / CG;                  // B's rows in each CTA
constexpr int kSlab = 64;                    // elements of the contraction per stage
constexpr int kABytes = 2 * 128 * 128, kBBytes = 2 * BR * 128;
constexpr int kStage = kABytes + kBBytes;
constexpr int kStages = 3;
constexpr int kChunk = 4;                    // slabs per accumulator: the 256 rows that share a power of two
constexpr int kGemmThreads = 384;
constexpr int kWarpBuf = 32 * 128;           // a warp's buffer: 128 bytes of 32 rows
constexpr int kGemmSmem = kStages * kStage + 8 * kWarpBuf + 1024 + 256;
constexpr int kLean = 56, kFull = 224;       // 128 * 56 + 256 * 224 = 384 * 168 registers
static_assert(128 * kLean + 256 * kFull == kGemmThreads * 168, "all of the registers");

// (Release at the CTA's scope: what it says is read lies in tensor memory, and its
// loads have completed; at the cluster's scope it would wait for the stores of the
// tile before.)
__device__ __forceinline__ void pair_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D (+)= A B of the pair, issued by the lane of the first CTA with lead != 0.
__device__ __forceinline__ void pair_mma(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kSw128High), "r"(lead)
      : "memory");
}
// Arrives on `bar` of both CTAs once the MMAs issued before have completed.
__device__ __forceinline__ void pair_commit(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(lead), "h"((uint16_t)3)
      : "memory");
}
// Loads into this CTA's shared memory that complete on a barrier of the pair's
// first CTA.
__device__ __forceinline__ void pair_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void pair_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
      "%5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// Waits for a phase, bounded, or until some role of the CTA has given up.
__device__ __forceinline__ bool wait_or_fail(uint64_t* bar, uint32_t parity, int* failed) {
  for (uint32_t i = 0; i < kWaitIters; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 63 && *(volatile int*)failed) return false;
  }
  atomicExch(failed, 1);
  return false;
}

// ---- the matrix products --------------------------------------------------------------

enum HeadMode { kScores, kScoreGrad, kProducts };

struct GemmDev {
  HeadDev d;
  int v0, Vc, Vcp;       // the piece of the vocabulary, rounded up to whole tiles
  const float* hdown;    // 2^e: of the hidden rows
  const float* wdown;    // of every 256 rows of the piece
  const float* gdown;    // of every 256 rows of g h
  HeadPart* part;        // kScores: [column half tile][ld]
  __half* dx;            // kScoreGrad: [2][Np][ld]
  int64_t ld, plane;
  // kProducts
  int dtiles;            // tiles along the width
  int splits, slabs;     // parts of dh's contraction and their slabs
  int wsplits, wslabs;   // of dw's
  int dh_first;
  float *dh_part, *dw_part;  // [split][rows of whole tiles][dtiles * 256] where there are several
  int add;               // dh collects an earlier piece
  int* err;
};

// A tile: rows from m0, columns from n0, `n` slabs of the contraction from k0.
struct GemmItem {
  int m0, n0, k0, n, split;
  int cols;              // of the tile: 256, or 128
  bool dw;
};

// Scores: tiles that are left over by whole rounds of all pairs are taken in halves
// of 128 columns where those fit one round (250 tiles over 74 pairs: 58 us, so 55; a
// step of 6 tiles of 2688 elements 205 us, so 162).
__device__ __forceinline__ int gemm_halved(int tiles, int pairs) {
  const int rest = tiles % pairs;
  return 2 * rest <= pairs ? rest : 0;
}

template <int MODE>
__device__ __forceinline__ int gemm_items(const GemmDev& g, int live, int pairs) {
  const int mt = (live + BM - 1) / BM, vt = g.Vcp / BN;
  if (MODE != kProducts) return mt * vt + gemm_halved(mt * vt, pairs);
  return (g.d.dh.p ? mt * g.dtiles * g.splits : 0) + (g.d.dw ? vt * g.dtiles * g.wsplits : 0);
}

template <int MODE>
__device__ __forceinline__ GemmItem gemm_item(const GemmDev& g, int live, int item, int pairs) {
  const int mt = (live + BM - 1) / BM, vt = g.Vcp / BN;
  GemmItem w;
  w.k0 = 0;
  w.split = 0;
  w.dw = false;
  w.cols = BN;
  auto place = [&](int i, int rows, int cols) {  // groups of 8 row tiles, their columns in order
    const int group = i / (8 * cols), first = group * 8, high = min(8, rows - first);
    const int at = i - group * 8 * cols;
    w.m0 = (first + at % high) * BM;
    w.n0 = at / high * BN;
  };
  if (MODE != kProducts) {
    const int whole = mt * vt - gemm_halved(mt * vt, pairs), over = item - whole;
    place(over < 0 ? item : whole + over / 2, mt, vt);
    if (over >= 0) {
      w.n0 += over % 2 * (BN / 2);
      w.cols = BN / 2;
    }
    w.n = (g.d.D + kSlab - 1) / kSlab;
    return w;
  }
  const int nh = g.d.dh.p ? mt * g.dtiles * g.splits : 0, nw = g.d.dw ? vt * g.dtiles * g.wsplits : 0;
  bool dh = g.dh_first ? item < nh : item >= nw;
  const int i = dh ? item - (g.dh_first ? 0 : nw) : item - (g.dh_first ? nh : 0);
  if (dh) {
    const int tiles = mt * g.dtiles;
    w.split = i / tiles;
    place(i % tiles, mt, g.dtiles);
    const int all = (g.Vc + kSlab - 1) / kSlab;
    w.k0 = min(all, w.split * g.slabs);
    w.n = min(all, w.k0 + g.slabs) - w.k0;
  } else {
    const int tiles = vt * g.dtiles;
    w.split = i / tiles;
    place(i % tiles, vt, g.dtiles);
    w.dw = true;
    const int all = (live + kSlab - 1) / kSlab;
    w.k0 = min(all, w.split * g.wslabs);
    w.n = min(all, w.k0 + g.wslabs) - w.k0;
  }
  if (g.d.D - w.n0 <= BN / 2) w.cols = BN / 2;
  return w;
}

__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pk(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void upk(uint64_t x, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// 128 bytes of each of 32 rows through a warp's buffer, so that a store writes whole
// lines: a lane puts in its row, 16 bytes at a time, in an order by its row that
// keeps both sides free of bank conflicts.  (A tile of 256 x 256 takes 4 to 8 us
// when all pairs write at once, 12 us where rows lie off 16 bytes.)
__device__ __forceinline__ void rows_put(float* buf, int lane, const uint32_t (&x)[32]) {
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 8; ++u)
    reinterpret_cast<uint4*>(buf)[lane * 8 + (u ^ (lane & 7))] = make_uint4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
  __syncwarp();
}
__device__ __forceinline__ uint4 rows_get(const float* buf, int r, int u) {
  return reinterpret_cast<const uint4*>(buf)[r * 8 + (u ^ (r & 7))];
}

// A row's entries inside a tile, rows of the warp one after another, a row's
// entries 32 at a time: its scores (or, for the gradient, its target weights) meet
// them in the warp's buffer.  `e`: this thread's row's first entry not below
// `first`, `id` its token; entries below `end` belong to the tile.
template <bool GRAD>
__device__ __forceinline__ float tile_entries(const HeadDev& d, float* buf, int lane, int orig, int e, int id, int first,
                                              int end, float (&acc)[128]) {
  float dot = 0.f;
  uint32_t hits = __ballot_sync(0xffffffffu, id < end);
  while (hits) {
    const int r = __ffs(hits) - 1;
    hits &= hits - 1;
    const int64_t row = (int64_t)__shfl_sync(0xffffffffu, orig, r) * d.K;
    const int e0 = __shfl_sync(0xffffffffu, e, r);
    float4* b4 = reinterpret_cast<float4*>(buf);
    if (GRAD) {
      b4[lane] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else if (lane == r) {
#pragma unroll
      for (int i = 0; i < 32; ++i) b4[i] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
    }
    __syncwarp();
    float sum = 0.f;
    for (int at = e0 + lane;; at += 32) {
      const int v = at < d.K ? d.eid[row + at] : kNoToken;
      if (v < end) {
        const float t = d.ew[row + at];
        // of a token that comes twice, all but the first add 0: any order gives one result
        if (GRAD) atomicAdd(&buf[v - first], t);
        else if (t != 0.f) sum = __fmaf_rn(t, buf[v - first], sum);
      }
      if (!__all_sync(0xffffffffu, v < end)) break;
    }
    __syncwarp();
    if (GRAD) {
      if (lane == r) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float4 t = b4[i];
          acc[4 * i] -= t.x, acc[4 * i + 1] -= t.y, acc[4 * i + 2] -= t.z, acc[4 * i + 3] -= t.w;
        }
      }
    } else {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == r) dot = sum;
    }
    __syncwarp();
  }
  return dot;
}

// What a thread of the results' warpgroups knows of its row of a tile.
struct TileRow {
  int row, col;          // the tile's row and first column of this thread
  int orig;              // the token of the row
  int e, id;             // its first entry not below the column, and that entry's token
  float f, lse2;
};

// The finished tile's 128 columns of this thread's row.
template <int MODE>
__device__ __forceinline__ void finish_tile(const GemmDev& g, const GemmItem& w, int live, const TileRow& t, float* buf,
                                            int lane, float (&acc)[128]) {
  const HeadDev& d = g.d;
  const int row = t.row, col = t.col;
  if (MODE == kScores) {
    const int limit = g.Vc - col;
    if (limit < 128) {
#pragma unroll
      for (int i = 0; i < 128; ++i)
        if (i >= limit) acc[i] = -INFINITY;
    }
    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 128; i += 2) mx4[i / 2 % 4] = fmaxf(fmaxf(mx4[i / 2 % 4], acc[i]), acc[i + 1]);
    HeadPart p;
    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
    p.m = mx * t.f;
    const float base = p.m == -INFINITY ? 0.f : -p.m;
    // Exponents are products less the rounded largest one.  What that was rounded by stays
    // in the sum while it is small, and is taken out where the exponential would not bear
    // it (scores near 2^43: up to 2^19).
    const float off = fabsf(p.m) >= 0x1p20f && fabsf(p.m) < INFINITY ? __fmaf_rn(mx, t.f, base) : 0.f;
    float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 128; ++i) s4[i % 4] += head_ex2(__fmaf_rn(acc[i], t.f, base) - off);
    p.s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    p.dot = tile_entries<false>(d, buf, lane, t.orig, t.e, t.id, g.v0 + col, g.v0 + col + min(limit, 128), acc) * t.f;
    p.sum = 0.f;
    if (d.share != 0.f) {
      float t4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 128; ++i)
        if (i < limit) t4[i % 4] += acc[i];
      p.sum = ((t4[0] + t4[1]) + (t4[2] + t4[3])) * t.f;
    }
    if (row < live) *reinterpret_cast<float4*>(&g.part[(int64_t)((g.v0 + col) / 128) * g.ld + row]) =
        make_float4(p.m, p.s, p.dot, p.sum);
  } else if (MODE == kScoreGrad) {
    const int limit = row < live ? g.Vc - col : 0;
#pragma unroll
    for (int i = 0; i < 128; ++i) acc[i] = head_softmax(__fmaf_rn(acc[i], t.f, -t.lse2)) - d.share;
    tile_entries<true>(d, buf, lane, t.orig, t.e, t.id, g.v0 + col, g.v0 + col + min(g.Vc - col, 128), acc);
    __half* to = g.dx + (int64_t)(row - lane) * g.ld + col;  // the warp's first row
#pragma unroll
    for (int i = 0; i < 128; i += 64) {
      uint32_t hi[32], lo[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float a = i + 2 * j < limit ? acc[i + 2 * j] * 0x1p15f : 0.f;
        const float b = i + 2 * j + 1 < limit ? acc[i + 2 * j + 1] * 0x1p15f : 0.f;
        const __half2 h = __floats2half2_rn(a, b);
        const float2 back = __half22float2(h);
        const __half2 l = __floats2half2_rn(a - back.x, b - back.y);
        hi[j] = *reinterpret_cast<const uint32_t*>(&h);
        lo[j] = *reinterpret_cast<const uint32_t*>(&l);
      }
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        rows_put(buf, lane, p ? lo : hi);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int r = q * 4 + lane / 8;
          *reinterpret_cast<uint4*>(to + p * g.plane + r * g.ld + i + lane % 8 * 8) = rows_get(buf, r, lane % 8);
        }
      }
    }
  } else {
    float* to = nullptr;   // the row's column col
    int64_t sd = 1, step = 0;  // step: from row to row, where that is one number
    bool vec, add = false;
    float f2 = 1.f;
    const int width = min(128, d.D - col), row0 = row - lane;  // row0: the warp's first row
    int rows;
    if (w.dw) {
      to = d.dw + (int64_t)(g.v0 + row) * d.dwv + (int64_t)col * d.dwd;
      step = d.dwv;
      sd = d.dwd;
      vec = d.vec_dw;
      rows = g.Vc - row0;
      if (g.wsplits > 1) {
        step = (int64_t)g.dtiles * BN;
        sd = 1;
        to = g.dw_part + ((int64_t)w.split * g.Vcp + row) * step + col;
        vec = true;
      }
    } else {
      rows = live - row0;
      if (row < live) f2 = *head_row<const float>(d, d.gl, t.orig) * d.temp;
      if (g.splits > 1) {
        const int64_t np = (live + BM - 1) / BM * BM;
        step = (int64_t)g.dtiles * BN;
        to = g.dh_part + (w.split * np + row) * step + col;
        vec = true;
      } else {
        sd = d.dh.sd;
        vec = d.vec_dh;
        add = g.add;
        if (row < live) to = head_row<float>(d, d.dh, t.orig) + col * sd;
      }
    }
    if (width <= 0 || rows <= 0) return;
    if (sd == 1) {  // through the warp's buffer: whole lines of 128 bytes of each row
      float* first = to - lane * step;
#pragma unroll
      for (int i = 0; i < 128; i += 32) {
        if (i >= width) continue;
        uint32_t x[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(acc[i + j] * f2);
        rows_put(buf, lane, x);
        if (vec) {
          const int c = i + lane % 8 * 4;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int r = q * 4 + lane / 8;
            float* p = step ? first + r * step : reinterpret_cast<float*>(__shfl_sync(0xffffffffu, (unsigned long long)to, r));
            if (r >= rows || c >= width) continue;
            const uint4 y = rows_get(buf, r, lane % 8);
            float4 z = make_float4(__uint_as_float(y.x), __uint_as_float(y.y), __uint_as_float(y.z), __uint_as_float(y.w));
            if (add) {
              const float4 b = *reinterpret_cast<const float4*>(p + c);
              z.x += b.x, z.y += b.y, z.z += b.z, z.w += b.w;
            }
            *reinterpret_cast<float4*>(p + c) = z;
          }
        } else {
          const int c = i + lane;
#pragma unroll 8
          for (int r = 0; r < 32; ++r) {
            float* p = step ? first + r * step : reinterpret_cast<float*>(__shfl_sync(0xffffffffu, (unsigned long long)to, r));
            if (r >= rows || c >= width) continue;
            const float z = buf[(r * 8 + (lane / 4 ^ (r & 7))) * 4 + lane % 4];
            p[c] = add ? p[c] + z : z;
          }
        }
      }
    } else {  // columns apart: the rows lie closer
      if (lane >= rows) return;
#pragma unroll
      for (int i = 0; i < 128; ++i) {
        if (i >= width) continue;
        const float x = acc[i] * f2;
        to[i * sd] = add ? to[i * sd] + x : x;
      }
    }
  }
}

template <int MODE>
__global__ void __cluster_dims__(CG, 1, 1) __launch_bounds__(kGemmThreads, 1)
head_gemm_kernel(const __grid_constant__ CUtensorMap ma, const __grid_constant__ CUtensorMap mb,
                 const __grid_constant__ CUtensorMap ma2, const __grid_constant__ CUtensorMap mb2,
                 const __grid_constant__ GemmDev g) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* bufs = reinterpret_cast<float*>(smem + kStages * kStage);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kStages * kStage + 8 * kWarpBuf);  // of the first CTA: both CTAs' slabs are there
  uint64_t* empty = full + kStages;   // of each CTA: the pair's MMAs have read the stage
  uint64_t* tfull = empty + kStages;  // [2] of each CTA: an accumulator is complete
  uint64_t* tempty = tfull + 2;       // [2] of the first CTA: both CTAs' warps have read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cta_rank();

  if (threadIdx.x == 32) {
    for (const CUtensorMap* m : {&ma, &mb, &ma2, &mb2})
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], CG * 8);
    }
    *failed = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) pair_tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA's barriers are there before anything arrives on them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();  // everything from here on reads what earlier kernels wrote
  const int live = *g.d.live;
  const int pairs = gridDim.x / CG, pair = blockIdx.x / CG, items = gemm_items<MODE>(g, live, pairs);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kLean));
    if (warp == 9 && lane == 0) {  // TMA
      int li = 0;
      bool ok = true;
      for (int item = pair; item < items && ok; item += pairs) {
        const GemmItem w = gemm_item<MODE>(g, live, item, pairs);
        for (int i = 0; i < w.n; ++i, ++li) {
          const int s = li % kStages;
          if (li >= kStages && !(ok = wait_or_fail(&empty[s], (uint32_t)(li / kStages - 1) & 1u, failed))) break;
          if (rank == 0) mbar_arrive_expect_tx(&full[s], CG * kStage);
          const uint32_t bar = cluster_addr(&full[s], 0);
          unsigned char* a = smem + s * kStage;
          const int k = (w.k0 + i) * kSlab, m = w.m0 + rank * 128, n = w.n0 + rank * (w.cols / CG);
          if (MODE != kProducts) {
            pair_load_3d(a, &ma, k, m, 0, bar);
            pair_load_3d(a + kABytes, &mb, k, n, 0, bar);
          } else if (w.dw) {
            pair_load_4d(a, &ma2, 0, k, m / 64, 0, bar);
            pair_load_4d(a + kABytes, &mb2, 0, k, n / 64, 0, bar);
          } else {
            pair_load_3d(a, &ma, k, m, 0, bar);
            pair_load_4d(a + kABytes, &mb, 0, k, n / 64, 0, bar);
          }
        }
      }
      // every copy has landed and been read, and the arrival that says so has come,
      // before the CTA ends; after a failure, which tells nothing about the other
      // CTA's copies, they are given time
      for (int s = 0; s < kStages && s < li && ok; ++s)
        ok = wait_or_fail(&empty[s], (uint32_t)((li - 1 - s) / kStages) & 1u, failed);
      if (!ok)
        for (int i = 0; i < 100; ++i) __nanosleep(100000);
    } else if (warp == 8 && rank == 0) {  // MMA: the warp stays whole, one lane issues
      const uint32_t lead = elect_lane(), tm = uniform(tmem);
      auto wait_all = [&](uint64_t* bar, uint32_t phase) {
        return __all_sync(0xffffffffu, wait_or_fail(bar, phase & 1u, failed)) != 0;
      };
      int li = 0, ci = 0;
      bool ok = true;
      for (int item = pair; item < items && ok; item += pairs) {
        const GemmItem w = gemm_item<MODE>(g, live, item, pairs);
        const bool amn = MODE == kProducts && w.dw, bmn = MODE == kProducts;
        const uint32_t idesc = uniform((1u << 4) | (amn ? 1u << 15 : 0u) | (bmn ? 1u << 16 : 0u) |
                                       ((uint32_t)(w.cols >> 3) << 17) | ((uint32_t)(BM >> 4) << 24));
        const uint32_t astep = amn ? 128u : 2u, bstep = bmn ? 128u : 2u;
        const uint32_t da0 = uniform(sw128_low(smem, amn ? 64 * 128 : 16));
        const uint32_t db0 = uniform(sw128_low(smem + kABytes, bmn ? 64 * 128 : 16));
        for (int i = 0; i < w.n && ok; ++i, ++li) {
          const int s = li % kStages;
          if (i % kChunk == 0 && ci >= 2 && !(ok = wait_all(&tempty[ci & 1], (uint32_t)(ci / 2 - 1)))) break;
          if (!(ok = wait_all(&full[s], (uint32_t)(li / kStages)))) break;
          tc_fence_after();
          const uint32_t dst = tm + (ci & 1) * BN;
          const uint32_t a = da0 + s * (kStage / 16), b = db0 + s * (kStage / 16);
          constexpr uint32_t ALO = 128 * 128 / 16, BLO = BR * 128 / 16;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            pair_mma(lead, dst, a + ALO + k * astep, b + k * bstep, idesc, i % kChunk != 0 || k > 0);
            pair_mma(lead, dst, a + k * astep, b + BLO + k * bstep, idesc, 1);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) pair_mma(lead, dst, a + k * astep, b + k * bstep, idesc, 1);
          pair_commit(lead, &empty[s]);
          if (i % kChunk == kChunk - 1 || i + 1 == w.n) {
            pair_commit(lead, &tfull[ci & 1]);
            ++ci;
          }
        }
      }
      // all MMAs are complete before the pair's shared memory and tensor memory go
      if (ci > 0) wait_all(&tfull[(ci - 1) & 1], (uint32_t)((ci - 1) / 2));
    }
  } else {  // results: a row per thread, 128 columns per warpgroup
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFull));
    const int half = warp / 4, rl = (warp % 4) * 32 + lane;
    const uint32_t src = tmem + ((uint32_t)((warp % 4) * 32) << 16) + half * 128;
    const uint32_t bars[2] = {cluster_addr(&tempty[0], 0), cluster_addr(&tempty[1], 0)};
    int ci = 0;
    bool ok = true;
    for (int item = pair; item < items && ok; item += pairs) {
      const GemmItem w = gemm_item<MODE>(g, live, item, pairs);
      TileRow t;
      t.row = w.m0 + (int)rank * 128 + rl;
      t.col = w.n0 + half * 128;
      t.id = kNoToken;
      t.f = t.lse2 = 0.f;
      t.orig = t.e = 0;
      if (!w.dw && t.row < live) {
        t.orig = g.d.rows[t.row];
        if (MODE != kProducts) {
          // a power of two and the factor onto units of log2: neither 0 nor inf
          t.f = fminf(fmaxf(mul3(g.hdown[t.row], g.wdown[w.n0 / BN], g.d.inv_temp * kHeadLog2e), 0x1p-126f), FLT_MAX);
          const int* ids = g.d.eid + (int64_t)t.orig * g.d.K;
          int hi = g.d.K;
          while (t.e < hi) {
            const int mid = (t.e + hi) / 2;
            if (ids[mid] < g.v0 + t.col) t.e = mid + 1; else hi = mid;
          }
          if (t.e < g.d.K) t.id = ids[t.e];
          if (MODE == kScoreGrad) t.lse2 = *head_row<const float>(g.d, g.d.lse, t.orig) * kHeadLog2e;
        }
      }
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      for (int i = 0; i < w.n; i += kChunk, ++ci) {
        // the powers of two of the 256 rows that the chunk contracted along, and of dx
        uint64_t scale2 = 0;
        if (MODE == kProducts) {
          const float f = (w.dw ? g.gdown : g.wdown)[(w.k0 + i) / kChunk] * 0x1p-15f;
          scale2 = pk(f, f);
        }
        ok = __all_sync(0xffffffffu, wait_or_fail(&tfull[ci & 1], (uint32_t)(ci / 2) & 1u, failed)) != 0;
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t x[32];
          tmem_ld32_issue(src + (ci & 1) * BN + cc * 32, x);
          tmem_ld_done(x);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const uint64_t now = pk(acc[cc * 32 + j], acc[cc * 32 + j + 1]), more = pk(__uint_as_float(x[j]), __uint_as_float(x[j + 1]));
            upk(MODE == kProducts ? fma2(more, scale2, now) : add2(now, more), &acc[cc * 32 + j], &acc[cc * 32 + j + 1]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) pair_arrive(bars[ci & 1]);
      }
      if (ok && half * 128 < w.cols) finish_tile<MODE>(g, w, live, t, bufs + warp * (kWarpBuf / 4), lane, acc);
    }
  }
  if (threadIdx.x % 32 == 0 && *(volatile int*)failed) atomicOr(g.err, kAsyncWaitTimeout);
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  if (warp == 0) pair_tmem_dealloc(tmem, 512);
}

// A row of dh, or of dw, from the parts of its contraction, in order.
template <bool DW>
__global__ void __launch_bounds__(256) head_parts_kernel(const __grid_constant__ GemmDev g) {
  pdl_launch_dependents();
  pdl_wait();
  const HeadDev& d = g.d;
  const int live = *d.live, r = blockIdx.x, splits = DW ? g.wsplits : g.splits;
  if (r >= (DW ? g.Vc : live)) return;
  const int64_t rows = DW ? g.Vcp : (live + BM - 1) / BM * BM, ld = (int64_t)g.dtiles * BN;
  const float* part = (DW ? g.dw_part : g.dh_part) + r * ld;
  float* to = DW ? d.dw + (int64_t)(g.v0 + r) * d.dwv : head_row<float>(d, d.dh, d.rows[r]);
  const int64_t sd = DW ? d.dwd : d.dh.sd;
  for (int c = blockIdx.y * 256 + threadIdx.x; c < d.D; c += gridDim.y * 256) {
    float sum = !DW && g.add ? to[c * sd] : 0.f;
    for (int s0 = 0; s0 < splits; s0 += 8) {
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = s0 + k < splits ? part[(s0 + k) * rows * ld + c] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += x[k];
    }
    to[c * sd] = sum;
  }
}

// ---- host side --------------------------------------------------------------------------

Error make_map(const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
               CUtensorMap* map) {
  Error e;
  EncodeTiled enc = encode_fn(&e);
  if (!enc) return e;
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box,
                         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return make_error(TRS_ERR_CUDA, "head: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return Error{};
}

// Planes [2][rows][pitch] whose contraction runs along the pitch: boxes of 64
// elements by `high` rows by both planes.
Error map_rows(const __half* p, int64_t rows, int64_t pitch, int64_t plane, int high, CUtensorMap* map) {
  const cuuint64_t dims[3] = {(cuuint64_t)pitch, (cuuint64_t)rows, 2};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)plane * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)high, 2};
  return make_map(p, 3, dims, strides, box, map);
}
// The same planes with the contraction along the rows: boxes of 64 rows by 128
// columns, as blocks of 64, by both planes.
Error map_cols(const __half* p, int64_t rows, int64_t pitch, int64_t plane, CUtensorMap* map) {
  const cuuint64_t dims[4] = {64, (cuuint64_t)rows, (cuuint64_t)pitch / 64, 2};
  const cuuint64_t strides[3] = {(cuuint64_t)pitch * 2, 128, (cuuint64_t)plane * 2};
  const cuuint32_t box[4] = {64, kSlab, 2, 2};
  return make_map(p, 4, dims, strides, box, map);
}

int max_pairs(const void* kernel) {
  static DeviceCache<const void*> cache;
  const DeviceInfo& info = current_device_info();
  return cache.get(info.device, kernel, [&] {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(info.sm_count / CG * CG));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = kGemmSmem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) == cudaSuccess) return n;
    cudaGetLastError();
    return 0;
  });
}

template <int MODE>
Error launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& a2, const CUtensorMap& b2, const GemmDev& g,
                  int64_t most, cudaStream_t s) {
  auto k = head_gemm_kernel<MODE>;
  allow_smem((const void*)k, kGemmSmem);
  const int64_t pairs = std::min<int64_t>(most, max_pairs((const void*)k));
  if (pairs < 1) return Error{};
  return launch_after(k, dim3((unsigned)(pairs * CG)), kGemmThreads, kGemmSmem, s, "head matrix product kernel", a, b, a2, b2, g);
}

int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

constexpr int64_t kPieceBytes = 512ll << 20;  // planes of a piece

}  // namespace

Error head_tc_plan(const HeadDev& d, bool backward, HeadTcPlan* out) {
  HeadTcPlan& p = *out;
  std::memset(static_cast<void*>(&p), 0, sizeof(p));
  const int sms = current_device_info().sm_count;
  p.Np = round_up(std::max(d.N, 1), BM);
  p.Dp = round_up(d.D, kSlab);
  p.dtiles = (d.D + BN - 1) / BN;
  // pieces of the vocabulary of one size, whole tiles each
  const int64_t row_bytes = 4 * p.Dp + (backward ? 4 * p.Np : 0);
  p.pieces = std::max<int64_t>(1, (round_up(d.V, BN) * row_bytes + kPieceBytes - 1) / kPieceBytes);
  p.Vp = round_up((d.V + p.pieces - 1) / p.pieces, BN);
  p.pieces = (d.V + p.Vp - 1) / p.Vp;
  if (p.Np / BM * std::max(p.Vp / BN, p.dtiles * 64) + p.Vp / BN * p.dtiles >= (1ll << 31))
    return make_error(TRS_ERR_SHAPE, "head: 2^31 or more tiles of 256 x 256");
  p.htiles = p.Np / BM * p.dtiles;
  p.wtiles = p.Vp / BN * p.dtiles;
  p.splits = p.wsplits = 1;
  if (backward && d.N > 0) {
    // few tiles with a long contraction: parts of about a third of a pair's share of the work, 8 slabs at least
    const int64_t work = (d.dh.p ? p.htiles * p.Vp : 0) + (d.dw ? p.wtiles * p.Np : 0);
    const int64_t part = std::max<int64_t>(512, work / std::max(1, sms / CG) / 3);
    if (d.dh.p) p.splits = (int)std::min<int64_t>(64, std::max<int64_t>(1, (p.Vp + part / 2) / part));
    if (d.dw) p.wsplits = (int)std::min<int64_t>(64, std::max<int64_t>(1, (p.Np + part / 2) / part));
  }
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += (size_t)round_up(bytes, 256);
    return here;
  };
  p.wdown = take(4 * (p.Vp * p.pieces / BN));
  p.gdown = take(4 * (p.Np / 256));
  p.hdown = take(4 * p.Np);
  p.h = take(4 * p.Np * p.Dp);
  p.w = take(4 * p.Vp * p.Dp);
  p.gh = take(backward && d.dw ? 4 * p.Np * p.Dp : 0);
  p.x = take(backward ? 4 * p.Np * p.Vp : 0);
  p.part = take(backward ? 0 : (int64_t)sizeof(HeadPart) * (p.Vp * p.pieces / 128) * p.Np);
  p.dh = take(p.splits > 1 ? 4 * p.splits * p.Np * p.dtiles * BN : 0);
  p.dw = take(p.wsplits > 1 ? 4 * p.wsplits * p.Vp * p.dtiles * BN : 0);
  p.bytes = at;
  return Error{};
}

Error head_tc(const HeadDev& d, bool backward, const HeadTcPlan& plan, char* base, cudaStream_t s) {
  const int64_t Np = plan.Np, Dp = plan.Dp, Vp = plan.Vp, pieces = plan.pieces, htiles = plan.htiles, wtiles = plan.wtiles;
  int* err = async_error_word();
  if (!err) return make_error(TRS_ERR_CUDA, "head: no async-error word");
  Error e;
  GemmDev g;
  std::memset(static_cast<void*>(&g), 0, sizeof(g));
  g.d = d;
  g.err = err;
  g.dtiles = (int)plan.dtiles;
  g.splits = plan.splits;
  g.wsplits = plan.wsplits;
  g.slabs = (int)round_up((Vp / kSlab + g.splits - 1) / g.splits, kChunk);
  g.wslabs = (int)round_up((Np / kSlab + g.wsplits - 1) / g.wsplits, kChunk);
  g.dh_first = Vp / g.splits >= d.N;

  const int64_t hplane = Np * Dp, wplane = Vp * Dp, xplane = backward ? Np * Vp : 0;
  __half *hp = reinterpret_cast<__half*>(base + plan.h), *wp = reinterpret_cast<__half*>(base + plan.w);
  __half *gp = reinterpret_cast<__half*>(base + plan.gh), *xp = reinterpret_cast<__half*>(base + plan.x);

  PlanesDev hid, p;
  std::memset(static_cast<void*>(&p), 0, sizeof(p));
  p.d = d;
  p.Dp = (int)Dp;
  hid = p;
  hid.to = hp;
  hid.gto = backward && d.dw ? gp : nullptr;
  hid.plane = hplane;
  hid.down = reinterpret_cast<float*>(base + plan.hdown);
  hid.gdown = reinterpret_cast<float*>(base + plan.gdown);

  g.hdown = reinterpret_cast<float*>(base + plan.hdown);
  g.gdown = hid.gdown;
  g.part = reinterpret_cast<HeadPart*>(base + plan.part);
  g.ld = backward ? Vp : Np;
  g.dx = xp;
  g.plane = xplane;
  g.dh_part = reinterpret_cast<float*>(base + plan.dh);
  g.dw_part = reinterpret_cast<float*>(base + plan.dw);
  g.Vcp = (int)Vp;
  const int64_t av = d.wv < 0 ? -d.wv : d.wv, ad = d.wd < 0 ? -d.wd : d.wd;
  p.along_v = d.V > 1 && d.D > 1 && av < ad;
  for (int64_t i = 0; i < pieces; ++i) {
    g.v0 = (int)(i * Vp);
    g.Vc = (int)std::min<int64_t>(Vp, d.V - i * Vp);
    g.Vcp = (int)round_up(g.Vc, BN);
    g.add = i > 0;
    p.to = wp;
    p.plane = wplane;
    p.down = reinterpret_cast<float*>(base + plan.wdown) + i * (Vp / BN);
    g.wdown = p.down;
    p.v0 = g.v0;
    p.n = g.Vc;
    const int hidden = i == 0 ? (int)(Np / 32) : 0;
    e = launch_after(backward ? head_pack_kernel<kPackHiddenGrad> : head_pack_kernel<kPackHidden>,
                     dim3((unsigned)(hidden + g.Vcp / 32)), kPackWarps * 32, 0, s, "head planes kernel", hid, p, hidden);
    CUtensorMap ha, wb, xa, wc, xc, gc;
    if (e.ok()) e = map_rows(hp, Np, Dp, hplane, 128, &ha);
    if (e.ok()) e = map_rows(wp, g.Vc, Dp, wplane, BR, &wb);
    if (!e.ok()) return e;
    const int64_t tiles = Np / BM * (g.Vcp / BN);
    if (!backward) {
      e = launch_gemm<kScores>(ha, wb, ha, wb, g, 2 * tiles, s);
      if (!e.ok()) return e;
      continue;
    }
    e = launch_gemm<kScoreGrad>(ha, wb, ha, wb, g, 2 * tiles, s);
    if (e.ok()) e = map_rows(xp, Np, Vp, xplane, 128, &xa);
    if (e.ok()) e = map_cols(xp, Np, Vp, xplane, &xc);
    if (e.ok()) e = map_cols(wp, g.Vc, Dp, wplane, &wc);
    gc = wc;
    if (e.ok() && d.dw) e = map_cols(gp, Np, Dp, hplane, &gc);
    if (e.ok()) e = launch_gemm<kProducts>(xa, wc, xc, gc, g, htiles * g.splits + wtiles * g.wsplits, s);
    const unsigned across = (unsigned)std::min<int64_t>(16, (d.D + 255) / 256);
    if (e.ok() && g.splits > 1)
      e = launch_after(head_parts_kernel<false>, dim3((unsigned)d.N, across), 256, 0, s, "head hidden gradient join kernel", g);
    if (e.ok() && g.wsplits > 1)
      e = launch_after(head_parts_kernel<true>, dim3((unsigned)g.Vc, across), 256, 0, s, "head weight gradient join kernel", g);
    if (!e.ok()) return e;
  }
  if (backward) return e;
  return head_join(d, g.part, (int)((d.V + 127) / 128), Np, 1, false, s);
}

}  // namespace trs
