// cross_tc.cu -- cross attention and its gradient on the 5th-generation tensor
// cores, for f32 tensors with head sizes up to 128.
//
// Products.  A tile x of an operand is written x = 2^e (hi + lo) with hi and lo
// in fp16: e places the tile's largest magnitude in [2^14, 2^15), hi is x 2^-e
// rounded to 11 bits and lo the rest rounded to 11 more.  A product is taken
// as hi hi + (hi lo + lo hi), three tcgen05.mma with f32 accumulation; lo lo
// (below 2^-22 of it) is dropped.  Elements down to 2^-17 of the tile's
// largest keep all 22 bits, and below that the error is 2^-40 of the largest:
// an f32 result, at a third of the fp16 rate instead of the CUDA cores' rate.
// P and dS are split the same way in registers, P by the fixed 2^15 of its
// range, dS by a bound on its row (|dout_i| |v_j| + |delta_i|).  The scales of the
// tiles meet in f32 as powers of two, in an order that keeps every step in range.
// The small products of a tile are accumulated before the large ones, and every tile's
// result leaves the accumulator for f32 registers, so that a long sum is not
// carried through the tensor core's own (truncating) additions.
//
//   cross_pack_kernel     splits q, k, v (and dout) into planes [hi, lo] of
//                         [problem][rows][DP], DP = 64 or 128, zeros behind the
//                         last row, key length and head size: strides, ragged
//                         lengths and odd head sizes end here.  Also delta, and
//                         the norms that bound dS.  Bound by HBM: three tensors
//                         of 33.5 MB in 33 us (6.1 TB/s read and written), the
//                         gradient's five in 65 us (4.6).
//   cross_forward_kernel  persistent CTAs; an item is MT = 1 or 2 tiles of 128
//                         query rows, walked over key tiles of KN (128 for DP 64,
//                         64 for DP 128).  A warp streams K and V tiles by TMA
//                         through a ring of 32 KiB slots; a warp per row tile
//                         issues its MMAs; a warpgroup per row tile, one thread
//                         per row, keeps the running maximum and sum of the
//                         softmax, turns S (TMEM) into the two planes of P in
//                         place, and adds O.  The row tiles run half a period
//                         apart: one is in the softmax while the other has the
//                         tensor core.  4 x 16 heads of 64, 2048 x 2048 tokens:
//                         214 us (226 with the split), 320 TFLOP/s of f32
//                         products (960 of fp16, two thirds of the sustained
//                         cuBLAS rate).
//   cross_backward_kernel dq (rows: queries, walking keys) or dk and dv (rows:
//                         keys, walking queries); both need S and dP = dout v^T
//                         of the tile, and write each result once: no atomics,
//                         at the price of computing S and dP twice.  Two
//                         warpgroups share the 128 rows and halve the columns.
//                         The same case: 297 us and 402 us (1040 and 1025
//                         TFLOP/s of fp16 products).
//   cross_join_kernel (cross_attention.cu), cross_sum_kernel
//                         join the parts of a walk that was split over CTAs, in
//                         a fixed order.
//
// What bounds the two tensor-core kernels: the hand-overs between softmax and
// tensor core.  Per 128 x 128 tile the MMAs of the forward take 1560 cycles
// (every product at the full rate), the softmax of a warp 1700, and each of the
// three hand-overs (S, P, O) about 500.
//
// Every wait is bounded; a CTA whose wait runs out sets the async-error word,
// waits (bounded) for its own copies and MMAs, frees its tensor memory and
// returns.
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <string>

#include "cross.h"
#include "cross_exact.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace trs {

Error cross_join(const CrossDev& c, int splits, int rows, int ld, const float* part, const float* part_m,
                 const float* part_l, cudaStream_t stream);

namespace {

constexpr int kSlot = 32 * 1024;             // a streamed tile: KN x DP, two fp16 planes
constexpr int kTileElems = 8192;             // elements of a packed tile (KN rows of DP)

// ---- pack --------------------------------------------------------------------

struct PackSrc {
  HeadsDev x;
  int G, T;              // rows of a problem: G * T
  int keys;              // rows end at the key length
  int rows_p;            // rows of a problem in the planes
  __half *hi, *lo;
  float* inv;            // [problem][tile] 2^e
  float* norm;           // [problem][tile] largest row 2-norm, in units of 2^e; or null
  float sign;
  // the output gradient's tiles also carry, per row: 15 - lse in units of log2
  // (-inf behind the last row: no weight), delta, the row's norm in units of
  // 2^e; per tile the largest |delta|
  int grad;
  HeadsDev out;
  float *bias, *delta, *rnorm, *dmax;
  FastDiv f_T;
};
struct PackDev {
  PackSrc s[4];
  uint32_t first[5];     // first CTA of each source
  int n;
  int Hk, D;
  const void* len;
  int len64;
  int64_t len_s;
  int Tk;
  const float* lse;
  int64_t ls_b, ls_h, ls_t;
  int* nonfinite;
};

template <int L>
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ float block_max(float x, float* sm) {  // 256 threads, x >= 0
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = x;
  __syncthreads();
  x = sm[threadIdx.x % 8];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  return x;
}

template <bool VEC>
__device__ __forceinline__ float4 head4(const float* p, int d, int D, int64_t sd) {
  if (VEC) return *reinterpret_cast<const float4*>(p + d);  // D is a multiple of 4 and d < D
  float4 r;
  r.x = p[d * sd];
  r.y = d + 1 < D ? p[(d + 1) * sd] : 0.f;
  r.z = d + 2 < D ? p[(d + 2) * sd] : 0.f;
  r.w = d + 3 < D ? p[(d + 3) * sd] : 0.f;
  return r;
}

// One CTA per tile of KN = 8192 / DP rows; DP / 4 lanes per row.
template <int DP, bool VEC>
__global__ void __launch_bounds__(256) cross_pack_kernel(const __grid_constant__ PackDev d) {
  constexpr int L = DP / 4, PT = kTileElems / DP, RP = 256 / L, NP = PT / RP;
  __shared__ float sm[8];
  int w = 0;
  while (w + 1 < d.n && blockIdx.x >= d.first[w + 1]) ++w;
  const PackSrc& s = d.s[w];
  const int tiles = s.rows_p / PT;
  const int at = (int)(blockIdx.x - d.first[w]), pr = at / tiles, tile = at % tiles;
  const int b = pr / d.Hk, hk = pr % d.Hk;
  const int n = s.keys ? key_count(d.len, d.len64, d.len_s, d.Tk, b) : s.G * s.T;
  const int lane = threadIdx.x % L, r0 = tile * PT + threadIdx.x / L, dd = lane * 4;
  pdl_launch_dependents();
  float4 x[NP];
  float dl[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = r0 + i * RP;
    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < n && dd < d.D) {
      const int g = (int)fdiv((uint32_t)row, s.f_T), t = row - g * s.T, h = hk * s.G + g;
      x[i] = head4<VEC>(static_cast<const float*>(s.x.p) + b * s.x.sb + t * s.x.st + h * s.x.sh, dd, d.D, s.x.sd);
    }
  }
  if (s.grad) {
    float4 o[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = r0 + i * RP;
      o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < n && dd < d.D) {
        const int g = (int)fdiv((uint32_t)row, s.f_T), t = row - g * s.T, h = hk * s.G + g;
        o[i] = head4<VEC>(static_cast<const float*>(s.out.p) + b * s.out.sb + t * s.out.st + h * s.out.sh, dd, d.D, s.out.sd);
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i)
      dl[i] = __fmaf_rn(x[i].x, o[i].x, __fmaf_rn(x[i].y, o[i].y, __fmaf_rn(x[i].z, o[i].z, x[i].w * o[i].w)));
  }
  float mx = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[i].x), fabsf(x[i].y)), fmaxf(fabsf(x[i].z), fabsf(x[i].w))));
    bad |= !(fabsf(x[i].x) <= 3e38f && fabsf(x[i].y) <= 3e38f && fabsf(x[i].z) <= 3e38f && fabsf(x[i].w) <= 3e38f);
  }
  if (__any_sync(0xffffffffu, bad) && threadIdx.x % 32 == 0) atomicOr(d.nonfinite, 1);
  mx = block_max(mx, sm);
  // up = 2^(14 - exponent of mx), within what an f32 holds; a tile of zeros
  // (and of the smallest magnitudes) takes 2^126
  int e = (int)(__float_as_uint(mx) >> 23) - 127;
  int k = 14 - e;
  k = k > 126 ? 126 : k;
  const float up = __uint_as_float((uint32_t)(k + 127) << 23), down = __uint_as_float((uint32_t)(127 - k) << 23);
  if (threadIdx.x == 0) s.inv[pr * tiles + tile] = down;
  const float us = up * s.sign;
  float nm = 0.f, dm = 0.f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = r0 + i * RP;
    const float v[4] = {x[i].x * us, x[i].y * us, x[i].z * us, x[i].w * us};
    __half h[4], l[4];
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = __float2half_rn(v[j]);
      l[j] = __float2half_rn(v[j] - __half2float(h[j]));
      ss = __fmaf_rn(v[j], v[j], ss);
    }
    const int64_t o = ((int64_t)pr * s.rows_p + row) * DP + dd;
    *reinterpret_cast<uint2*>(s.hi + o) = *reinterpret_cast<uint2*>(h);
    *reinterpret_cast<uint2*>(s.lo + o) = *reinterpret_cast<uint2*>(l);
    if (s.norm) {
      const float rn = sqrtf(lanes_sum<L>(ss));
      nm = fmaxf(nm, rn);
      if (s.grad) {
        const float dlt = lanes_sum<L>(dl[i]);
        dm = fmaxf(dm, fabsf(dlt));
        if (lane == 0) {
          const int64_t at_r = (int64_t)pr * s.rows_p + row;
          float ls = -INFINITY;
          if (row < n) {
            const int g = (int)fdiv((uint32_t)row, s.f_T), t = row - g * s.T;
            ls = d.lse[b * d.ls_b + (hk * s.G + g) * d.ls_h + t * d.ls_t];
            if (ls != -INFINITY) ls = __fmaf_rn(ls, -kLog2e, 15.f);  // scores of -inf alone: no weight either
          }
          s.bias[at_r] = ls;
          s.delta[at_r] = dlt;
          s.rnorm[at_r] = rn;
        }
      }
    }
  }
  if (s.norm) {
    nm = block_max(nm, sm);
    dm = block_max(dm, sm);
    if (threadIdx.x == 0) {
      s.norm[pr * tiles + tile] = nm;
      if (s.grad) s.dmax[pr * tiles + tile] = dm;
    }
  }
}

// ---- shared pieces of the tensor-core kernels ------------------------------------

// Far scores.  A tile's scores (in units of log2) are f x with |x| < 2^30 DP, so
// f alone says how large they can be.
// An exponent 15 + S - m has to stay below 16, what fp16 holds: m and 15 - m are
// off by half a unit of m each, 2^-4 at 2^20.  Above that the forward takes S - m
// from rounded scores, which is 0 for a row's largest (inside the branch that
// cuts off absent keys, where it costs nothing; a branch of its own 2 %, a
// second copy of the loop 7 %).
template <int DP> constexpr float kFarMax = 0x1p-10f / DP;
// S - lse of the gradients, whose S is another sum than the one that lse came
// from: both are off by less than 80 2^-24 of |q| |k|, together 0.7 at 2^16.
// Above that the exponent is cut to that of P = 1.
template <int DP> constexpr float kFarSum = 0x1p-14f / DP;

// a b c, in an order in which no step leaves the range when the product does not:
// the extremes first.  The factors of a tile are powers of two (and the scale).
__device__ __forceinline__ float mul3(float a, float b, float c) {
  const float lo = fminf(fminf(a, b), c), hi = fmaxf(fmaxf(a, b), c);
  return lo * hi * fmaxf(fminf(a, b), fminf(fmaxf(a, b), c));
}

// A packed operand as the kernels see it.
struct Planes {
  int rows_p;            // rows of a problem
  int rows_all;          // rows of all problems: where the lo plane starts
  const float* inv;
  const float* norm;
};

// A warp's arrival: one lane, after the others' work.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if (threadIdx.x % 32 == 0) mbar_arrive(bar);
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

// The same for the MMA warps, without the suspension of try_wait: a hand-over
// to the tensor core is on the path between two tiles.
__device__ __forceinline__ bool spin_or_fail(uint64_t* bar, uint32_t parity, int* failed) {
  for (uint32_t i = 0; i < (1u << 27); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((i & 255) == 255 && *(volatile int*)failed) return false;
  }
  atomicExch(failed, 1);
  return false;
}

// Rows [row, row + ROWS) of a problem, both planes, as [plane][64-column
// block][ROWS][64] with 128-byte swizzle.
template <int DP, int ROWS>
__device__ __forceinline__ void load_planes(unsigned char* dst, const CUtensorMap* map, const Planes& p, int row,
                                            uint64_t* bar) {
#pragma unroll
  for (int pl = 0; pl < 2; ++pl)
#pragma unroll
    for (int h = 0; h < DP / 64; ++h)
      tma_load_2d(dst + (pl * (DP / 64) + h) * ROWS * 128, map, h * 64, pl * p.rows_all + row, bar);
}

// fp16 x fp16 -> f32, M 128, N columns; B K-major, or MN-major (bit 16)
constexpr uint32_t idesc_f16(int n, bool mn) {
  return (1u << 4) | (mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// Head sizes up to DE (64, 96, 128) take the products over DE elements; DP (64,
// 128) is what a row of the planes holds, zeros from the head size on.

// D = A B^T over DE: A 128 rows, B KN rows, both in shared memory (planes as
// load_planes leaves them); the two small products first.
template <int DP, int DE, int KN>
__device__ __forceinline__ void mma_abt(uint32_t lead, uint32_t dst, uint32_t a, uint32_t b) {
  constexpr uint32_t id = idesc_f16(KN, false);
  constexpr int HA = 128 * 128 / 16, HB = KN * 128 / 16, NH = DP / 64;
#pragma unroll
  for (int k = 0; k < DE / 16; ++k) {
    const int ka = k / 4 * HA + k % 4 * 2, kb = k / 4 * HB + k % 4 * 2;
    umma_f16_ss<id>(lead, dst, a + NH * HA + ka, b + kb, k > 0);
    umma_f16_ss<id>(lead, dst, a + ka, b + NH * HB + kb, 1);
  }
#pragma unroll
  for (int k = 0; k < DE / 16; ++k)
    umma_f16_ss<id>(lead, dst, a + k / 4 * HA + k % 4 * 2, b + k / 4 * HB + k % 4 * 2, 1);
}

// D = A B over KN: A 128 x KN in tensor memory (chunks of 32 columns: 16
// columns of hi, 16 of lo), B KN rows of DE columns in shared memory.
template <int DP, int DE, int KN>
__device__ __forceinline__ void mma_ab(uint32_t lead, uint32_t dst, uint32_t a, uint32_t b) {
  constexpr uint32_t id = idesc_f16(DE, true);
  constexpr int LO = DP / 64 * KN * 128 / 16;
#pragma unroll
  for (int k = 0; k < KN / 16; ++k) {
    const uint32_t ak = a + 32 * (k / 2) + 8 * (k % 2);
    umma_f16_ts<id>(lead, dst, ak + 16, b + 128 * k, k > 0);
    umma_f16_ts<id>(lead, dst, ak, b + LO + 128 * k, 1);
  }
#pragma unroll
  for (int k = 0; k < KN / 16; ++k) umma_f16_ts<id>(lead, dst, a + 32 * (k / 2) + 8 * (k % 2), b + 128 * k, 1);
}
// The descriptors' low words of the operands above.
__device__ __forceinline__ uint32_t rows_desc(const unsigned char* tile) { return sw128_low(tile); }
template <int KN>
__device__ __forceinline__ uint32_t cols_desc(const unsigned char* tile) { return sw128_low(tile, KN * 128); }

// The two planes of two values below 2^16: hi = the value cut to 11 bits, lo =
// the rest (exact) rounded to 11.
__device__ __forceinline__ void split2(uint64_t x, uint32_t* hi, uint32_t* lo) {
  float a, b, c, d;
  unpack2(x, &a, &b);
  const float ah = __uint_as_float(__float_as_uint(a) & 0xFFFFE000u);
  const float bh = __uint_as_float(__float_as_uint(b) & 0xFFFFE000u);
  unpack2(fma2(pack2(ah, bh), pack2(-1.f, -1.f), x), &c, &d);
  const __half2 h = __floats2half2_rn(ah, bh), l = __floats2half2_rn(c, d);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// Before a CTA ends, its TMA thread waits for its copies and its MMA warps for
// their products, whether or not some role gave up: a role cannot know that the
// others will still read what it has in flight.  The copies are the latest of
// every slot.
__device__ __forceinline__ void drain(uint64_t* full, int slots, int issued) {
  for (int s = 0; s < slots && s < issued; ++s) {
    const int last = (issued - 1 - s) / slots;  // uses of this slot so far, less one
    mbar_wait(&full[s], (uint32_t)last & 1u);
  }
}

// A launch of 384 threads holds 168 registers each.  The warpgroup of the MMA
// and TMA warps gives up all but LEAN and the two others take FULL, with
// 128 LEAN + 256 FULL = 384 * 168: (56, 224) where a thread holds a row of
// results and of scores, (88, 208) where half a row is enough.
template <int LEAN>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(LEAN)); }
template <int LEAN>
__device__ __forceinline__ void take_registers() {
  static_assert((384 * 168 - 128 * LEAN) % 256 == 0, "all of the registers");
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"((384 * 168 - 128 * LEAN) / 256));
}

// ---- forward ---------------------------------------------------------------------

struct FwdDev {
  CrossDev c;
  Planes q, k, v;
  int mtiles, splits;    // items: mtiles * problems * splits
  int items;
  float *part, *part_m, *part_l;  // [split][problem][q.rows_p](DP) when splits > 1
  float f;               // |scale| log2 e
  int* err;
};

template <int DP, int MT>
struct FwdShape {
  static constexpr int KN = kTileElems / DP;
  static constexpr int q_bytes = MT * 128 * DP * 4;
  static constexpr int slots = MT == 2 ? (DP == 64 ? 5 : 3) : 4;
  static constexpr int smem = q_bytes + slots * kSlot + 1024 + 512;
  static constexpr int OB = DP == 64 ? 2 : 1;       // output accumulators per row tile
  static constexpr int cols = KN + OB * DP;         // tensor-memory columns per row tile
  static constexpr int threads = MT * 128 + 128;    // the row tiles' warpgroups; MT MMA warps, a TMA warp, idle ones
};

// One item of a persistent CTA: a block of MT row tiles, a problem, a part of
// its keys.
struct FwdItem {
  int mtile, pr, sp, b, hk, len, j0, n;  // n key tiles from j0
};
template <int KN>
__device__ __forceinline__ FwdItem fwd_item(const FwdDev& d, int item) {
  const CrossDev& c = d.c;
  FwdItem w;
  w.mtile = item % d.mtiles;
  item /= d.mtiles;
  const int np = c.B * c.Hk;
  w.pr = item % np;
  w.sp = item / np;
  w.b = w.pr / c.Hk;
  w.hk = w.pr % c.Hk;
  w.len = key_count(c.len, c.len64, c.len_s, c.Tk, w.b);
  const int all = (w.len + KN - 1) / KN, per = (all + d.splits - 1) / d.splits;
  w.j0 = min(all, w.sp * per);
  w.n = min(all, w.j0 + per) - w.j0;
  return w;
}

template <int DP, int DE, int MT>
__global__ void __launch_bounds__(MT * 128 + 128, 1)
cross_forward_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const __grid_constant__ FwdDev d) {
  using S = FwdShape<DP, MT>;
  constexpr int KN = S::KN, OB = S::OB, NS = S::slots;
  static_assert(MT * S::cols <= 512, "tensor memory");
  const CrossDev& c = d.c;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sq = smem;
  unsigned char* ring = smem + S::q_bytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + NS * kSlot);
  uint64_t* empty = full + NS;
  uint64_t* q_full = empty + NS;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;   // [MT] S of the next key tile, and P V of the last, are there
  uint64_t* p_ready = s_full + MT;  // [MT] P is there, and the output buffer it goes to has been read
  uint64_t* o_read = p_ready + MT;  // [MT] an item's last output has been read
  uint64_t* first_p = o_read + MT;  // row tile 0 has its first P of an item
  uint64_t* done = first_p + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + MT);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], MT);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, MT);
    mbar_init(first_p, 4);
    for (int t = 0; t < MT; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_ready[t], 4);
      mbar_init(&o_read[t], 4);
      mbar_init(&done[t], 1);
    }
    *failed = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int np = c.B * c.Hk;
  pdl_launch_dependents();
  pdl_wait();  // everything from here on reads what the pack kernel wrote
  if (*(volatile const int*)c.nonfinite != 0) {
    exact_rows(c, (int64_t)blockIdx.x * (blockDim.x / 32) + warp, (int64_t)gridDim.x * (blockDim.x / 32));
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
    return;
  }

  if (warp >= MT * 4) {
    if (MT == 2) give_registers<56>();
    if (warp == MT * 5 && lane == 0) {  // TMA
      int li = 0, qi = 0;               // tiles and query blocks loaded so far
      bool ok = true;
      for (int item = blockIdx.x; item < d.items && ok; item += gridDim.x) {
        const FwdItem w = fwd_item<KN>(d, item);
        if (w.n == 0) continue;
        if (qi > 0 && !(ok = wait_or_fail(q_empty, (uint32_t)(qi - 1) & 1u, failed))) break;
        mbar_arrive_expect_tx(q_full, S::q_bytes);
#pragma unroll 1
        for (int t = 0; t < MT; ++t)
          load_planes<DP, 128>(sq + t * 128 * DP * 4, &mq, d.q, w.pr * d.q.rows_p + (w.mtile * MT + t) * 128, q_full);
        ++qi;
        for (int i = 0; i < 2 * w.n; ++i, ++li) {
          const int s = li % NS;
          if (li >= NS && !(ok = wait_or_fail(&empty[s], (uint32_t)(li / NS - 1) & 1u, failed))) break;
          mbar_arrive_expect_tx(&full[s], kSlot);
          const int row = w.pr * d.k.rows_p + (w.j0 + i / 2) * KN;
          if (i & 1) load_planes<DP, KN>(ring + s * kSlot, &mv, d.v, row, &full[s]);
          else load_planes<DP, KN>(ring + s * kSlot, &mk, d.k, row, &full[s]);
        }
      }
      if (qi > 0) mbar_wait(q_full, (uint32_t)(qi - 1) & 1u);
      drain(full, NS, li);
    } else if (warp < MT * 5) {  // MMA of row tile t: the warp stays whole, one lane issues
      const int t = warp - MT * 4;
      const uint32_t lead = elect_lane(), ts = uniform(tmem + t * S::cols);
      const uint32_t dq = uniform(rows_desc(sq + t * 128 * DP * 4)), dk = uniform(rows_desc(ring));
      const uint32_t dv = uniform(cols_desc<KN>(ring));
      constexpr uint32_t SLOT = kSlot / 16;  // in descriptor units
      auto wait_all = [&](uint64_t* bar, int phase) {
        return __all_sync(0xffffffffu, spin_or_fail(bar, (uint32_t)phase & 1u, failed)) != 0;
      };
      int slot = 0, ph = 0, qi = 0, pc = 0;  // next tile's slot and its phase; query blocks and P's so far
      bool ok = true;
      for (int item = blockIdx.x; item < d.items && ok; item += gridDim.x) {
        const int n = fwd_item<KN>(d, item).n;
        if (n == 0) continue;
        ok = wait_all(q_full, qi) && wait_all(&full[slot], ph) && (qi == 0 || wait_all(&o_read[t], qi - 1));
        // the second row tile starts when the first has left the softmax, so that
        // from then on one is in the softmax while the other has the tensor core
        if (ok && t == 1) ok = wait_all(first_p, qi);
        if (!ok) break;
        ++qi;
        tc_fence_after();
        mma_abt<DP, DE, KN>(lead, ts, dq, dk + slot * SLOT);
        umma_commit(lead, &s_full[t]);
        umma_commit(lead, &empty[slot]);
        if (n == 1) umma_commit(lead, q_empty);
        if (++slot == NS) { slot = 0; ++ph; }
        for (int j = 0; j < n; ++j) {
          const bool more = j + 1 < n;
          const int sv = slot, sk = slot + 1 == NS ? 0 : slot + 1, pk = sk ? ph : ph + 1;
          // with three slots the next K may still be on its way when P is there
          ok = wait_all(&full[sv], ph) && (NS < 5 || !more || wait_all(&full[sk], pk)) && wait_all(&p_ready[t], pc);
          if (!ok) break;
          ++pc;
          tc_fence_after();
          mma_ab<DP, DE, KN>(lead, ts + KN + (OB == 2 ? (j & 1) * DP : 0), ts, dv + sv * SLOT);
          if (NS < 5) umma_commit(lead, &empty[sv]);
          if (more) {
            if (NS < 5 && !(ok = wait_all(&full[sk], pk))) break;
            mma_abt<DP, DE, KN>(lead, ts, dq, dk + sk * SLOT);
          }
          umma_commit(lead, &s_full[t]);
          if (NS >= 5) umma_commit(lead, &empty[sv]);
          slot = sk;
          ph = pk;
          if (more) {
            umma_commit(lead, &empty[sk]);
            if (j + 2 == n) umma_commit(lead, q_empty);
            if (++slot == NS) { slot = 0; ++ph; }
          }
        }
      }
      umma_commit(lead, &done[t]);
      mbar_wait(&done[t], 0);
    }
  } else {  // softmax: one thread per row
    if (MT == 2) take_registers<56>();
    const int t = warp / 4, rl = (warp % 4) * 32 + lane;
    const uint32_t sbase = tmem + ((uint32_t)((warp % 4) * 32) << 16) + t * S::cols, obase = sbase + KN;
    const int qtiles = d.q.rows_p / KN, ktiles = d.k.rows_p / KN;
    int sc = 0;  // S's taken so far
    bool ok = true;
    for (int item = blockIdx.x; item < d.items && ok; item += gridDim.x) {
      int n, kt, limit;  // key tiles, the first one's index among all, keys from it on
      float iq;
      {
        const FwdItem w = fwd_item<KN>(d, item);
        n = w.n;
        kt = w.pr * ktiles + w.j0;
        limit = w.len - w.j0 * KN;
        iq = d.q.inv[w.pr * qtiles + ((w.mtile * MT + t) * 128 + rl) / KN];
      }
      float m = -FLT_MAX, l = 0.f, keep = 0.f;  // keep: what the output so far is scaled by when the next tile is added
      float acc[DE];
#pragma unroll
      for (int i = 0; i < DE; ++i) acc[i] = 0.f;
      // adds tile j's P V, complete, to the output; P's 2^15 goes here, an exact
      // power of two, so that the output stays in range wherever sum P |v| does
      auto add_output = [&](int j) {
        const uint32_t src = obase + (OB == 2 ? (j & 1) * DP : 0);
        const float fv = d.v.inv[kt + j] * 0x1p-15f;
        const uint64_t fv2 = pack2(fv, fv), keep2 = pack2(keep, keep);
#pragma unroll
        for (int cc = 0; cc < DE / 32; ++cc) {
          uint32_t o[32];
          tmem_ld32_issue(src + cc * 32, o);
          tmem_ld_done(o);
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            uint64_t a2 = mul2(pack2(acc[cc * 32 + i], acc[cc * 32 + i + 1]), keep2);
            a2 = fma2(pack2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), fv2, a2);
            unpack2(a2, &acc[cc * 32 + i], &acc[cc * 32 + i + 1]);
          }
        }
      };
      for (int j = 0; j < n; ++j, limit -= KN) {
        // neither 0 nor inf: -inf stands for an absent key below, and a score of 0 stays 0
        float f = fminf(fmaxf(mul3(d.f, iq, d.k.inv[kt + j]), 0x1p-126f), FLT_MAX);
        const bool far = __any_sync(0xffffffffu, f >= kFarMax<DP>);
        ok = __all_sync(0xffffffffu, wait_or_fail(&s_full[t], (uint32_t)sc & 1u, failed)) != 0;
        if (!ok) break;
        ++sc;
        tc_fence_after();
        if (OB == 1 && j > 0) add_output(j - 1);
        uint32_t x[KN / 32][32];  // the row of S, then of P
#pragma unroll
        for (int cc = 0; cc < KN / 32; ++cc) tmem_ld32_issue(sbase + cc * 32, x[cc]);
        tmem_ld_done(x[0]);
#pragma unroll
        for (int cc = 1; cc < KN / 32; ++cc) tmem_ld_tie(x[cc]);
        float base = 0.f;
        if (far || limit < KN) {
#pragma unroll
          for (int cc = 0; cc < KN / 32; ++cc)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (cc * 32 + i >= limit) x[cc][i] = 0xff800000u;  // behind the last key: no weight
          if (far) {  // this tile's scores relative to the largest so far
            float mx = __uint_as_float(x[0][0]);
#pragma unroll
            for (int i = 1; i < KN; ++i) mx = fmaxf(mx, __uint_as_float(x[i / 32][i % 32]));
            base = fmaxf(m, mx * f);
#pragma unroll
            for (int i = 0; i < KN; ++i) x[i / 32][i % 32] = __float_as_uint(__uint_as_float(x[i / 32][i % 32]) * f - base);
            m -= base;
            f = 1.f;
          }
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int cc = 0; cc < KN / 32; ++cc)
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx4[i / 2 % 4] = fmaxf(fmaxf(mx4[i / 2 % 4], __uint_as_float(x[cc][i])), __uint_as_float(x[cc][i + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        const float mn = fmaxf(m, mx * f);
        const float alpha = ex2(m - mn);
        m = mn + base;
        const uint64_t f2 = pack2(f, f), b2 = pack2(15.f - mn, 15.f - mn);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int cc = 0; cc < KN / 32; ++cc) {
          uint32_t y[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float p0, p1;
            unpack2(fma2(pack2(__uint_as_float(x[cc][2 * i]), __uint_as_float(x[cc][2 * i + 1])), f2, b2), &p0, &p1);
            const uint64_t p = pack2(ex2(p0), ex2(p1));
            sum[i & 1] = add2(sum[i & 1], p);
            split2(p, &y[i], &y[16 + i]);
          }
          tmem_st32(sbase + cc * 32, y);
        }
        float sum0, sum1;
        unpack2(add2(sum[0], sum[1]), &sum0, &sum1);
        l = __fmaf_rn(l, alpha, sum0 + sum1);
        tmem_st_done();
        tc_fence_before();
        warp_arrive(&p_ready[t]);
        if (MT == 2 && t == 0 && j == 0) warp_arrive(first_p);
        if (OB == 2 && j > 0) add_output(j - 1);
        keep = alpha;
      }
      if (ok && n > 0) {
        ok = __all_sync(0xffffffffu, wait_or_fail(&s_full[t], (uint32_t)sc & 1u, failed)) != 0;
        if (!ok) break;
        ++sc;
        tc_fence_after();
        add_output(n - 1);
        tc_fence_before();
        warp_arrive(&o_read[t]);
      }
      const FwdItem w = fwd_item<KN>(d, item);
      const int row = (w.mtile * MT + t) * 128 + rl;
      if (ok && row < c.M) {
        if (d.splits > 1) {
          const int64_t at = ((int64_t)w.sp * np + w.pr) * d.q.rows_p + row;
          float4* o = reinterpret_cast<float4*>(d.part + at * DP);
#pragma unroll
          for (int i = 0; i < DE / 4; ++i) o[i] = make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]);
          d.part_m[at] = m;
          d.part_l[at] = l * 0x1p-15f;  // l carries P's 2^15
        } else {
          const int g = (int)fdiv((uint32_t)row, c.f_Tq), tt = row - g * c.Tq, h = w.hk * c.G + g;
          float* op = static_cast<float*>(c.out.p) + w.b * c.out.sb + tt * c.out.st + h * c.out.sh;
          const float inv = l == 0.f ? 0.f : 0x1p15f / l;  // l carries P's 2^15
          if (c.vec) {
#pragma unroll
            for (int i = 0; i < DE / 4; ++i)
              if (4 * i < c.D)
                reinterpret_cast<float4*>(op)[i] =
                    make_float4(acc[4 * i] * inv, acc[4 * i + 1] * inv, acc[4 * i + 2] * inv, acc[4 * i + 3] * inv);
          } else {
#pragma unroll
            for (int i = 0; i < DE; ++i)
              if (i < c.D) op[i * c.out.sd] = acc[i] * inv;
          }
          if (c.lse) c.lse[w.b * c.ls_b + h * c.ls_h + tt * c.ls_t] = l == 0.f ? -INFINITY : (m + log2f(l * 0x1p-15f)) * kLn2;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed && d.err) atomicOr(d.err, kAsyncWaitTimeout);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// ---- backward --------------------------------------------------------------------

// The items of a persistent CTA: its first by its number, then whichever is
// next of all (a counter in global memory), so that ragged lengths even out.  The
// TMA thread takes them, one ahead, and passes them on through two slots; -1
// ends the CTA.  Which CTA walks an item changes no result.  Forward and backward
// against every grid-th item: 8 ragged heads of 128, 7 x 500 queries on up to 900
// keys, 334 -> 301 us; 16 of 64, 4 x 1024 on up to 1500, 340 -> 327; equal lengths
// (16 heads of 128, 2 x 2048 on 2048) 1091 -> 1073.  The forward kernel keeps every
// grid-th: its items are short, and taking them cost 82 -> 84 us (4 x 1024 on up to
// 1500, 16 heads of 64) to 143 -> 159 (6 x 403 on up to 1878, heads of 80).
struct ItemRing {
  int slot[2];
  uint64_t full[2], empty[2];
};
__device__ __forceinline__ void items_init(ItemRing& r, uint32_t takers) {
  for (int i = 0; i < 2; ++i) {
    mbar_init(&r.full[i], 1);
    mbar_init(&r.empty[i], takers);
  }
}
// The TMA thread passes on the k-th item.
__device__ __forceinline__ bool items_put(ItemRing& r, int k, int item, int* failed) {
  if (k >= 2 && !wait_or_fail(&r.empty[k & 1], (uint32_t)(k / 2 - 1) & 1u, failed)) return false;
  *(volatile int*)&r.slot[k & 1] = item;
  mbar_arrive(&r.full[k & 1]);
  return true;
}
// A warp takes the k-th item: -1 after the last, or when some role gave up.
__device__ __forceinline__ int items_take(ItemRing& r, int k, int* failed) {
  if (!__all_sync(0xffffffffu, wait_or_fail(&r.full[k & 1], (uint32_t)(k / 2) & 1u, failed))) return -1;
  const int item = __shfl_sync(0xffffffffu, *(volatile int*)&r.slot[k & 1], 0);
  warp_arrive(&r.empty[k & 1]);
  return item;
}

struct BwdDev {
  CrossDev c;
  Planes a1, a2, b1, b2;       // dq: q, dout, k, v;  dk/dv: k, v, q, dout
  int mtiles, splits, items;
  int* next;                   // items taken beyond the first of every CTA
  const float *bias, *delta, *rnorm, *dmax;  // per query row; per query tile
  float *part1, *part2;        // [split][problem][a1.rows_p][DP] when splits > 1: dq, or dk and dv
  float f;                     // |scale| log2 e
  float out_scale, out_pow;    // of dq (scale) or dk (|scale|), as [1, 2) times a power of two
  int* err;
};

template <int DP>
struct BwdShape {
  static constexpr int KN = kTileElems / DP;
  static constexpr int a_bytes = 128 * DP * 4;
  static constexpr int n1 = DP == 64 ? 3 : 2, n2 = DP == 64 ? 2 : 1;
  static constexpr bool ahead = n1 == 3;  // room for S two tiles ahead
  static constexpr int smem = 2 * a_bytes + (n1 + n2) * kSlot + 1024 + 512;
  static constexpr int threads = 384;
};

// One item of a persistent CTA: a row tile, a problem, a part of the walk.
struct BwdItem {
  int mtile, pr, sp, b, hk, rows, cols, j0, n;  // rows with work, columns, n column tiles from j0
};
template <int KN, bool KV>
__device__ __forceinline__ BwdItem bwd_item(const BwdDev& d, int item) {
  const CrossDev& c = d.c;
  BwdItem w;
  w.mtile = item % d.mtiles;
  item /= d.mtiles;
  const int np = c.B * c.Hk;
  w.pr = item % np;
  w.sp = item / np;
  w.b = w.pr / c.Hk;
  w.hk = w.pr % c.Hk;
  const int len = key_count(c.len, c.len64, c.len_s, c.Tk, w.b);
  w.cols = KV ? c.M : len;
  w.rows = KV ? len : c.M;
  const int all = w.mtile * 128 >= w.rows || len == 0 ? 0 : (w.cols + KN - 1) / KN;
  const int per = (all + d.splits - 1) / d.splits;
  w.j0 = min(all, w.sp * per);
  w.n = min(all, w.j0 + per) - w.j0;
  return w;
}

template <int DP, int DE, bool KV>
__global__ void __launch_bounds__(384, 1)
cross_backward_kernel(const __grid_constant__ CUtensorMap ma1, const __grid_constant__ CUtensorMap ma2,
                      const __grid_constant__ CUtensorMap mb1, const __grid_constant__ CUtensorMap mb2,
                      const __grid_constant__ BwdDev d) {
  using S = BwdShape<DP>;
  constexpr int KN = S::KN, N1 = S::n1, N2 = S::n2, HC = KN / 2;  // HC: columns of a warpgroup
  constexpr int AC = KV ? DE : (DE + 63) / 64 * 32;               // result columns of a warpgroup (of 96: 64 and 32)
  // dq needs no plane of P, so dS takes the place of S, and the next dP can be
  // issued before the product that reads dS
  constexpr bool DS_IN_S = !KV && S::ahead;
  static_assert(3 * KN + (KV ? 2 : 1) * DP <= 512, "tensor memory");
  const CrossDev& c = d.c;
  __shared__ ItemRing items;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* sa1 = smem;
  unsigned char* sa2 = smem + S::a_bytes;
  unsigned char* ring1 = sa2 + S::a_bytes;
  unsigned char* ring2 = ring1 + N1 * kSlot;
  uint64_t* full1 = reinterpret_cast<uint64_t*>(ring2 + N2 * kSlot);
  uint64_t* empty1 = full1 + N1;
  uint64_t* full2 = empty1 + N1;
  uint64_t* empty2 = full2 + N2;
  uint64_t* a_full = empty2 + N2;
  uint64_t* a_empty = a_full + 1;
  uint64_t* s_full = a_empty + 1;   // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* p_ready = dp_full + 1;  // [2]: may run a phase ahead of the MMA warp
  uint64_t* ds_ready = p_ready + 2;
  uint64_t* r_full = ds_ready + 1;  // a tile's results are there
  uint64_t* r_free = r_full + 1;    // dv's accumulator has been read
  uint64_t* done = r_free + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  int* failed = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < N1; ++s) {
      mbar_init(&full1[s], 1);
      mbar_init(&empty1[s], 1);
    }
    for (int s = 0; s < N2; ++s) {
      mbar_init(&full2[s], 1);
      mbar_init(&empty2[s], 1);
    }
    items_init(items, 9);
    mbar_init(a_full, 1);
    mbar_init(a_empty, 1);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(dp_full, 1);
    mbar_init(&p_ready[0], 8);
    mbar_init(&p_ready[1], 8);
    mbar_init(ds_ready, 8);
    mbar_init(r_full, 1);
    mbar_init(r_free, 4);
    mbar_init(done, 1);
    *failed = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int np = c.B * c.Hk;
  pdl_launch_dependents();
  pdl_wait();  // everything from here on reads what the pack kernel wrote
  if (*(volatile const int*)c.nonfinite != 0) {
    const int64_t w0 = (int64_t)blockIdx.x * (blockDim.x / 32) + warp, nw = (int64_t)gridDim.x * (blockDim.x / 32);
    if (KV) exact_dkv_rows(c, w0, nw);
    else exact_dq_rows(c, w0, nw);
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
    return;
  }
  // tensor-memory columns: S (two buffers), dP, then the results (dq; dk, dv)

  if (warp >= 8) {
    give_registers<KV ? 56 : 88>();
    if (warp == 9 && lane == 0) {  // TMA
      int t = 0, i2 = 0, ai = 0;   // column tiles of either operand and row tiles loaded so far
      bool ok = true;
      for (int k = 0, item = blockIdx.x, next; ok; item = next, ++k) {
        if (!(ok = items_put(items, k, item < d.items ? item : -1, failed)) || item >= d.items) break;
        next = gridDim.x + atomicAdd(d.next, 1);
        const BwdItem w = bwd_item<KN, KV>(d, item);
        if (w.n == 0) continue;
        if (ai > 0 && !(ok = wait_or_fail(a_empty, (uint32_t)(ai - 1) & 1u, failed))) break;
        mbar_arrive_expect_tx(a_full, 2 * S::a_bytes);
        load_planes<DP, 128>(sa1, &ma1, d.a1, w.pr * d.a1.rows_p + w.mtile * 128, a_full);
        load_planes<DP, 128>(sa2, &ma2, d.a2, w.pr * d.a2.rows_p + w.mtile * 128, a_full);
        ++ai;
        for (int j = 0; j < w.n; ++j) {
          const int row = w.pr * d.b1.rows_p + (w.j0 + j) * KN;
          const int s1 = t % N1, s2 = t % N2;
          if (t >= N1 && !(ok = wait_or_fail(&empty1[s1], (uint32_t)(t / N1 - 1) & 1u, failed))) break;
          mbar_arrive_expect_tx(&full1[s1], kSlot);
          load_planes<DP, KN>(ring1 + s1 * kSlot, &mb1, d.b1, row, &full1[s1]);
          ++t;
          if (i2 >= N2 && !(ok = wait_or_fail(&empty2[s2], (uint32_t)(i2 / N2 - 1) & 1u, failed))) break;
          mbar_arrive_expect_tx(&full2[s2], kSlot);
          load_planes<DP, KN>(ring2 + s2 * kSlot, &mb2, d.b2, row, &full2[s2]);
          ++i2;
        }
      }
      if (ai > 0) mbar_wait(a_full, (uint32_t)(ai - 1) & 1u);
      drain(full1, N1, t);
      drain(full2, N2, i2);
    } else if (warp == 8) {  // MMA: the warp stays whole, one lane issues
      const uint32_t lead = elect_lane(), tm = uniform(tmem);
      const uint32_t d1 = uniform(rows_desc(sa1)), d2 = uniform(rows_desc(sa2));
      const uint32_t r1 = uniform(rows_desc(ring1)), r2 = uniform(rows_desc(ring2));
      const uint32_t c1 = uniform(cols_desc<KN>(ring1)), c2 = uniform(cols_desc<KN>(ring2));
      constexpr uint32_t SLOT = kSlot / 16;
      const uint32_t dpc = tm + 2 * KN, rc1 = tm + 3 * KN, rc2 = rc1 + DP;
      auto wait_all = [&](uint64_t* bar, int phase) {
        return __all_sync(0xffffffffu, spin_or_fail(bar, (uint32_t)phase & 1u, failed)) != 0;
      };
      // t: column tiles of all items so far, which the slots and phases go by
      auto s_ready = [&](int t) { return wait_all(&full1[t % N1], t / N1); };
      auto dp_ready = [&](int t) { return wait_all(&full2[t % N2], t / N2); };
      auto s_mma = [&](int t) {
        mma_abt<DP, DE, KN>(lead, tm + (t & 1) * KN, d1, r1 + t % N1 * SLOT);
        umma_commit(lead, &s_full[t & 1]);
      };
      auto dp_mma = [&](int t) {
        mma_abt<DP, DE, KN>(lead, dpc, d2, r2 + t % N2 * SLOT);
        umma_commit(lead, dp_full);
      };
      int t0 = 0, ai = 0;
      bool ok = true;
      for (int k = 0; ok; ++k) {
        const int item = items_take(items, k, failed);
        if (item < 0) break;
        const int n = bwd_item<KN, KV>(d, item).n;
        if (n == 0) continue;
        ok = wait_all(a_full, ai) && s_ready(t0) && dp_ready(t0);
        if (!ok) break;
        ++ai;
        tc_fence_after();
        s_mma(t0);
        dp_mma(t0);
        if (!KV) umma_commit(lead, &empty2[t0 % N2]);
        if (S::ahead && n > 1) {
          if (!(ok = s_ready(t0 + 1))) break;
          s_mma(t0 + 1);
        }
        if (n == 1) umma_commit(lead, a_empty);
        for (int j = 0; j < n; ++j) {
          const int t = t0 + j;
          const bool more = j + 1 < n, more2 = S::ahead && j + 2 < n;
          if (S::ahead && more && !(ok = dp_ready(t + 1))) break;  // on its way long since
          if (KV) {
            ok = wait_all(&p_ready[t & 1], t >> 1) && (t == 0 || wait_all(r_free, t - 1));
            if (!ok) break;
            tc_fence_after();
            mma_ab<DP, DE, KN>(lead, rc2, tm + (t & 1) * KN, c2 + t % N2 * SLOT);  // P^T dout
            umma_commit(lead, &empty2[t % N2]);
          }
          if (!S::ahead && more) {
            if (!(ok = s_ready(t + 1))) break;
            s_mma(t + 1);
          }
          if (!(ok = wait_all(ds_ready, t))) break;
          tc_fence_after();
          if (DS_IN_S && more) dp_mma(t + 1);
          mma_ab<DP, DE, KN>(lead, rc1, DS_IN_S ? tm + (t & 1) * KN : dpc, c1 + t % N1 * SLOT);  // dS k, or dS^T q
          if (!KV && S::ahead && more) umma_commit(lead, &empty2[(t + 1) % N2]);
          umma_commit(lead, r_full);
          umma_commit(lead, &empty1[t % N1]);
          if (!DS_IN_S && more) {
            if (!S::ahead && !(ok = dp_ready(t + 1))) break;
            dp_mma(t + 1);
            if (!KV) umma_commit(lead, &empty2[(t + 1) % N2]);
          }
          if (more2) {
            if (!(ok = s_ready(t + 2))) break;
            s_mma(t + 2);
          }
          if (j + 2 == n) umma_commit(lead, a_empty);
        }
        t0 += n;
      }
      umma_commit(lead, done);
      mbar_wait(done, 0);
    }
  } else {
    take_registers<KV ? 56 : 88>();
    const int wg = warp / 4, rl = (warp % 4) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t t_dp = tmem + lanes + 2 * KN + wg * HC;
    // wg 0 of (dk, dv) takes dv, wg 1 dk; of dq each takes half of the columns
    const uint32_t t_res = tmem + lanes + 3 * KN + (KV ? (wg == 0 ? DP : 0) : wg * AC);
    const int at1 = d.a1.rows_p / KN, bt = d.b1.rows_p / KN;
    int t = 0;  // column tiles so far
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int item = items_take(items, k, failed);
      if (item < 0) break;
      int n, kt, limit;  // column tiles, the first one's index among all, columns of this half from it on
      int64_t qrow;      // per query row: of this row (dq) or of the columns (dk, dv)
      float ia1, ia2, r_norm;
      {
        const BwdItem w = bwd_item<KN, KV>(d, item);
        n = w.n;
        kt = w.pr * bt + w.j0;
        limit = w.cols - w.j0 * KN - wg * HC;
        const int row = w.mtile * 128 + rl;
        ia1 = d.a1.inv[w.pr * at1 + row / KN];
        ia2 = d.a2.inv[w.pr * at1 + row / KN];
        qrow = (int64_t)w.pr * (KV ? d.b1.rows_p : d.a1.rows_p) + (KV ? w.j0 * KN + wg * HC : row);
        r_norm = KV ? d.a2.norm[w.pr * at1 + row / KN] : d.rnorm[qrow];
      }
      const float r_bias = KV ? 0.f : d.bias[qrow] - 15.f, r_delta = KV ? 0.f : d.delta[qrow];
      float acc[AC];
#pragma unroll
      for (int i = 0; i < AC; ++i) acc[i] = 0.f;
      // what the last tile's results are multiplied by, powers of two: all at once
      // (wt), or up before wt where the product is too small for an f32
      float wt = 0.f, up = 1.f;
      // adds a tile's results, complete, to those so far
      auto add_results = [&]() {
        const bool tiny = __any_sync(0xffffffffu, up != 1.f);
        const uint64_t wt2 = pack2(wt, wt);
#pragma unroll
        for (int cc = 0; cc < AC / 32; ++cc) {
          if (!KV && wg * AC + cc * 32 >= DE) continue;
          uint32_t o[32];
          tmem_ld32_issue(t_res + cc * 32, o);
          tmem_ld_done(o);
          if (tiny) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * up);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            unpack2(fma2(pack2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), wt2,
                         pack2(acc[cc * 32 + i], acc[cc * 32 + i + 1])),
                    &acc[cc * 32 + i], &acc[cc * 32 + i + 1]);
        }
      };
      auto wait_warp = [&](uint64_t* bar, int phase) {
        return __all_sync(0xffffffffu, wait_or_fail(bar, (uint32_t)phase & 1u, failed)) != 0;
      };
      for (int j = 0; j < n; ++j, ++t, limit -= KN) {
        // the tile's factors, ahead of the waits (behind them dk and dv 403 -> 411 us)
        const float ib1 = d.b1.inv[kt + j];
        const float f = fminf(mul3(d.f, ia1, ib1), FLT_MAX);  // a score of 0 stays 0
        const bool far = __any_sync(0xffffffffu, f >= kFarSum<DP>);
        // |dS| <= |dout_i| |v_j| + |delta_i|, the largest of the tile; scaled below
        // 2^15.  A norm counts as 1 of its tile's units at least, so that a row of
        // zeros beside large ones keeps a finite factor
        const float ib2 = d.b2.inv[kt + j];
        const float bound = mul3(fmaxf(r_norm * d.b2.norm[kt + j], 1.f), ia2, ib2) + (KV ? d.dmax[kt + j] : fabsf(r_delta));
        uint32_t eb = __float_as_uint(bound) >> 23;
        eb = eb < 15u ? 15u : eb;
        const float ds_up = __uint_as_float((268u - eb) << 23) * (KV ? 0x1p-15f : 1.f);
        const float gu1 = mul3(ia2, ib2, ds_up);
        const bool is_dv = KV && wg == 0;  // of P 2^15 alone
        const float w1 = is_dv ? ib2 : ib1, w2 = is_dv ? 0x1p-15f : __uint_as_float((eb - 14u) << 23);
        const float w3 = is_dv ? 1.f : d.out_pow;
        float wt_next = mul3(w1, w2, w3), up_next = 1.f;
        if (wt_next < 0x1p-126f) {
          wt_next = fminf(fminf(w1, w2), w3);
          up_next = fmaxf(fmaxf(w1, w2), w3) * fmaxf(fminf(w1, w2), fminf(fmaxf(w1, w2), w3));
        }
        const uint32_t sb = tmem + lanes + (t & 1) * KN + wg * HC;
        float p[HC];  // the exponent's bias, then P (dk, dv: P 2^15)
        if (KV) {
          const float4* bi = reinterpret_cast<const float4*>(d.bias + qrow + j * KN);
#pragma unroll
          for (int i = 0; i < HC / 4; ++i) {
            const float4 x = __ldg(bi + i);
            p[4 * i] = x.x;
            p[4 * i + 1] = x.y;
            p[4 * i + 2] = x.z;
            p[4 * i + 3] = x.w;
          }
        }
        if (!(ok = wait_warp(&s_full[t & 1], t >> 1))) break;
        tc_fence_after();
        const uint64_t f2 = pack2(f, f);
        {
          uint32_t a[HC / 32][32];
#pragma unroll
          for (int cc = 0; cc < HC / 32; ++cc) tmem_ld32_issue(sb + cc * 32, a[cc]);
          tmem_ld_done(a[0]);
#pragma unroll
          for (int cc = 1; cc < HC / 32; ++cc) tmem_ld_tie(a[cc]);
#pragma unroll
          for (int cc = 0; cc < HC / 32; ++cc) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float& p0 = p[cc * 32 + i];
              float& p1 = p[cc * 32 + i + 1];
              const uint64_t bias = KV ? pack2(p0, p1) : pack2(r_bias, r_bias);
              unpack2(fma2(pack2(__uint_as_float(a[cc][i]), __uint_as_float(a[cc][i + 1])), f2, bias), &p0, &p1);
            }
          }
          if (far) {
#pragma unroll
            for (int i = 0; i < HC; ++i) p[i] = min_nan(p[i], KV ? 15.f : 0.f);
          }
#pragma unroll
          for (int cc = 0; cc < HC / 32; ++cc) {
#pragma unroll
            for (int i = 0; i < 32; ++i) p[cc * 32 + i] = ex2(p[cc * 32 + i]);
            if (KV) {
              uint32_t w[32];
#pragma unroll
              for (int i = 0; i < 16; ++i) split2(pack2(p[cc * 32 + 2 * i], p[cc * 32 + 2 * i + 1]), &w[i], &w[16 + i]);
              tmem_st32(sb + cc * 32, w);
            }
          }
        }
        if (KV) {
          tmem_st_done();
          tc_fence_before();
          warp_arrive(&p_ready[t & 1]);
        }
        const uint64_t gu = pack2(gu1, gu1), nup = pack2(-ds_up, -ds_up), ndu = pack2(-r_delta * ds_up, -r_delta * ds_up);
        if (!(ok = wait_warp(dp_full, t))) break;
        // the last tile's results: for (dk, dv) complete before this dP was
        // issued; for dq behind it, and read at the end
        if (KV && j > 0 && !(ok = wait_warp(r_full, t - 1))) break;
        tc_fence_after();
        if (KV && j > 0) {
          add_results();
          tc_fence_before();
          if (wg == 0) warp_arrive(r_free);
        }
#pragma unroll
        for (int cc = 0; cc < HC / 32; ++cc) {
          uint32_t a[32], w[32];
          float4 dl[8];
          if (KV) {
            const float4* de = reinterpret_cast<const float4*>(d.delta + qrow + j * KN + cc * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) dl[i] = __ldg(de + i);
          }
          tmem_ld32_issue(t_dp + cc * 32, a);
          tmem_ld_done(a);
          const bool part = !KV && limit < (cc + 1) * 32;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float4& q = dl[i / 2];
            const uint64_t nd = KV ? mul2(i % 2 ? pack2(q.z, q.w) : pack2(q.x, q.y), nup) : ndu;
            uint64_t x = mul2(pack2(p[cc * 32 + 2 * i], p[cc * 32 + 2 * i + 1]),
                              fma2(pack2(__uint_as_float(a[2 * i]), __uint_as_float(a[2 * i + 1])), gu, nd));
            if (part) {
              float x0, x1;
              unpack2(x, &x0, &x1);
              x = pack2(cc * 32 + 2 * i < limit ? x0 : 0.f, cc * 32 + 2 * i + 1 < limit ? x1 : 0.f);
            }
            split2(x, &w[i], &w[16 + i]);
          }
          tmem_st32((DS_IN_S ? sb : t_dp) + cc * 32, w);
        }
        if (!KV && j > 0) {
          if (!(ok = wait_warp(r_full, t - 1))) break;
          tc_fence_after();
          add_results();
        }
        tmem_st_done();
        tc_fence_before();
        warp_arrive(ds_ready);
        wt = wt_next;
        up = up_next;
      }
      if (!ok) break;
      if (n > 0) {
        if (!(ok = wait_warp(r_full, t - 1))) break;
        tc_fence_after();
        add_results();
        tc_fence_before();
        if (KV && wg == 0) warp_arrive(r_free);
        if (!KV || wg == 1) {
#pragma unroll
          for (int i = 0; i < AC; ++i) acc[i] *= d.out_scale;
        }
      }
      const BwdItem w = bwd_item<KN, KV>(d, item);
      const int row = w.mtile * 128 + rl;
      const int stored = KV ? c.Tk : c.M;  // rows of the result; those without work hold zeros
      if (row < stored) {
        const bool live = row < w.rows;
        if (d.splits > 1) {
          float* pp = (KV && wg == 0 ? d.part2 : d.part1) + (((int64_t)w.sp * np + w.pr) * d.a1.rows_p + row) * DP + (KV ? 0 : wg * AC);
#pragma unroll
          for (int i = 0; i < AC / 4; ++i)
            reinterpret_cast<float4*>(pp)[i] = live ? make_float4(acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3])
                                                    : make_float4(0.f, 0.f, 0.f, 0.f);
        } else {
          const HeadsDev& o = KV ? (wg == 0 ? c.dv : c.dk) : c.dq;
          const int g = KV ? 0 : (int)fdiv((uint32_t)row, c.f_Tq), tt = KV ? row : row - g * c.Tq;
          const int h = KV ? w.hk : w.hk * c.G + g, c0 = KV ? 0 : wg * AC;
          float* op = static_cast<float*>(o.p) + w.b * o.sb + tt * o.st + h * o.sh;
#pragma unroll
          for (int i = 0; i < AC; i += 4) {
            const float4 x = live ? make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
            if (c.vec) {
              if (c0 + i < c.D) *reinterpret_cast<float4*>(op + c0 + i) = x;
            } else {
              if (c0 + i < c.D) op[(c0 + i) * o.sd] = x.x;
              if (c0 + i + 1 < c.D) op[(c0 + i + 1) * o.sd] = x.y;
              if (c0 + i + 2 < c.D) op[(c0 + i + 2) * o.sd] = x.z;
              if (c0 + i + 3 < c.D) op[(c0 + i + 3) * o.sd] = x.w;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *failed && d.err) atomicOr(d.err, kAsyncWaitTimeout);
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// result[row] = the parts added in order, of up to three results (blockIdx.y)
struct SumOne {
  const float* part;
  HeadsDev out;
  int splits, rows_p, G, T;
  FastDiv f_T;
  int64_t n;             // problems * G * T * (ld / 4)
};
struct SumDev {
  SumOne r[3];
  int np, ld, Hk, D;
  const int* nonfinite;
};
__global__ void __launch_bounds__(256) cross_sum_kernel(const __grid_constant__ SumDev d) {
  pdl_wait();
  const SumOne& r = d.r[blockIdx.y];
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= r.n || *(volatile const int*)d.nonfinite != 0) return;
  const int q = d.ld / 4, c = (int)(i % q) * 4;
  const int64_t w = i / q;
  const int row = (int)(w % (r.G * r.T)), pr = (int)(w / (r.G * r.T));
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  const float* p = r.part + ((int64_t)pr * r.rows_p + row) * d.ld + c;
  const int64_t step = (int64_t)d.np * r.rows_p * d.ld;
  for (int k = 0; k < r.splits; k += 4) {
    float4 x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      x[u] = k + u < r.splits ? *reinterpret_cast<const float4*>(p + (k + u) * step) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      s.x += x[u].x;
      s.y += x[u].y;
      s.z += x[u].z;
      s.w += x[u].w;
    }
  }
  const int g = (int)fdiv((uint32_t)row, r.f_T), t = row - g * r.T;
  float* o = static_cast<float*>(r.out.p) + (pr / d.Hk) * r.out.sb + t * r.out.st + (pr % d.Hk * r.G + g) * r.out.sh;
  if (c < d.D) o[c * r.out.sd] = s.x;
  if (c + 1 < d.D) o[(c + 1) * r.out.sd] = s.y;
  if (c + 2 < d.D) o[(c + 2) * r.out.sd] = s.z;
  if (c + 3 < d.D) o[(c + 3) * r.out.sd] = s.w;
}

// ---- host side -------------------------------------------------------------------

// The planes, scales and norms of one operand inside the workspace.
struct Packed {
  __half *hi = nullptr, *lo = nullptr;
  float *inv = nullptr, *norm = nullptr;
  int rows_p = 0, rows_all = 0;
  CUtensorMap map128, mapKN;
  Planes planes() const { return Planes{rows_p, rows_all, inv, norm}; }
};

struct Arena {  // sizes first (base null), then places
  char* base = nullptr;
  size_t used = 0;
  template <class T> T* take(size_t n) {
    T* p = reinterpret_cast<T*>(base + used);
    used += (n * sizeof(T) + 1023) / 1024 * 1024;
    return p;
  }
};

Error plane_map(EncodeTiled enc, CUtensorMap* map, const __half* hi, int64_t rows2, int DP, int box) {
  const cuuint64_t dims[2] = {(cuuint64_t)DP, (cuuint64_t)rows2};
  const cuuint64_t strides[1] = {(cuuint64_t)DP * 2};
  const cuuint32_t bx[2] = {64, (cuuint32_t)box};
  const cuuint32_t es[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half*>(hi), dims, strides, bx, es,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return make_error(TRS_ERR_CUDA, "cross_attention: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return Error{};
}

int up_to(int x, int m) { return (x + m - 1) / m * m; }

void place(Arena& a, Packed& p, int np, int rows, int DP, bool norm, int pad = 128) {
  p.rows_p = up_to(rows, pad);
  p.rows_all = np * p.rows_p;
  p.hi = a.take<__half>((size_t)p.rows_all * DP * 2);
  p.lo = p.hi + (size_t)p.rows_all * DP;
  const int tiles = p.rows_all / (kTileElems / DP);
  p.inv = a.take<float>(tiles);
  p.norm = norm ? a.take<float>(tiles) : nullptr;
}

// The operand's maps: boxes of a row tile (128 rows), of a streamed tile.
Error maps(EncodeTiled enc, Packed& p, int DP, bool rows, bool stream) {
  const int KN = kTileElems / DP;
  Error e;
  if (rows || KN == 128) e = plane_map(enc, &p.map128, p.hi, 2ll * p.rows_all, DP, 128);
  if (KN == 128) p.mapKN = p.map128;
  else if (e.ok() && stream) e = plane_map(enc, &p.mapKN, p.hi, 2ll * p.rows_all, DP, KN);
  return e;
}

void add_source(PackDev& d, const CrossDev& c, const HeadsDev& x, const Packed& p, int G, int T, bool keys, int DP) {
  PackSrc& s = d.s[d.n];
  s.x = x;
  s.G = G;
  s.T = T;
  s.f_T = make_fastdiv((uint32_t)T);
  s.keys = keys;
  s.rows_p = p.rows_p;
  s.hi = p.hi;
  s.lo = p.lo;
  s.inv = p.inv;
  s.norm = p.norm;
  s.sign = 1.f;
  if (d.n == 0) d.first[0] = 0;
  d.first[d.n + 1] = d.first[d.n] + (uint32_t)(p.rows_all / (kTileElems / DP));
  ++d.n;
}

Error run_pack(PackDev& d, const CrossDev& c, int DP, int* nonfinite, cudaStream_t stream) {
  d.Hk = c.Hk;
  d.D = c.D;
  d.len = c.len;
  d.len64 = c.len64;
  d.len_s = c.len_s;
  d.Tk = c.Tk;
  d.lse = c.lse;
  d.ls_b = c.ls_b;
  d.ls_h = c.ls_h;
  d.ls_t = c.ls_t;
  d.nonfinite = nonfinite;
  auto k = DP == 64 ? (c.vec ? cross_pack_kernel<64, true> : cross_pack_kernel<64, false>)
                    : (c.vec ? cross_pack_kernel<128, true> : cross_pack_kernel<128, false>);
  k<<<d.first[d.n], 256, 0, stream>>>(d);
  return check_launch("cross attention pack kernel");
}

Error too_large(const CrossDev& c) {
  // planes of rows and their lo half within a tensor map's 31-bit coordinate
  const int64_t np = (int64_t)c.B * c.Hk;
  if (np * (c.M + 256ll) >= (1ll << 29) || np * (c.Tk + 256ll) >= (1ll << 29))
    return make_error(TRS_ERR_SHAPE, "cross_attention: 2^29 or more rows of all heads");
  return Error{};
}

template <int DP, int DE, int MT>
Error launch_forward(const Packed& q, const Packed& k, const Packed& v, FwdDev& f, cudaStream_t stream) {
  using S = FwdShape<DP, MT>;
  auto kern = cross_forward_kernel<DP, DE, MT>;
  allow_smem((const void*)kern, S::smem);
  f.items = f.mtiles * f.c.B * f.c.Hk * f.splits;
  return launch_after(kern, dim3((unsigned)std::min(f.items, current_device_info().sm_count)), S::threads, S::smem, stream,
                      "cross attention forward kernel", q.map128, k.mapKN, v.mapKN, f);
}

template <int DP, int DE, bool KV>
Error launch_backward(const Packed& a1, const Packed& a2, const Packed& b1, const Packed& b2, BwdDev& f,
                      cudaStream_t stream) {
  using S = BwdShape<DP>;
  auto kern = cross_backward_kernel<DP, DE, KV>;
  allow_smem((const void*)kern, S::smem);
  f.items = f.mtiles * f.c.B * f.c.Hk * f.splits;
  return launch_after(kern, dim3((unsigned)std::min(f.items, current_device_info().sm_count)), S::threads, S::smem, stream,
                      KV ? "cross attention key gradient kernel" : "cross attention query gradient kernel", a1.map128,
                      a2.map128, b1.mapKN, b2.mapKN, f);
}

void add_sum(SumOne& s, const float* part, const HeadsDev& out, int splits, int rows_p, int G, int T, int np, int DP) {
  s.part = part;
  s.out = out;
  s.splits = splits;
  s.rows_p = rows_p;
  s.G = G;
  s.T = T;
  s.f_T = make_fastdiv((uint32_t)T);
  s.n = (int64_t)np * G * T * (DP / 4);
}

// Zeroed words: one that the pack kernel sets when an input is not finite, and
// the item counters of the two gradient kernels.
Error flag_word(Scratch& flag, CrossDev& c, cudaStream_t stream, int** word) {
  Error e = flag.alloc(3 * sizeof(int), stream);
  if (!e.ok()) return e;
  const cudaError_t ce = cudaMemsetAsync(flag.get(), 0, 3 * sizeof(int), stream);
  if (ce != cudaSuccess) return cuda_error(ce, "cudaMemsetAsync");
  *word = flag.as<int>();
  c.nonfinite = *word;
  return Error{};
}

// Parts of a walk of `tiles` column tiles so that `ctas` items fill the SMs;
// every part walks two tiles at least.  Whole walks and parts: 32 queries of 32
// heads on 32768 keys of 4 heads 1344 and 120 us, 200 queries of 4 x 8 heads on
// 2048 keys 61 and 47, the gradient of 333 on 777 of 3 x 2 heads 140 and 111
// (with the forward).
int pick_splits(int64_t ctas, int tiles) {
  const int sms = current_device_info().sm_count;
  int64_t s = ctas >= sms ? 1 : sms / ctas;
  if (s > tiles / 2) s = tiles / 2;
  return s < 1 ? 1 : (int)s;
}

}  // namespace

Error cross_tc_forward(const CrossDev& call, cudaStream_t stream) {
  CrossDev c = call;
  Error e = too_large(c);
  if (!e.ok()) return e;
  Scratch flag;
  int* nonfinite = nullptr;
  e = flag_word(flag, c, stream, &nonfinite);
  if (!e.ok()) return e;
  EncodeTiled enc = encode_fn(&e);
  if (!enc) return e;
  const int DP = c.D <= 64 ? 64 : 128, KN = kTileElems / DP, np = c.B * c.Hk;
  // two row tiles a CTA as soon as there are two: K and V are read once for both,
  // and one softmax overlaps the other's products (4 x 16 heads, 2048 queries on
  // 2048 keys, with the split: 225 us against 287 with one; 1024 on 1500: 80 and 85)
  const int MT = c.M > 128 ? 2 : 1;
  FwdDev f;
  std::memset(static_cast<void*>(&f), 0, sizeof(f));
  f.c = c;
  f.mtiles = (c.M + MT * 128 - 1) / (MT * 128);
  f.splits = pick_splits((int64_t)f.mtiles * np, (c.Tk + KN - 1) / KN);
  Packed q, k, v;
  Scratch buf;
  for (int pass = 0; pass < 2; ++pass) {
    Arena a;
    if (pass) a.base = buf.as<char>();
    place(a, q, np, c.M, DP, false, MT * 128);
    place(a, k, np, c.Tk, DP, false);
    place(a, v, np, c.Tk, DP, false);
    if (f.splits > 1) {
      const size_t rows = (size_t)f.splits * np * q.rows_p;
      f.part = a.take<float>(rows * DP);
      f.part_m = a.take<float>(rows);
      f.part_l = a.take<float>(rows);
    }
    if (!pass) {
      e = buf.alloc(a.used, stream);
      if (!e.ok()) return e;
    }
  }
  e = maps(enc, q, DP, true, false);
  if (e.ok()) e = maps(enc, k, DP, false, true);
  if (e.ok()) e = maps(enc, v, DP, false, true);
  if (!e.ok()) return e;
  PackDev p;
  std::memset(static_cast<void*>(&p), 0, sizeof(p));
  add_source(p, c, c.q, q, c.G, c.Tq, false, DP);
  if (c.scale < 0.f) p.s[0].sign = -1.f;
  add_source(p, c, c.k, k, 1, c.Tk, true, DP);
  add_source(p, c, c.v, v, 1, c.Tk, true, DP);
  e = run_pack(p, c, DP, nonfinite, stream);
  if (!e.ok()) return e;
  f.q = q.planes();
  f.k = k.planes();
  f.v = v.planes();
  f.f = fabsf(c.scale) * kLog2e;
  f.err = async_error_word();
  if (DP == 64) e = MT == 2 ? launch_forward<64, 64, 2>(q, k, v, f, stream) : launch_forward<64, 64, 1>(q, k, v, f, stream);
  else if (c.D <= 96) e = MT == 2 ? launch_forward<128, 96, 2>(q, k, v, f, stream) : launch_forward<128, 96, 1>(q, k, v, f, stream);
  else e = MT == 2 ? launch_forward<128, 128, 2>(q, k, v, f, stream) : launch_forward<128, 128, 1>(q, k, v, f, stream);
  if (!e.ok() || f.splits == 1) return e;
  return cross_join(c, f.splits, q.rows_p, DP, f.part, f.part_m, f.part_l, stream);
}

Error cross_tc_backward(const CrossDev& call, cudaStream_t stream) {
  CrossDev c = call;
  Error e = too_large(c);
  if (!e.ok()) return e;
  Scratch flag;
  int* nonfinite = nullptr;
  e = flag_word(flag, c, stream, &nonfinite);
  if (!e.ok()) return e;
  EncodeTiled enc = encode_fn(&e);
  if (!enc) return e;
  const int DP = c.D <= 64 ? 64 : 128, KN = kTileElems / DP, np = c.B * c.Hk;
  BwdDev q_d, k_d;
  std::memset(static_cast<void*>(&q_d), 0, sizeof(q_d));
  q_d.c = c;
  q_d.f = fabsf(c.scale) * kLog2e;
  q_d.next = nonfinite + 1;
  q_d.err = async_error_word();
  k_d = q_d;
  k_d.next = nonfinite + 2;
  q_d.mtiles = (c.M + 127) / 128;
  q_d.splits = pick_splits((int64_t)q_d.mtiles * np, (c.Tk + KN - 1) / KN);
  int e2 = 0;
  q_d.out_scale = 2.f * frexpf(c.scale, &e2);
  q_d.out_pow = ldexpf(1.f, e2 - 1);
  k_d.mtiles = (c.Tk + 127) / 128;
  k_d.splits = pick_splits((int64_t)k_d.mtiles * np, (c.M + KN - 1) / KN);
  k_d.out_scale = fabsf(q_d.out_scale);
  k_d.out_pow = q_d.out_pow;
  Packed q, k, v, g;
  float *bias = nullptr, *delta = nullptr, *rnorm = nullptr, *dmax = nullptr;
  Scratch buf;
  for (int pass = 0; pass < 2; ++pass) {
    Arena a;
    if (pass) a.base = buf.as<char>();
    place(a, q, np, c.M, DP, false);
    place(a, g, np, c.M, DP, true);
    place(a, k, np, c.Tk, DP, false);
    place(a, v, np, c.Tk, DP, true);
    bias = a.take<float>(q.rows_all);
    delta = a.take<float>(q.rows_all);
    rnorm = a.take<float>(q.rows_all);
    dmax = a.take<float>(q.rows_all / KN);
    if (q_d.splits > 1) q_d.part1 = a.take<float>((size_t)q_d.splits * q.rows_all * DP);
    if (k_d.splits > 1) {
      k_d.part1 = a.take<float>((size_t)k_d.splits * k.rows_all * DP);
      k_d.part2 = a.take<float>((size_t)k_d.splits * k.rows_all * DP);
    }
    if (!pass) {
      e = buf.alloc(a.used, stream);
      if (!e.ok()) return e;
    }
  }
  for (Packed* x : {&q, &g, &k, &v}) {
    e = maps(enc, *x, DP, true, true);
    if (!e.ok()) return e;
  }
  if (!e.ok()) return e;
  PackDev p;
  std::memset(static_cast<void*>(&p), 0, sizeof(p));
  add_source(p, c, c.q, q, c.G, c.Tq, false, DP);
  if (c.scale < 0.f) p.s[0].sign = -1.f;
  add_source(p, c, c.k, k, 1, c.Tk, true, DP);
  add_source(p, c, c.v, v, 1, c.Tk, true, DP);
  add_source(p, c, c.dout, g, c.G, c.Tq, false, DP);
  PackSrc& gs = p.s[3];
  gs.grad = 1;
  gs.out = c.out;
  gs.bias = bias;
  gs.delta = delta;
  gs.rnorm = rnorm;
  gs.dmax = dmax;
  e = run_pack(p, c, DP, nonfinite, stream);
  if (!e.ok()) return e;
  for (BwdDev* x : {&q_d, &k_d}) {
    x->bias = bias;
    x->delta = delta;
    x->rnorm = rnorm;
    x->dmax = dmax;
  }
  q_d.a1 = q.planes();
  q_d.a2 = g.planes();
  q_d.b1 = k.planes();
  q_d.b2 = v.planes();
  k_d.a1 = k.planes();
  k_d.a2 = v.planes();
  k_d.b1 = q.planes();
  k_d.b2 = g.planes();
  e = DP == 64      ? launch_backward<64, 64, false>(q, g, k, v, q_d, stream)
      : c.D <= 96 ? launch_backward<128, 96, false>(q, g, k, v, q_d, stream)
                    : launch_backward<128, 128, false>(q, g, k, v, q_d, stream);
  if (!e.ok()) return e;
  e = DP == 64      ? launch_backward<64, 64, true>(k, v, q, g, k_d, stream)
      : c.D <= 96 ? launch_backward<128, 96, true>(k, v, q, g, k_d, stream)
                    : launch_backward<128, 128, true>(k, v, q, g, k_d, stream);
  if (!e.ok()) return e;
  if (q_d.splits > 1 || k_d.splits > 1) {
    SumDev sd;
    std::memset(static_cast<void*>(&sd), 0, sizeof(sd));
    sd.np = np;
    sd.ld = DP;
    sd.Hk = c.Hk;
    sd.D = c.D;
    sd.nonfinite = nonfinite;
    int m = 0;
    int64_t most = 0;
    if (q_d.splits > 1) add_sum(sd.r[m++], q_d.part1, c.dq, q_d.splits, q.rows_p, c.G, c.Tq, np, DP);
    if (k_d.splits > 1) {
      add_sum(sd.r[m++], k_d.part1, c.dk, k_d.splits, k.rows_p, 1, c.Tk, np, DP);
      add_sum(sd.r[m++], k_d.part2, c.dv, k_d.splits, k.rows_p, 1, c.Tk, np, DP);
    }
    for (int i = 0; i < m; ++i) most = std::max(most, sd.r[i].n);
    e = launch_after(cross_sum_kernel, dim3((unsigned)((most + 255) / 256), (unsigned)m), 256, 0, stream,
                     "cross attention sum kernel", sd);
  }
  return e;
}

}  // namespace trs
