// head_few.cu -- a model's last layer with its loss for few rows: the weight
// is read in f32, once for 8 or 16 rows, and HBM bounds it all.
//
//   head_rows_kernel     scores: teams of warps take 16 vocabulary rows at a time.  f32
//                        by three TF32 products (mma.sync: HBM sets the pace, and a
//                        result lies whole with one lane, so that no shuffles fold
//                        it); then the softmax's running maximum and sum, or dx
//   head_columns_kernel  dw = dx^T h and its part of dh = dx w: a warp per 128 (9 to
//                        16 rows: 64) columns walks down the vocabulary, h and dh of
//                        its columns in registers, the weight through a ring of bulk
//                        copies of its own
//   head_grad_kernel     the same for weights whose rows bulk copies cannot take (off
//                        16 bytes, or columns apart), by plain loads
//   head_grad_join_kernel  dh from the parts of the vocabulary, in order
//
// TF32 products: x = hi + lo, 11 significant bits each; lo hi + hi lo + hi hi, with
// the sums taken over to f32 additions every 16 elements, since the tensor core cuts
// instead of rounding (the small products first; all of a warp's columns in one sum:
// 1.1e-6 of the lse of rows of 2944 and more).
//
// Measured, 32000 x 1024 (131 MB): scores of 4 rows 31 us (of 131072 x 1024 97: 5.5
// TB/s), dw and dh of 8 rows 51 us (262 MB read and written: 5.1 TB/s).  On the way:
// dot products on the CUDA cores, two steps of 512 bytes per warp in flight, 31 us
// for 4 rows and 44 for 8; a ring of bulk copies per CTA 36 and 40, per warp 39 and
// 45; the gradient of the columns on the CUDA cores 63.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <string>

#include "../../include/trs.h"
#include "head.h"

namespace trs {
namespace {

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

// Four elements of row p from column c on; zeros behind the width.
template <bool VEC>
__device__ __forceinline__ float4 head_load4(const float* p, int c, int D, int64_t sd) {
  if (VEC) return c < D ? __ldg(reinterpret_cast<const float4*>(p + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
  float4 r;
  r.x = c < D ? p[c * sd] : 0.f;
  r.y = c + 1 < D ? p[(c + 1) * sd] : 0.f;
  r.z = c + 2 < D ? p[(c + 2) * sd] : 0.f;
  r.w = c + 3 < D ? p[(c + 3) * sd] : 0.f;
  return r;
}

// D += A B for A 16 x 8 (row major), B 8 x 8, in TF32: the upper 19 bits of each
// element are read.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo; the tensor core reads the upper 11 bits of lo.  hi: x's upper 11
// significant bits for the weight, and for the other operand x rounded to 11 (to the
// largest such number where that would overflow), so that lo has either sign and the
// products lo lo, which are left out, add up to nothing (both cut: 3e-7 of every sum,
// and ten times that of the gradients of scores of 10; both rounded: 2 us of 32).
__device__ __forceinline__ void tf32_cut(float x, uint32_t* hi, uint32_t* lo) {
  *hi = __float_as_uint(x) & 0xFFFFE000u;
  *lo = __float_as_uint(x - __uint_as_float(*hi));
}
__device__ __forceinline__ void tf32_split(float x, uint32_t* hi, uint32_t* lo) {
  const float top = __uint_as_float(0x7F7FE000u);
  const float h = fminf(fmaxf(__uint_as_float((__float_as_uint(x) + 0x1000u) & 0xFFFFE000u), -top), top);
  *hi = __float_as_uint(h);
  *lo = __float_as_uint(x - h);
}

// The call rows of this block and, from shared memory [NR][pitch], their elements
// (zeros behind the width and for rows without a target).
template <int NR>
__device__ __forceinline__ void few_hidden(const HeadDev& d, int r0, int blocks, float* s_h, int* s_row) {
  const int pitch = blocks * 16 + 16;
  if (threadIdx.x < NR) {
    const int r = r0 + threadIdx.x;
    s_row[threadIdx.x] = r < d.N && head_first_id(d, r) != kNoToken ? r : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NR * blocks * 4; i += blockDim.x) {
    const int n = i / (blocks * 4), c = i % (blocks * 4) * 4;
    *reinterpret_cast<float4*>(&s_h[n * pitch + c]) =
        s_row[n] < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
        : d.vec_h    ? head_load4<true>(head_row<const float>(d, d.hid, s_row[n]), c, d.D, 1)
                     : head_load4<false>(head_row<const float>(d, d.hid, s_row[n]), c, d.D, d.hid.sd);
  }
}

// part += one block of 16 columns: y, 4 columns (4 lt and on) of vocabulary rows lg
// and lg + 8, which the lane supplies to two MMAs; the order of the columns inside a
// block does not matter as long as the hidden rows take the same.
template <int NT>
__device__ __forceinline__ void few_block(const float4 (&y)[2], const float* h, int pitch, float (&part)[NT][4]) {
  uint32_t hi[2][4], lo[2][4];  // [columns 0 and 1, columns 2 and 3]
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    tf32_cut(y[j].x, &hi[0][j], &lo[0][j]);
    tf32_cut(y[j].y, &hi[0][2 + j], &lo[0][2 + j]);
    tf32_cut(y[j].z, &hi[1][j], &lo[1][j]);
    tf32_cut(y[j].w, &hi[1][2 + j], &lo[1][2 + j]);
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const float4 x = *reinterpret_cast<const float4*>(h + i * 8 * pitch);
    uint32_t hh[4], hl[4];
    tf32_split(x.x, &hh[0], &hl[0]);
    tf32_split(x.y, &hh[1], &hl[1]);
    tf32_split(x.z, &hh[2], &hl[2]);
    tf32_split(x.w, &hh[3], &hl[3]);
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      mma_tf32(sum, lo[k], hh[2 * k], hh[2 * k + 1]);
      mma_tf32(sum, hi[k], hl[2 * k], hl[2 * k + 1]);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) mma_tf32(sum, hi[k], hh[2 * k], hh[2 * k + 1]);
#pragma unroll
    for (int j = 0; j < 4; ++j) part[i][j] += sum[j];
  }
}
struct HeadRowsDev {
  HeadDev d;
  int blocks;            // the width in blocks of 16, rounded up
  HeadPart* part;        // forward: [row][CTA]
  float* dx;             // backward, of up to 8 NT rows: [V][8 NT]
  int lg;                // 2^lg warps share a row's columns
};

// ---- scores --------------------------------------------------------------------------------

constexpr int kFewThreads = 512;
constexpr int kAhead = 4;    // blocks of 16 columns in flight per warp (6: 34.6 us against 32.7, for the registers)

// Teams of 2^lg warps take groups of 16 vocabulary rows, a warp its share of their
// columns (so that what a CTA reads at a time are whole rows: a warp that reads 64
// bytes each of rows of its own leaves DRAM's pages half used, 45 us for 131 MB
// instead of 31).  The results of G groups meet in shared memory, where every
// thread finishes some of them, always of one call row.
template <int NT, bool VEC, bool GRAD>
__global__ void __launch_bounds__(kFewThreads, 1) head_rows_kernel(const __grid_constant__ HeadRowsDev a) {
  constexpr int W = kFewThreads / 32, NR = 8 * NT, G = 4 / NT;
  extern __shared__ float4 s_raw[];
  __shared__ int s_row[NR];
  const HeadDev& d = a.d;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r0 = blockIdx.y * NR;
  const int lg = lane / 4, lt = lane % 4, pitch = a.blocks * 16 + 16;
  const int ts = 1 << a.lg, teams = W >> a.lg, team = warp >> a.lg, me = warp & (ts - 1), tid = threadIdx.x & (ts * 32 - 1);
  float4* red = s_raw + team * (G * NT * ts * 32);               // [G][NT][ts][32]
  float* s_h = reinterpret_cast<float*>(s_raw + G * NT * W * 32);  // [NR][pitch]
  auto team_sync = [&] {
    if (ts == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(ts * 32) : "memory");
  };
  pdl_launch_dependents();
  pdl_wait();
  const int share = (a.blocks + ts - 1) / ts, b0 = me * share, n = max(0, min(share, a.blocks - b0));  // this warp's blocks
  const int groups = (d.V + 15) / 16, hop = gridDim.x * teams, g0 = blockIdx.x * teams + team;
  int gl = g0, bl = 0;                                           // the loads' group and block
  const float* wl[2];
  auto rows = [&] {
#pragma unroll
    for (int j = 0; j < 2; ++j) wl[j] = d.w + (int64_t)min(gl * 16 + lg + 8 * j, d.V - 1) * d.wv + (VEC ? b0 * 16 + lt * 4 : 0);
  };
  rows();
  auto fetch = [&](float4 (&x)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (VEC) {
        x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (gl < groups && (b0 + bl) * 16 + lt * 4 < d.D)
          asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(x[j].x), "=f"(x[j].y), "=f"(x[j].z), "=f"(x[j].w)
                       : "l"(wl[j] + bl * 16));
      } else {
        x[j] = gl < groups ? head_load4<false>(wl[j], (b0 + bl) * 16 + lt * 4, d.D, d.wd) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if (++bl == n) {
      bl = 0;
      gl += hop;
      rows();
    }
  };
  float4 x[kAhead][2];
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(x[i]);
  }
  few_hidden<NR>(d, r0, a.blocks, s_h, s_row);
  __syncthreads();
  // what this thread finishes: call row fn, of every batch the values tid, tid + 32 ts, ..
  const int fn = tid % NR, row = s_row[fn];
  Entries ent;
  ent.left = 0;
  ent.next = kNoToken;
  float lse2 = 0.f, gr = 0.f;
  const float f = d.inv_temp * kHeadLog2e;
  if (row >= 0) {
    if (d.distill) ent.begin(d, row);
    else ent.next = head_id(d, d.ids, row, 0);
    if (GRAD) {
      lse2 = *head_row<const float>(d, d.lse, row) * kHeadLog2e;
      gr = *head_row<const float>(d, d.gl, row) * d.temp;
    }
  }
  // from the lowest finite maximum: a first score of -inf adds 0, not the NaN of inf - inf
  HeadPart pt = {-FLT_MAX, 0.f, 0.f, 0.f};
  float* dx = a.dx;
  float part[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[i][j] = 0.f;
  int g = g0, b = 0, batch = 0;
  const float* h0 = s_h + lg * pitch + b0 * 16 + lt * 4;
  auto finish = [&] {  // the warp's results of group g; the batch, when it is whole
    if (batch == 0) team_sync();  // the batch before has been read
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      red[((batch * NT + i) * ts + me) * 32 + lane] = make_float4(part[i][0], part[i][1], part[i][2], part[i][3]);
#pragma unroll
      for (int j = 0; j < 4; ++j) part[i][j] = 0.f;
    }
    g += hop;
    if (++batch < G && g < groups) return;
    team_sync();
    for (int q = tid / NR; q < batch * 16; q += ts * 32 / NR) {
      // the result of (vocabulary row fv, fn) lies with lane (fv % 8) * 4 + fn % 8 / 2, element fv / 8 * 2 + fn % 2
      const int fj = q / 16, fv = q % 16, v = (g - (batch - fj) * hop) * 16 + fv;
      const float* p = reinterpret_cast<const float*>(red + (fj * NT + fn / 8) * ts * 32 + (fv % 8) * 4 + fn % 8 / 2) + fv / 8 * 2 + fn % 2;
      float z = p[0];
      for (int i = 1; i < ts; ++i) z += p[i * 128];
      z *= f;  // in units of log2
      if (v >= d.V) continue;
      float t = 0.f;
      if (ent.next <= v) {
        if (d.distill) {
          if (ent.next < v) ent.skip_to(v);
          t = ent.take(v);
        } else if (ent.next == v) {
          t = d.weight;
        }
      }
      if (GRAD) {
        dx[(int64_t)v * NR + fn] = row < 0 ? 0.f : gr * (head_softmax(z - lse2) - t - d.share);
      } else {
        const float m = fmaxf(pt.m, z);  // passes over a NaN, which makes the sum NaN for good
        pt.s = pt.s * head_ex2(pt.m - m) + head_ex2(z - m);
        pt.m = m;
        if (t != 0.f) pt.dot = __fmaf_rn(t, z, pt.dot);
        pt.sum += z;
      }
    }
    batch = 0;
  };
  if (n == 0) {  // more warps than blocks: only the meetings
    while (g < groups) finish();
  } else {
    while (g < groups) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (g >= groups) break;
        few_block<NT>(x[i], h0 + b * 16, pitch, part);
        fetch(x[i]);
        if (++b == n) {
          b = 0;
          finish();
        }
      }
    }
  }
  if (GRAD) return;
  // the CTA's part of a row: 512 / NR threads, folded in a fixed order
  HeadPart* sp = reinterpret_cast<HeadPart*>(s_raw);
  const int q = threadIdx.x / NR;
  __syncthreads();
  sp[threadIdx.x] = pt;
  for (int k = kFewThreads / NR / 2; k > 0; k /= 2) {
    __syncthreads();
    HeadPart y;
    if (q < k) y = head_add(sp[2 * q * NR + fn], sp[(2 * q + 1) * NR + fn]);
    __syncthreads();
    if (q < k) sp[q * NR + fn] = y;
  }
  if (q == 0 && r0 + fn < d.N) a.part[(int64_t)(r0 + fn) * gridDim.x + blockIdx.x] = sp[fn];
}

// ---- the gradients -------------------------------------------------------------------------

struct HeadGradDev {
  HeadDev d;
  int lg;                // head_grad_kernel: 2^lg threads along the width, the rest along the vocabulary
  int slices, parts;     // head_columns_kernel: warps along the width, along the vocabulary
  const float* dx;
  float* part;           // [part of the vocabulary][NR][D] of dh
  int* err;
};

constexpr int kColSteps = 3;                 // steps of 16 vocabulary rows in flight
constexpr int kColWarps = 8;
// A warp's columns, and its rows in shared memory: four rows' 32 bytes lie in different
// banks.
template <int NT> constexpr int kColumns = 128 / NT;
template <int NT> constexpr int kColPitch = kColumns<NT> + 8;
template <int NT> constexpr int kColStep = 16 * kColPitch<NT>;  // floats

__device__ __forceinline__ bool step_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0;
}

// Rows [v, v + rows) of the weight, `bytes` of each from column c on, by one copy per
// lane, into rows of PITCH floats.
template <int PITCH>
__device__ __forceinline__ void step_copy(const HeadDev& d, float* to, int64_t v, int rows, int c, uint32_t bytes, uint64_t* bar,
                                          int lane) {
  fence_proxy_async();  // what was read here has been read
  if (lane == 0) mbar_arrive_expect_tx(bar, bytes * rows);
  __syncwarp();
  if (lane < rows) bulk_g2s(to + lane * PITCH, d.w + (v + lane) * d.wv + c, bytes, bar);
}

// dw and a part of dh of 8 NT call rows for 128 / NT columns per warp: as many warps as
// the width takes, one after another, then the next part of the vocabulary, 16 rows of
// it a step.
//   dw: rows of dx as the left operand, h as the right one, in registers for good:
//       column 4 (m / 2) + m % 2 of a block of 16 is column m of one MMA, the one 2
//       to its right of the other, so that a lane ends with four neighbours
//   dh^T += w^T dx: 4 neighbouring columns of a lane are the rows of four MMAs
template <int NT>
__global__ void __launch_bounds__(kColWarps * 32, 1) head_columns_kernel(const __grid_constant__ HeadGradDev a) {
  constexpr int CW = kColumns<NT>, NB = CW / 16, HF = CW / 64, PITCH = kColPitch<NT>, STEP = kColStep<NT>;
  extern __shared__ float4 s_raw[];
  __shared__ uint64_t full[kColWarps][kColSteps];
  const HeadDev& d = a.d;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, lg = lane / 4, lt = lane % 4;
  const int at_w = blockIdx.x * kColWarps + warp, parts = a.parts, part = at_w / a.slices, c0 = at_w % a.slices * CW;
  float* ring = reinterpret_cast<float*>(s_raw) + warp * (kColSteps * STEP);
  pdl_launch_dependents();
  pdl_wait();
  if (part >= parts) return;
  if (lane == 0) {
    for (int s = 0; s < kColSteps; ++s) mbar_init(&full[warp][s], 1);
    fence_mbar_init();
  }
  // what no copy writes only has to be finite: it meets zeros of dx, or columns that nothing takes
  for (int i = lane; i < kColSteps * STEP / 4; i += 32) reinterpret_cast<float4*>(ring)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  __syncwarp();
  const int groups = (d.V + 15) / 16, g1 = (int)((int64_t)groups * (part + 1) / parts);
  int g = (int)((int64_t)groups * part / parts), gl = g;
  const uint32_t bytes = (uint32_t)min(CW, d.D - c0) * 4;
  const bool want_h = d.dh.p != nullptr;
  auto copy = [&](int s) {
    if (!want_h || gl >= g1) return;
    step_copy<PITCH>(d, ring + s * STEP, (int64_t)gl * 16, min(16, d.V - gl * 16), c0, bytes, &full[warp][s], lane);
    ++gl;
  };
#pragma unroll
  for (int s = 0; s < kColSteps; ++s) copy(s);
  // h of the warp's columns: [block of 16][its two MMAs][eight rows][hidden rows lt, lt + 4 of them]
  uint32_t hh[NB][2][NT][2], hl[NB][2][NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float* row[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = n * 8 + lt + 4 * e;
      row[e] = r < d.N && head_first_id(d, r) != kNoToken ? head_row<const float>(d, d.hid, r) : nullptr;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = c0 + b * 16 + 4 * (lg / 2) + lg % 2 + 2 * q;
          tf32_split(row[e] && c < d.D ? row[e][c * d.hid.sd] : 0.f, &hh[b][q][n][e], &hl[b][q][n][e]);
        }
  }
  float acc[4 * HF][NT][4];  // dh^T: [half of 64 columns, column 4 lg + i][..]
#pragma unroll
  for (int i = 0; i < 4 * HF; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.f;
  // dx of a group: this lane's elements of both operands
  float xa[NT][4], xb[NT][4];
  auto fetch = [&](int at) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t va = (int64_t)at * 16 + lg + e % 2 * 8, vb = (int64_t)at * 16 + lt + 4 * e;
        xa[n][e] = at < g1 && va < d.V ? a.dx[va * (8 * NT) + n * 8 + lt + e / 2 * 4] : 0.f;
        xb[n][e] = at < g1 && vb < d.V ? a.dx[vb * (8 * NT) + n * 8 + lg] : 0.f;
      }
  };
  fetch(g);
  const float* w0 = ring + lt * PITCH + 4 * lg;
  int slot = 0, phase = 0;
  bool ok = true;
  for (; g < g1; ++g) {
    uint32_t ah[NT][4], al[NT][4], bh[NT][4], bl[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        tf32_split(xa[n][e], &ah[n][e], &al[n][e]);
        tf32_split(xb[n][e], &bh[n][e], &bl[n][e]);
      }
    fetch(g + 1);
    if (d.dw) {
      const int64_t v = (int64_t)g * 16 + lg;
      float* to[2] = {d.dw + v * d.dwv + (c0 + 4 * lt) * d.dwd, d.dw + (v + 8) * d.dwv + (c0 + 4 * lt) * d.dwd};
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float o[2][4];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[q][e] = 0.f;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_tf32(o[q], al[n], hh[b][q][n][0], hh[b][q][n][1]);
            mma_tf32(o[q], ah[n], hl[b][q][n][0], hl[b][q][n][1]);
            mma_tf32(o[q], ah[n], hh[b][q][n][0], hh[b][q][n][1]);
          }
        }
        const int c = c0 + b * 16 + 4 * lt;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (v + 8 * e >= d.V || c >= d.D) continue;
          const float ys[4] = {o[0][2 * e], o[0][2 * e + 1], o[1][2 * e], o[1][2 * e + 1]};
          if (d.vec_dw) {
            *reinterpret_cast<float4*>(to[e] + b * 16) = make_float4(ys[0], ys[1], ys[2], ys[3]);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (c + k < d.D) to[e][(b * 16 + k) * d.dwd] = ys[k];
          }
        }
      }
    }
    if (!want_h) continue;
    if (ok) ok = step_wait(&full[warp][slot], (uint32_t)phase);
    const float* w = w0 + slot * STEP;
#pragma unroll
    for (int hf = 0; hf < HF; ++hf) {
      float sum[4][NT][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) sum[i][n][j] = 0.f;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        float y[4][4];  // [operand element][column]
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float4 z = *reinterpret_cast<const float4*>(w + (p * 8 + e / 2 * 4) * PITCH + hf * 64 + e % 2 * 32);
          y[e][0] = z.x, y[e][1] = z.y, y[e][2] = z.z, y[e][3] = z.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t wh[4], wl[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) tf32_cut(y[e][i], &wh[e], &wl[e]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_tf32(sum[i][n], wl, bh[n][2 * p], bh[n][2 * p + 1]);
            mma_tf32(sum[i][n], wh, bl[n][2 * p], bl[n][2 * p + 1]);
            mma_tf32(sum[i][n], wh, bh[n][2 * p], bh[n][2 * p + 1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[hf * 4 + i][n][j] += sum[i][n][j];
    }
    copy(slot);
    if (++slot == kColSteps) {
      slot = 0;
      phase ^= 1;
    }
  }
  if (!ok) {  // copies may still be under way
    for (int i = 0; i < 100; ++i) __nanosleep(100000);
    if (lane == 0) atomicOr(a.err, kAsyncWaitTimeout);
  }
  if (!want_h) return;
#pragma unroll
  for (int i = 0; i < 4 * HF; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = c0 + i / 4 * 64 + j / 2 * 32 + 4 * lg + i % 4, r = n * 8 + 2 * lt + j % 2;
        if (c < d.D) a.part[((int64_t)part * (8 * NT) + r) * d.D + c] = acc[i][n][j];
      }
}

// A thread per 4 columns; blockIdx.y and the thread's group: a range of the
// vocabulary.
__global__ void __launch_bounds__(256, 2) head_grad_kernel(const __grid_constant__ HeadGradDev a) {
  constexpr int NR = 8, U = 4;  // U: rows of the vocabulary in flight
  const HeadDev& d = a.d;
  pdl_launch_dependents();
  const int c = (blockIdx.x * 256 + (threadIdx.x & ((1 << a.lg) - 1))) * 4;
  const int groups = 256 >> a.lg, part = blockIdx.y * groups + (threadIdx.x >> a.lg), parts = gridDim.y * groups;
  pdl_wait();
  uint64_t h[NR][2], acc[NR][2];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < d.N && head_first_id(d, i) != kNoToken) x = head_load4<false>(head_row<const float>(d, d.hid, i), c, d.D, d.hid.sd);
    h[i][0] = pk(x.x, x.y), h[i][1] = pk(x.z, x.w);
    acc[i][0] = acc[i][1] = 0;
  }
  const float* dx = a.dx;
  const int lane = threadIdx.x % 32;
  const int64_t v1 = (int64_t)d.V * (part + 1) / parts;
  int64_t v = (int64_t)d.V * part / parts;
  // U rows of the weight, and one of their score gradients per lane
  auto fetch = [&](float4 (&w)[U], float& x, int64_t at) {
    x = at + lane / NR < v1 ? dx[at * NR + lane] : 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      w[j] = d.dh.p && at + j < v1 ? head_load4<false>(d.w + (at + j) * d.wv, c, d.D, d.wd) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  auto work = [&](float4 (&w)[U], float xs) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      uint64_t o0 = 0, o1 = 0;
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        const float x = __shfl_sync(0xffffffffu, xs, j * NR + i);
        const uint64_t xx = pk(x, x);
        if (d.dh.p) {
          acc[i][0] = fma2(xx, pk(w[j].x, w[j].y), acc[i][0]);
          acc[i][1] = fma2(xx, pk(w[j].z, w[j].w), acc[i][1]);
        }
        o0 = fma2(xx, h[i][0], o0);
        o1 = fma2(xx, h[i][1], o1);
      }
      if (!d.dw || v + j >= v1 || c >= d.D) continue;
      float o[4];
      upk(o0, &o[0], &o[1]);
      upk(o1, &o[2], &o[3]);
      float* to = d.dw + (v + j) * d.dwv;
      if (d.vec_dw) {
        __stcs(reinterpret_cast<float4*>(to + c), make_float4(o[0], o[1], o[2], o[3]));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < d.D) to[(c + k) * d.dwd] = o[k];
      }
    }
    v += U;
  };
  float4 wa[U], wb[U];
  float xa, xb;
  fetch(wa, xa, v);
  while (v < v1) {
    fetch(wb, xb, v + U);
    work(wa, xa);
    if (v >= v1) break;
    fetch(wa, xa, v + U);
    work(wb, xb);
  }
  if (!d.dh.p) return;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    float y[4];
    upk(acc[i][0], &y[0], &y[1]);
    upk(acc[i][1], &y[2], &y[3]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (c + k < d.D) a.part[((int64_t)part * NR + i) * d.D + c + k] = y[k];
  }
}

// dh from its parts, in order: 32 columns times 8 runs of parts
// per CTA; zeros for rows without a target.
__global__ void __launch_bounds__(256) head_grad_join_kernel(const __grid_constant__ HeadGradDev a, int parts, int NR) {
  __shared__ float s[8][32];
  const HeadDev& d = a.d;
  pdl_wait();
  const int c = blockIdx.x * 32 + threadIdx.x % 32, w = threadIdx.x / 32, r = blockIdx.y;
  float sum = 0.f;
  const int p1 = (int)((int64_t)parts * (w + 1) / 8);
  if (c < d.D)
    for (int p = (int)((int64_t)parts * w / 8); p < p1; p += 8) {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = p + j < p1 ? a.part[((int64_t)(p + j) * NR + r) * d.D + c] : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += x[j];
    }
  s[w][threadIdx.x % 32] = sum;
  __syncthreads();
  if (w != 0 || c >= d.D) return;
  for (int i = 1; i < 8; ++i) sum += s[i][threadIdx.x];
  head_row<float>(d, d.dh, r)[c * d.dh.sd] = head_first_id(d, r) != kNoToken ? sum : 0.f;
}

// ---- host side -------------------------------------------------------------------

template <int NT, bool GRAD>
Error launch_scores(HeadRowsDev& a, cudaStream_t s) {
  const HeadDev& d = a.d;
  // 8 blocks per warp, or half as many warps where that leaves fewer of them idle (width
  // 1360: 85 blocks are 16 shares of 6, of which 11 too many, or 8 of 11)
  a.lg = 0;
  while (a.lg < 4 && (8 << a.lg) < a.blocks) ++a.lg;
  auto taken = [&](int lg) { return ((a.blocks + (1 << lg) - 1) >> lg) << lg; };
  if (a.lg > 0 && taken(a.lg - 1) < taken(a.lg)) --a.lg;
  const int teams = (kFewThreads / 32) >> a.lg;
  const int ctas = std::max(1, std::min(current_device_info().sm_count, (d.V + 16 * teams - 1) / (16 * teams)));
  const int smem = 4 * (kFewThreads / 32) * 512 + 8 * NT * (a.blocks + 1) * 64;
  auto k = d.vec_w ? head_rows_kernel<NT, true, GRAD> : head_rows_kernel<NT, false, GRAD>;
  allow_smem((const void*)k, smem);
  Scratch mem;
  Error e;
  if (!GRAD) {
    e = mem.alloc(sizeof(HeadPart) * (size_t)d.N * ctas, s);
    if (!e.ok()) return e;
    a.part = mem.as<HeadPart>();
  }
  e = launch_after(k, dim3((unsigned)ctas, (unsigned)((d.N + 8 * NT - 1) / (8 * NT))), kFewThreads, smem, s, "head rows kernel", a);
  if (e.ok() && !GRAD) e = head_join(d, a.part, ctas, 1, ctas, true, s);
  return e;
}

}  // namespace

Error head_few(const HeadDev& d, bool backward, cudaStream_t s) {
  const int sms = current_device_info().sm_count;
  HeadRowsDev a;
  std::memset(static_cast<void*>(&a), 0, sizeof(a));
  a.d = d;
  a.blocks = (d.D + 15) / 16;
  // 16 rows share one read of the weight where the shared memory holds them
  const int nt = d.N > 8 && d.D <= 2560 ? 2 : 1;
  if (!backward) return nt == 1 ? launch_scores<1, false>(a, s) : launch_scores<2, false>(a, s);
  Scratch mem;
  Error e;
  HeadGradDev g;
  std::memset(static_cast<void*>(&g), 0, sizeof(g));
  g.d = d;
  g.err = async_error_word();
  if (!g.err) return make_error(TRS_ERR_CUDA, "head: no async-error word");
  int parts;  // of the vocabulary
  dim3 grid;
  if (d.vec_w) {
    const int columns = 128 / nt;
    g.slices = (d.D + columns - 1) / columns;
    parts = g.parts = std::max(1, std::min((d.V + 15) / 16, sms * kColWarps / g.slices));
    grid = dim3((unsigned)((g.slices * parts + kColWarps - 1) / kColWarps));
  } else {
    g.lg = 5;
    while (g.lg < 8 && (1 << g.lg) < (d.D + 3) / 4) ++g.lg;
    const int across = (d.D + 1023) / 1024, splits = std::max(1, std::min((d.V + 31) / 32, 2 * sms / across));
    parts = splits * (256 >> g.lg);
    grid = dim3((unsigned)across, (unsigned)splits);
  }
  const size_t nd = (size_t)d.V * 8 * nt;
  e = mem.alloc(sizeof(float) * (nd + (size_t)parts * 8 * nt * d.D), s);
  if (!e.ok()) return e;
  a.dx = mem.as<float>();
  e = nt == 1 ? launch_scores<1, true>(a, s) : launch_scores<2, true>(a, s);
  if (!e.ok()) return e;
  g.dx = a.dx;
  g.part = a.dx + nd;
  if (!d.vec_w) {
    e = launch_after(head_grad_kernel, grid, 256, 0, s, "head gradient kernel", g);
  } else {
    auto k = nt == 1 ? head_columns_kernel<1> : head_columns_kernel<2>;
    const int smem = kColWarps * kColSteps * 4 * (nt == 1 ? kColStep<1> : kColStep<2>);
    allow_smem((const void*)k, smem);
    e = launch_after(k, grid, kColWarps * 32, smem, s, "head columns kernel", g);
  }
  if (!e.ok() || !d.dh.p) return e;
  return launch_after(head_grad_join_kernel, dim3((unsigned)((d.D + 31) / 32), (unsigned)d.N), 256, 0, s,
                      "head gradient join kernel", g, parts, 8 * nt);
}

}  // namespace trs
