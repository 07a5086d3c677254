// head.cu -- the last linear layer of a language model with its loss, without
// the logits: softmax cross entropy against classes, and distillation from a
// teacher's largest logits.
//
//   x = h w^T / temperature, lse = ln sum_v exp x_v
//   cross entropy: loss = lse - (1 - s) x_target - s / V sum_v x_v
//   distillation:  p = softmax(z / temperature) over the teacher's K entries,
//                  loss = temperature^2 sum_j p_j (ln p_j - x_{id_j} + lse)
//   gradient:      dx = g temperature (softmax(x) - t), dh = dx w, dw = dx^T h,
//                  t the target distribution
//
// Rows without a target (masked positions) are listed out first and are not read.
// This file: the checks, the rows' targets (head_teacher_kernel,
// head_list_kernel), the join of the vocabulary's parts, and the kernels for few
// rows, which HBM bounds: the weight is read once in f32 and every element of it
// used for all rows.
//
//   head_rows_kernel  a warp per 16 vocabulary rows, 8 or 16 hidden rows in shared
//                     memory: f32 by three TF32 products (mma.sync, which leaves
//                     every result with one lane and needs no shuffles; HBM, not
//                     the tensor core, sets the pace); then the running maximum and
//                     sum of the softmax per lane, or the gradient of the scores
//   head_grad_kernel  a thread per 4 columns walks vocabulary rows: a row's dw from
//                     the hidden rows in registers, and its part of dh
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "../../include/trs.h"
#include "head.h"

namespace trs {

namespace {

// ---- targets ---------------------------------------------------------------------

constexpr int kMaxEntries = 1024;

__device__ __forceinline__ int head_id(const HeadDev& d, const RowsDev& ids, int row, int k) {
  const int64_t at = k * ids.sd;
  const int64_t v = d.ids64 ? head_row<const int64_t>(d, ids, row)[at] : head_row<const int32_t>(d, ids, row)[at];
  return v < 0 || v >= d.V ? kNoToken : (int)v;
}

// The first of a row's tokens in order (kNoToken: the row has no target).
__device__ __forceinline__ int head_first_id(const HeadDev& d, int row) {
  return d.distill ? d.eid[(int64_t)row * d.K] : head_id(d, d.ids, row, 0);
}

// A warp per row: the softmax of the entries that are there, sorted by token
// (the rank of an entry is counted: K is small).
__global__ void __launch_bounds__(256) head_teacher_kernel(const HeadDev d) {
  extern __shared__ int s_id[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int row = blockIdx.x * 8 + warp;
  pdl_launch_dependents();
  if (row >= d.N) return;
  int* ids = s_id + warp * 2 * d.K;
  float* ps = reinterpret_cast<float*>(ids + d.K);
  const float* z = head_row<const float>(d, d.z, row);
  float top = -INFINITY;
  for (int k = lane; k < d.K; k += 32) {
    const float x = z[k * d.z.sd];
    int id = head_id(d, d.ids, row, k);
    if (x == -INFINITY) id = kNoToken;
    ids[k] = id;
    ps[k] = x;
    if (id != kNoToken) top = fmaxf(top, x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float sum = 0.f;
  for (int k = lane; k < d.K; k += 32)
    if (ids[k] != kNoToken) sum += expf(__fdiv_rn(ps[k] - top, d.temp));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float ln_sum = logf(sum);
  double ent = 0.0;
  for (int k = lane; k < d.K; k += 32) {
    float p = 0.f;
    if (ids[k] != kNoToken) {
      const float a = __fdiv_rn(ps[k] - top, d.temp);
      p = __fdiv_rn(expf(a), sum);
      ent += (double)p * (double)(a - ln_sum);
    }
    ps[k] = p;
  }
  __syncwarp();
  for (int k = lane; k < d.K; k += 32) {
    const int id = ids[k];
    int rank = 0;
    bool first = true;
    float p = 0.f;
    for (int j = 0; j < d.K; ++j) {
      const int other = ids[j];
      rank += other < id || (other == id && j < k);
      if (other == id) {
        first = first && j >= k;
        p += ps[j];
      }
    }
    d.eid[(int64_t)row * d.K + rank] = id;
    d.ew[(int64_t)row * d.K + rank] = first ? p : 0.f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ent += __shfl_xor_sync(0xffffffffu, ent, o);
  if (lane == 0) d.ent[row] = (float)ent;
}

// One CTA: the rows with a target, in order (and a class's one entry); the others
// get their loss and lse of 0.
__global__ void __launch_bounds__(1024) head_list_kernel(const HeadDev d) {
  __shared__ int warps[32];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int done = 0;
  for (int r0 = 0; r0 < d.N; r0 += 1024) {
    const int row = r0 + threadIdx.x;
    int id = kNoToken;
    if (row < d.N) {
      if (d.distill) {
        id = d.eid[(int64_t)row * d.K];
      } else {
        id = head_id(d, d.ids, row, 0);
        d.eid[row] = id;
        d.ew[row] = d.weight;
      }
    }
    const bool there = id != kNoToken;
    if (row < d.N && !there && d.loss.p) {
      *head_row<float>(d, d.loss, row) = 0.f;
      if (d.lse.p) *head_row<float>(d, d.lse, row) = 0.f;
    }
    const uint32_t vote = __ballot_sync(0xffffffffu, there);
    if (lane == 0) warps[warp] = __popc(vote);
    __syncthreads();
    int mine = 0, all = 0;
    {
      const int n = warps[lane];
      int scan = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += y;
      }
      mine = __shfl_sync(0xffffffffu, scan - n, warp);
      all = __shfl_sync(0xffffffffu, scan, 31);
    }
    if (there) d.rows[done + mine + __popc(vote & ((1u << lane) - 1))] = row;
    done += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *d.live = done;
}

// Gradients of rows without a target.
__global__ void __launch_bounds__(256) head_masked_kernel(const HeadDev d) {
  pdl_launch_dependents();
  pdl_wait();
  for (int row = blockIdx.x * 8 + threadIdx.x / 32; row < d.N; row += gridDim.x * 8) {
    if (d.eid[(int64_t)row * d.K] != kNoToken) continue;
    float* to = head_row<float>(d, d.dh, row);
    for (int64_t c = threadIdx.x % 32; c < d.D; c += 32) to[c * d.dh.sd] = 0.f;
  }
}

// ---- joining the parts of the vocabulary -------------------------------------------

__device__ __forceinline__ HeadPart head_add(const HeadPart& a, const HeadPart& b) {
  HeadPart r;
  r.m = fmaxf(a.m, b.m);
  // a part of -inf alone has no sum; and scores of -inf alone stay one
  const float base = r.m == -INFINITY ? 0.f : r.m;
  r.s = a.s * exp2f(a.m - base) + b.s * exp2f(b.m - base);
  r.dot = a.dot + b.dot;
  r.sum = a.sum + b.sum;
  return r;
}

// LR rows per CTA times 256 / LR threads along a row's parts, folded in a fixed
// order.  FEW: parts of the call's rows, not of those with a target, which are
// not listed out; rows without one get their zeros here.
template <int LR, bool FEW>
__global__ void __launch_bounds__(256) head_join_kernel(const HeadDev d, const HeadPart* part, int parts, int64_t sp,
                                                        int64_t sr) {
  constexpr int LP = 256 / LR;
  __shared__ HeadPart s[LP][LR];
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * LR + threadIdx.x % LR, w = threadIdx.x / LR;
  const bool there = FEW ? head_first_id(d, r) != kNoToken : r < *d.live;
  HeadPart a = {-INFINITY, 0.f, 0.f, 0.f};
  if (there) {
    // runs of consecutive parts, so that the order of the sums is that of the vocabulary
    const int p0 = (int)((int64_t)parts * w / LP), p1 = (int)((int64_t)parts * (w + 1) / LP);
    for (int p = p0; p < p1; p += 4) {
      HeadPart x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[j] = p + j < p1 ? part[(p + j) * sp + r * sr] : HeadPart{-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j) a = head_add(a, x[j]);
    }
  }
  s[w][threadIdx.x % LR] = a;
  for (int n = LP / 2; n > 0; n /= 2) {
    __syncthreads();
    if (w < n) a = head_add(s[2 * w][threadIdx.x % LR], s[2 * w + 1][threadIdx.x % LR]);
    __syncthreads();
    if (w < n) s[w][threadIdx.x % LR] = a;
  }
  if (w != 0 || (!FEW && !there)) return;
  const int row = FEW ? r : d.rows[r];
  const double lse = kHeadLn2 * ((double)a.m + log2((double)a.s));
  double loss = lse - kHeadLn2 * (double)a.dot;
  if (d.share != 0.f) loss -= kHeadLn2 * (double)d.share * (double)a.sum;
  if (d.distill) loss = (loss + (double)d.ent[row]) * (double)d.temp * (double)d.temp;
  *head_row<float>(d, d.loss, row) = there ? (float)loss : 0.f;
  if (d.lse.p) *head_row<float>(d, d.lse, row) = there ? (float)lse : 0.f;
}

}  // namespace

Error head_join(const HeadDev& d, const HeadPart* part, int parts, int64_t sp, int64_t sr, bool few,
                cudaStream_t stream) {
  if (few)
    return launch_after(head_join_kernel<1, true>, dim3((unsigned)d.N), 256, 0, stream, "head join kernel", d, part, parts, sp, sr);
  return launch_after(head_join_kernel<8, false>, dim3((unsigned)((d.N + 7) / 8)), 256, 0, stream, "head join kernel", d, part,
                      parts, sp, sr);
}

namespace {

// ---- few rows ----------------------------------------------------------------------


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

// The same for a weight that is read once: not kept in L1.
template <bool VEC>
__device__ __forceinline__ float4 head_stream4(const float* p, int c, int D, int64_t sd) {
  if (!VEC) return head_load4<false>(p, c, D, sd);
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < D)
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(r.x), "=f"(r.y), "=f"(r.z), "=f"(r.w)
                 : "l"(p + c));
  return r;
}

// Up to 8 of the call's rows from r0 on.
template <int NR>
struct FewRows {
  int row[NR];           // a row with a target, or -1
  __device__ __forceinline__ void read(const HeadDev& d, int r0) {
#pragma unroll
    for (int i = 0; i < NR; ++i) row[i] = r0 + i < d.N && head_first_id(d, r0 + i) != kNoToken ? r0 + i : -1;
  }
};

// D += A B for A 16 x 8 (row major), B 8 x 8, in TF32: the upper 19 bits of each
// element are read.
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, hi its upper 11 significant bits; the tensor core reads the upper 11 of lo.
__device__ __forceinline__ void tf32_split(float x, uint32_t* hi, uint32_t* lo) {
  *hi = __float_as_uint(x) & 0xFFFFE000u;
  *lo = __float_as_uint(x - __uint_as_float(*hi));
}

struct HeadRowsDev {
  HeadDev d;
  int blocks;            // the width in blocks of 16, rounded up
  HeadPart* part;        // forward: [row][CTA]
  float* dx;             // backward: [row block][V][8 NT]
};

constexpr int kFewThreads = 512;
constexpr int kAhead = 6;    // blocks of 16 columns in flight per warp

// Up to 8 NT rows (blockIdx.y: which) against the whole vocabulary.  A warp takes 16
// vocabulary rows at a time; lane l reads columns 4 (l % 4) .. + 3 of each block of
// 16 from its rows l / 4 and l / 4 + 8, which are the elements that it supplies to
// two MMAs (the order of the columns inside a block does not matter as long as
// the hidden rows take the same).
template <int NT, bool GRAD>
__global__ void __launch_bounds__(kFewThreads, 1) head_rows_kernel(const __grid_constant__ HeadRowsDev a) {
  constexpr int W = kFewThreads / 32, NR = 8 * NT;
  extern __shared__ float s_h[];         // [NR][pitch]
  __shared__ int s_row[NR];
  __shared__ HeadPart s_part[W][NR];
  const HeadDev& d = a.d;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r0 = blockIdx.y * NR;
  const int lg = lane / 4, lt = lane % 4, pitch = a.blocks * 16 + 16;
  pdl_launch_dependents();
  // groups of 16 rows go around the CTAs before the warps, so that the SMs' shares differ by one at most
  const int hop = gridDim.x * W, groups = (d.V + 15) / 16;
  int gl = warp * gridDim.x + blockIdx.x, bl = 0;    // the loads' group and block
  auto fetch = [&](float4 (&x)[2]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int64_t v = (int64_t)gl * 16 + lg + 8 * j;
      x[j] = v < d.V ? head_load4<false>(d.w + v * d.wv, bl * 16 + lt * 4, d.D, d.wd) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if (++bl == a.blocks) {
      bl = 0;
      gl += hop;
    }
  };
  pdl_wait();
  float4 x[kAhead][2];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(x[i]);
  if (threadIdx.x < NR) {
    const int r = r0 + threadIdx.x;
    s_row[threadIdx.x] = r < d.N && head_first_id(d, r) != kNoToken ? r : -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < NR * a.blocks * 4; i += kFewThreads) {
    const int n = i / (a.blocks * 4), c = i % (a.blocks * 4) * 4;
    *reinterpret_cast<float4*>(&s_h[n * pitch + c]) =
        s_row[n] < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
        : d.vec_h    ? head_load4<true>(head_row<const float>(d, d.hid, s_row[n]), c, d.D, 1)
                     : head_load4<false>(head_row<const float>(d, d.hid, s_row[n]), c, d.D, d.hid.sd);
  }
  __syncthreads();
  // this lane's results: rows lg and lg + 8 of a group times call rows 2 lt, 2 lt + 1 of each eight
  constexpr int M = 2 * NT;
  int row[M], at[M], next[M];
  float lse2[M], gr[M];
  HeadPart pt[M];
#pragma unroll
  for (int i = 0; i < M; ++i) {
    row[i] = s_row[i / 2 * 8 + 2 * lt + i % 2];
    at[i] = 0;
    next[i] = row[i] < 0 ? kNoToken : head_first_id(d, row[i]);
    lse2[i] = gr[i] = 0.f;
    if (GRAD && row[i] >= 0) {
      lse2[i] = *head_row<const float>(d, d.lse, row[i]) * kHeadLog2e;
      gr[i] = *head_row<const float>(d, d.gl, row[i]) * d.temp;
    }
    pt[i] = HeadPart{-INFINITY, 0.f, 0.f, 0.f};
  }
  const float f = d.inv_temp * kHeadLog2e;
  float sum[NT][4], part[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = part[i][j] = 0.f;
  int g = warp * gridDim.x + blockIdx.x, b = 0;
  auto step = [&](float4 (&y)[2]) {
    uint32_t hi[2][4], lo[2][4];  // [columns 0 and 1, columns 2 and 3]
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      tf32_split(y[j].x, &hi[0][j], &lo[0][j]);
      tf32_split(y[j].y, &hi[0][2 + j], &lo[0][2 + j]);
      tf32_split(y[j].z, &hi[1][j], &lo[1][j]);
      tf32_split(y[j].w, &hi[1][2 + j], &lo[1][2 + j]);
    }
    fetch(y);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float4 h = *reinterpret_cast<const float4*>(&s_h[(i * 8 + lg) * pitch + b * 16 + lt * 4]);
      uint32_t hh[4], hl[4];
      tf32_split(h.x, &hh[0], &hl[0]);
      tf32_split(h.y, &hh[1], &hl[1]);
      tf32_split(h.z, &hh[2], &hl[2]);
      tf32_split(h.w, &hh[3], &hl[3]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mma_tf32(part[i], lo[k], hh[2 * k], hh[2 * k + 1]);
        mma_tf32(part[i], hi[k], hl[2 * k], hl[2 * k + 1]);
        mma_tf32(part[i], hi[k], hh[2 * k], hh[2 * k + 1]);
      }
    }
    // the tensor core cuts its sums: they go on in f32 every 256 columns
    if ((++b & 15) == 0 || b == a.blocks) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[i][j] += part[i][j];
          part[i][j] = 0.f;
        }
    }
    if (b < a.blocks) return;
    b = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int v = g * 16 + lg + 8 * j;
#pragma unroll
      for (int i = 0; i < M; ++i) {
        float& s = sum[i / 2][2 * j + i % 2];
        const float z = s * f;  // in units of log2
        s = 0.f;
        if (v >= d.V) continue;
        float t = 0.f;
        if (next[i] <= v) {
          if (d.distill) {
            const int* id = d.eid + (int64_t)row[i] * d.K;
            const float* w = d.ew + (int64_t)row[i] * d.K;
            while (next[i] <= v) {
              if (next[i] == v) t += w[at[i]];
              next[i] = ++at[i] < d.K ? id[at[i]] : kNoToken;
            }
          } else if (next[i] == v) {
            t = d.weight;
          }
        }
        if (GRAD) {
          a.dx[((int64_t)blockIdx.y * d.V + v) * NR + i / 2 * 8 + 2 * lt + i % 2] =
              row[i] < 0 ? 0.f : gr[i] * (head_ex2(z - lse2[i]) - t - d.share);
        } else {
          const float m = fmaxf(pt[i].m, z);
          pt[i].s = pt[i].s * head_ex2(pt[i].m - m) + head_ex2(z - m);
          if (m == -INFINITY) pt[i].s = 0.f;  // scores of -inf alone
          pt[i].m = m;
          if (t != 0.f) pt[i].dot = __fmaf_rn(t, z, pt[i].dot);
          pt[i].sum += z;
        }
      }
    }
    g += hop;
  };
  while (g < groups) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (g < groups) step(x[i]);
  }
  if (GRAD) return;
  // the CTA's part of a row: 8 lanes of each warp, then the warps
#pragma unroll
  for (int i = 0; i < M; ++i) {
    HeadPart y = pt[i];
#pragma unroll
    for (int o = 4; o < 32; o *= 2) {
      HeadPart z;
      z.m = __shfl_xor_sync(0xffffffffu, y.m, o);
      z.s = __shfl_xor_sync(0xffffffffu, y.s, o);
      z.dot = __shfl_xor_sync(0xffffffffu, y.dot, o);
      z.sum = __shfl_xor_sync(0xffffffffu, y.sum, o);
      y = lane & o ? head_add(z, y) : head_add(y, z);
    }
    if (lg == 0) s_part[warp][i / 2 * 8 + 2 * lt + i % 2] = y;
  }
  for (int k = W / 2; k > 0; k /= 2) {
    __syncthreads();
    const int w = threadIdx.x / NR, n = threadIdx.x % NR;
    HeadPart y;
    if (w < k) y = head_add(s_part[2 * w][n], s_part[2 * w + 1][n]);
    __syncthreads();
    if (w < k) s_part[w][n] = y;
  }
  __syncthreads();
  if (threadIdx.x < NR && r0 + threadIdx.x < d.N)
    a.part[(int64_t)(r0 + threadIdx.x) * gridDim.x + blockIdx.x] = s_part[0][threadIdx.x];
}

// ---- few rows, the weight through a ring of bulk copies --------------------------------

constexpr int kRingCols = 512;               // columns of a stage
constexpr int kRingPitch = kRingCols + 16;   // so that two rows' 64 bytes lie in different banks
constexpr int kRingStage = 16 * kRingPitch * 4;
constexpr int kRingWarps = 16;
constexpr int kRingThreads = kRingWarps * 32 + 32;
constexpr int kRingSmem = 224 * 1024;

enum RingMode { kRingScores, kRingScoreGrad, kRingGrad };

struct HeadRingDev {
  HeadDev d;
  int blocks;            // the width in blocks of 16, rounded up
  int chunks;            // stages of a group of 16 vocabulary rows
  int stages;
  HeadPart* part;        // kRingScores: [row][CTA]
  float* dx;             // kRingScoreGrad: [row block][V][8 NT]
  float* dh;             // kRingGrad: [CTA][8 NT][D]
  int* err;
};

__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, int* failed) {
  for (uint32_t i = 0; i < kWaitIters; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 63 && *(volatile int*)failed) return false;
  }
  atomicExch(failed, 1);
  return false;
}
__device__ __forceinline__ void ring_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// Up to 8 NT rows (blockIdx.y: which) against the whole vocabulary, 16 rows of it
// at a time per CTA: a warp copies row segments of 2 KB into the ring, 16 warps
// share a segment's columns, and their sums meet in shared memory.  kRingGrad: the
// group stays in the ring until its dw has been written and its part of dh been
// added, so that the weight is read once (widths up to 1024).
template <int NT, int MODE>
__global__ void __launch_bounds__(kRingThreads, 1) head_ring_kernel(const __grid_constant__ HeadRingDev a) {
  constexpr int NR = 8 * NT;
  extern __shared__ unsigned char smem_raw[];
  const HeadDev& d = a.d;
  float* ring = reinterpret_cast<float*>(smem_raw);                     // [stages][16][kRingPitch]
  float* s_h = ring + a.stages * (kRingStage / 4);                      // [NR][pitch]
  const int pitch = a.blocks * 16 + 16;
  float4* red = reinterpret_cast<float4*>(s_h + NR * pitch);            // [2][NT][warps][32]: every warp's results of a group
  float* s_dx = reinterpret_cast<float*>(red + 2 * NT * kRingWarps * 32);  // [16][NR]
  uint64_t* full = reinterpret_cast<uint64_t*>(s_dx + 16 * NR);
  uint64_t* empty = full + a.stages;
  __shared__ int s_row[NR], failed;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r0 = blockIdx.y * NR;
  const int groups = (d.V + 15) / 16;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kRingWarps);
    }
    failed = 0;
    fence_mbar_init();
  }
  // what no copy writes (columns behind the width, up to 16) meets zeros of the hidden rows: any number will do
  for (int i = threadIdx.x; i < a.stages * (kRingStage / 16); i += kRingThreads)
    reinterpret_cast<float4*>(ring)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  fence_proxy_async();
  __syncthreads();
  bool ok = true;
  pdl_wait();
  if (warp == kRingWarps) {  // copies
    int li = 0;
    for (int g = blockIdx.x; g < groups && ok; g += gridDim.x) {
      const int rows = min(16, d.V - g * 16);
      for (int c = 0; c < a.chunks; ++c, ++li) {
        const int s = li % a.stages;
        if (li >= a.stages && !(ok = __all_sync(0xffffffffu, ring_wait(&empty[s], (uint32_t)(li / a.stages - 1) & 1u, &failed)) != 0)) break;
        const uint32_t bytes = (uint32_t)min(kRingCols, d.D - c * kRingCols) * 4;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], bytes * rows);
        __syncwarp();
        if (lane < rows)
          bulk_g2s(ring + s * (kRingStage / 4) + lane * kRingPitch, d.w + ((int64_t)g * 16 + lane) * d.wv + c * kRingCols, bytes, &full[s]);
      }
    }
    if (!ok)  // what is under way lands before the CTA ends
      for (int s = 0; s < a.stages && s < li; ++s) mbar_wait(&full[s], (uint32_t)((li - 1 - s) / a.stages) & 1u);
  } else {
    if (threadIdx.x < NR) {
      const int r = r0 + threadIdx.x;
      s_row[threadIdx.x] = r < d.N && head_first_id(d, r) != kNoToken ? r : -1;
    }
    ring_sync();
    for (int i = threadIdx.x; i < NR * a.blocks * 4; i += kRingWarps * 32) {
      const int n = i / (a.blocks * 4), c = i % (a.blocks * 4) * 4;
      *reinterpret_cast<float4*>(&s_h[n * pitch + c]) =
          s_row[n] < 0 ? make_float4(0.f, 0.f, 0.f, 0.f)
          : d.vec_h    ? head_load4<true>(head_row<const float>(d, d.hid, s_row[n]), c, d.D, 1)
                       : head_load4<false>(head_row<const float>(d, d.hid, s_row[n]), c, d.D, d.hid.sd);
    }
    ring_sync();
    const int lg = lane / 4, lt = lane % 4;
    // the first 16 NR threads finish a group: vocabulary row fv, call row fn
    const int fn = threadIdx.x % NR, fv = threadIdx.x / NR;
    const bool fin = fv < 16;
    const int row = fin ? s_row[fn] : -1;
    Entries ent;
    ent.left = 0;
    ent.next = kNoToken;
    float lse2 = 0.f, gr = 0.f;
    if (row >= 0) {
      if (d.distill) ent.begin(d, row);
      else ent.next = head_id(d, d.ids, row, 0);
      if (MODE != kRingScores) {
        lse2 = *head_row<const float>(d, d.lse, row) * kHeadLog2e;
        gr = *head_row<const float>(d, d.gl, row) * d.temp;
      }
    }
    HeadPart pt = {-INFINITY, 0.f, 0.f, 0.f};
    const float f = d.inv_temp * kHeadLog2e;
    // kRingGrad: two columns per thread
    const int col = threadIdx.x * 2;
    const bool mine = MODE == kRingGrad && col < d.D;
    uint64_t hc[NR], acc[NR];
    if (MODE == kRingGrad) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        hc[n] = mine ? pk(s_h[n * pitch + col], s_h[n * pitch + col + 1]) : 0;
        acc[n] = 0;
      }
    }
    int li = 0, k = 0;
    for (int g = blockIdx.x; g < groups; g += gridDim.x, ++k) {
      float sum[NT][4];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] = 0.f;
      const int first = li;
      for (int c = 0; c < a.chunks; ++c, ++li) {
        const int s = li % a.stages;
        if (ok) ok = __all_sync(0xffffffffu, ring_wait(&full[s], (uint32_t)(li / a.stages) & 1u, &failed)) != 0;
        const float* w = ring + s * (kRingStage / 4);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int b = warp * 2 + q, at = c * (kRingCols / 16) + b;  // block of the stage, of the width
          if (at >= a.blocks) break;
          uint32_t hi[2][4], lo[2][4];  // [columns 0 and 1, columns 2 and 3]
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float4 y = *reinterpret_cast<const float4*>(&w[(lg + 8 * j) * kRingPitch + b * 16 + lt * 4]);
            tf32_split(y.x, &hi[0][j], &lo[0][j]);
            tf32_split(y.y, &hi[0][2 + j], &lo[0][2 + j]);
            tf32_split(y.z, &hi[1][j], &lo[1][j]);
            tf32_split(y.w, &hi[1][2 + j], &lo[1][2 + j]);
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const float4 h = *reinterpret_cast<const float4*>(&s_h[(i * 8 + lg) * pitch + at * 16 + lt * 4]);
            uint32_t hh[4], hl[4];
            tf32_split(h.x, &hh[0], &hl[0]);
            tf32_split(h.y, &hh[1], &hl[1]);
            tf32_split(h.z, &hh[2], &hl[2]);
            tf32_split(h.w, &hh[3], &hl[3]);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              mma_tf32(sum[i], lo[p], hh[2 * p], hh[2 * p + 1]);
              mma_tf32(sum[i], hi[p], hl[2 * p], hl[2 * p + 1]);
              mma_tf32(sum[i], hi[p], hh[2 * p], hh[2 * p + 1]);
            }
          }
        }
        if (MODE != kRingGrad) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&empty[s]);
        }
      }
      float4* buf = red + (k & 1) * NT * kRingWarps * 32;
#pragma unroll
      for (int i = 0; i < NT; ++i)
        buf[(i * kRingWarps + warp) * 32 + lane] = make_float4(sum[i][0], sum[i][1], sum[i][2], sum[i][3]);
      ring_sync();
      if (fin) {
        // the result of (fv, fn) lies with lane (fv % 8) * 4 + fn % 8 / 2, element fv / 8 * 2 + fn % 2
        const float* p = reinterpret_cast<const float*>(buf + fn / 8 * kRingWarps * 32 + (fv % 8) * 4 + fn % 8 / 2) + fv / 8 * 2 + fn % 2;
        float z = 0.f;
#pragma unroll
        for (int i = 0; i < kRingWarps; ++i) z += p[i * 128];
        z *= f;  // in units of log2
        const int v = g * 16 + fv;
        float x = 0.f;
        if (v < d.V && row >= 0) {
          float t = 0.f;
          if (ent.next <= v) {
            if (d.distill) {
              ent.skip_to(v);
              t = ent.take(v);
            } else if (ent.next == v) {
              t = d.weight;
            }
          }
          if (MODE != kRingScores) {
            x = gr * (head_ex2(z - lse2) - t - d.share);
          } else {
            const float m = fmaxf(pt.m, z);
            pt.s = pt.s * head_ex2(pt.m - m) + head_ex2(z - m);
            if (m == -INFINITY) pt.s = 0.f;  // scores of -inf alone
            pt.m = m;
            if (t != 0.f) pt.dot = __fmaf_rn(t, z, pt.dot);
            pt.sum += z;
          }
        }
        if (MODE == kRingScoreGrad && v < d.V) a.dx[((int64_t)blockIdx.y * d.V + v) * NR + fn] = x;
        if (MODE == kRingGrad) s_dx[fv * NR + fn] = x;
      }
      if (MODE != kRingGrad) continue;
      ring_sync();
      const int rows = min(16, d.V - g * 16);
      if (mine) {
        const float* w = ring + (first + col / kRingCols) % a.stages * (kRingStage / 4) + col % kRingCols;
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
          const float2 y = *reinterpret_cast<const float2*>(&w[r * kRingPitch]);
          const uint64_t w2 = pk(y.x, y.y);
          uint64_t o = 0;
#pragma unroll
          for (int n = 0; n < NR; n += 4) {
            const float4 x = *reinterpret_cast<const float4*>(&s_dx[r * NR + n]);
            const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint64_t xx = pk(xs[i], xs[i]);
              acc[n + i] = fma2(xx, w2, acc[n + i]);
              o = fma2(xx, hc[n + i], o);
            }
          }
          if (!d.dw) continue;
          float o0, o1;
          upk(o, &o0, &o1);
          float* to = d.dw + ((int64_t)g * 16 + r) * d.dwv;
          if (d.vec_dw) {
            __stcs(reinterpret_cast<float2*>(to + col), make_float2(o0, o1));
          } else {
            to[col * d.dwd] = o0;
            if (col + 1 < d.D) to[(col + 1) * d.dwd] = o1;
          }
        }
      }
      __syncwarp();
      if (lane == 0)
        for (int c = 0; c < a.chunks; ++c) mbar_arrive(&empty[(first + c) % a.stages]);
    }
    if (MODE == kRingScores) {
      // the CTA's part of a row: 16 threads, folded in the order of their vocabulary rows
      HeadPart* sp = reinterpret_cast<HeadPart*>(red);
      ring_sync();
      if (fin) sp[fv * NR + fn] = pt;
      for (int n = 8; n > 0; n /= 2) {
        ring_sync();
        HeadPart y;
        if (fv < n) y = head_add(sp[2 * fv * NR + fn], sp[(2 * fv + 1) * NR + fn]);
        ring_sync();
        if (fv < n) sp[fv * NR + fn] = y;
      }
      if (fv == 0 && r0 + fn < d.N) a.part[(int64_t)(r0 + fn) * gridDim.x + blockIdx.x] = sp[fn];
    }
    if (mine && d.dh.p) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float x0, x1;
        upk(acc[n], &x0, &x1);
        float* to = a.dh + ((int64_t)blockIdx.x * NR + n) * d.D + col;
        to[0] = x0;
        if (col + 1 < d.D) to[1] = x1;
      }
    }
  }
  if (lane == 0 && !ok) atomicOr(a.err, kAsyncWaitTimeout);
}

struct HeadGradDev {
  HeadDev d;
  int block;             // of NR rows
  int64_t db;            // dx of the block: first element, and the distance of its rows
  int ds;
  int lg;                // 2^lg threads (whole warps) along the width, the rest along the vocabulary
  const float* dx;
  float* part;           // [part of the vocabulary][NR][D] of dh
};

// A thread per 4 columns; blockIdx.y and the thread's group: a range of the
// vocabulary.
template <int NR>
__global__ void __launch_bounds__(256, 2) head_grad_kernel(const __grid_constant__ HeadGradDev a) {
  constexpr int U = 4;   // rows of the vocabulary in flight
  const HeadDev& d = a.d;
  pdl_launch_dependents();
  const int c = (blockIdx.x * 256 + (threadIdx.x & ((1 << a.lg) - 1))) * 4;
  const int groups = 256 >> a.lg, part = blockIdx.y * groups + (threadIdx.x >> a.lg), parts = gridDim.y * groups;
  const int r0 = a.block * NR;
  const bool add = a.block > 0;  // behind earlier rows
  pdl_wait();
  uint64_t h[NR][2], acc[NR][2];
  {
    FewRows<NR> rows;
    rows.read(d, r0);
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (rows.row[i] >= 0) x = head_load4<false>(head_row<const float>(d, d.hid, rows.row[i]), c, d.D, d.hid.sd);
      h[i][0] = pk(x.x, x.y), h[i][1] = pk(x.z, x.w);
      acc[i][0] = acc[i][1] = 0;
    }
  }
  const float* dx = a.dx + a.db;
  const int lane = threadIdx.x % 32;
  const int64_t v1 = (int64_t)d.V * (part + 1) / parts;
  int64_t v = (int64_t)d.V * part / parts;
  // U rows of the weight, and one of their score gradients per lane
  auto fetch = [&](float4 (&w)[U], float& x, int64_t at) {
    x = lane < U * NR && at + lane / NR < v1 ? dx[(at + lane / NR) * a.ds + lane % NR] : 0.f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      w[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (d.dh.p && at + j < v1)
        w[j] = d.vec_w ? head_stream4<true>(d.w + (at + j) * d.wv, c, d.D, 1) : head_load4<false>(d.w + (at + j) * d.wv, c, d.D, d.wd);
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
        float4 y = make_float4(o[0], o[1], o[2], o[3]);
        if (add) {
          const float4 b = *reinterpret_cast<const float4*>(to + c);
          y.x += b.x, y.y += b.y, y.z += b.z, y.w += b.w;
        }
        __stcs(reinterpret_cast<float4*>(to + c), y);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (c + k < d.D) {
            float* e = to + (c + k) * d.dwd;
            *e = add ? *e + o[k] : o[k];
          }
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

// dh of up to NR rows from its parts, in order: 32 columns times 8 runs of parts
// per CTA; zeros for rows without a target.
template <int NR>
__global__ void __launch_bounds__(256) head_grad_join_kernel(const __grid_constant__ HeadGradDev a, int parts) {
  __shared__ float s[8][32];
  const HeadDev& d = a.d;
  pdl_wait();
  const int c = blockIdx.x * 32 + threadIdx.x % 32, w = threadIdx.x / 32, r = blockIdx.y, row = a.block * NR + r;
  if (row >= d.N) return;
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
  head_row<float>(d, d.dh, row)[c * d.dh.sd] = head_first_id(d, row) != kNoToken ? sum : 0.f;
}

// ---- host side -------------------------------------------------------------------

template <int NT, bool GRAD>
Error launch_rows(HeadRowsDev& a, int ctas, cudaStream_t s) {
  auto k = head_rows_kernel<NT, GRAD>;
  const int smem = 8 * NT * (a.blocks + 1) * 64;
  allow_smem((const void*)k, smem);
  return launch_after(k, dim3((unsigned)ctas, (unsigned)((a.d.N + 8 * NT - 1) / (8 * NT))), kFewThreads, smem, s,
                      "head rows kernel", a);
}

int ring_fixed(int nt, int blocks) {  // shared memory besides the stages
  return 8 * nt * (blocks + 1) * 64 + 2 * nt * kRingWarps * 512 + 16 * 8 * nt * 4 + 16 * 16;
}
template <int NT, int MODE>
Error launch_ring(HeadRingDev& a, int ctas, cudaStream_t s) {
  auto k = head_ring_kernel<NT, MODE>;
  const int fixed = ring_fixed(NT, a.blocks);
  a.chunks = (a.d.D + kRingCols - 1) / kRingCols;
  a.stages = std::min(8, (kRingSmem - fixed) / kRingStage);
  const int smem = fixed + a.stages * kRingStage;
  allow_smem((const void*)k, smem);
  a.err = async_error_word();
  if (!a.err) return make_error(TRS_ERR_CUDA, "head: no async-error word");
  return launch_after(k, dim3((unsigned)ctas, (unsigned)((a.d.N + 8 * NT - 1) / (8 * NT))), kRingThreads, smem, s,
                      "head ring kernel", a);
}
template <int NT>
Error launch_ring(HeadRingDev& a, int mode, int ctas, cudaStream_t s) {
  return mode == kRingScores ? launch_ring<NT, kRingScores>(a, ctas, s)
         : mode == kRingGrad ? launch_ring<NT, kRingGrad>(a, ctas, s) : launch_ring<NT, kRingScoreGrad>(a, ctas, s);
}

template <int NR>
Error launch_grad(HeadGradDev& a, int splits, cudaStream_t s) {
  Error e = launch_after(head_grad_kernel<NR>, dim3((unsigned)((a.d.D + 1023) / 1024), (unsigned)splits), 256, 0, s,
                         "head gradient kernel", a);
  if (!e.ok() || !a.d.dh.p) return e;
  return launch_after(head_grad_join_kernel<NR>, dim3((unsigned)((a.d.D + 31) / 32), (unsigned)NR), 256, 0, s,
                      "head gradient join kernel", a, splits * (256 >> a.lg));
}

Error run_rows(const HeadDev& d, bool backward, cudaStream_t s) {
  const int sms = current_device_info().sm_count;
  const int width = (d.D + 15) / 16;
  // 16 rows share one read of the weight where the shared memory holds them
  const int nt = d.N > 8 && ring_fixed(2, width) + 2 * kRingStage <= kRingSmem ? 2 : 1, blocks = (d.N + 8 * nt - 1) / (8 * nt);
  const int ctas = std::max(1, std::min(sms, (d.V + 15) / 16));
  HeadRowsDev a;
  std::memset(static_cast<void*>(&a), 0, sizeof(a));
  a.d = d;
  a.blocks = width;
  HeadRingDev r;
  std::memset(static_cast<void*>(&r), 0, sizeof(r));
  r.d = d;
  r.blocks = width;
  Scratch mem;
  Error e;
  if (!backward) {
    e = mem.alloc(sizeof(HeadPart) * (size_t)d.N * ctas, s);
    if (!e.ok()) return e;
    a.part = r.part = mem.as<HeadPart>();
    if (d.vec_w) e = nt == 1 ? launch_ring<1>(r, kRingScores, ctas, s) : launch_ring<2>(r, kRingScores, ctas, s);
    else e = nt == 1 ? launch_rows<1, false>(a, ctas, s) : launch_rows<2, false>(a, ctas, s);
    if (e.ok()) e = head_join(d, r.part, ctas, 1, ctas, true, s);
    return e;
  }
  HeadGradDev g;
  std::memset(static_cast<void*>(&g), 0, sizeof(g));
  g.d = d;
  // both stages of a group and the next one's first in the ring
  if (d.vec_w && d.D <= 2 * kRingCols && blocks == 1 &&
      ring_fixed(nt, width) + (d.D <= kRingCols ? 2 : 3) * kRingStage <= kRingSmem) {
    e = mem.alloc(sizeof(float) * (size_t)ctas * 8 * nt * d.D, s);
    if (!e.ok()) return e;
    g.part = r.dh = mem.as<float>();
    e = nt == 1 ? launch_ring<1>(r, kRingGrad, ctas, s) : launch_ring<2>(r, kRingGrad, ctas, s);
    if (!e.ok() || !d.dh.p) return e;
    const dim3 grid((unsigned)((d.D + 31) / 32), (unsigned)d.N);
    return nt == 1 ? launch_after(head_grad_join_kernel<8>, grid, 256, 0, s, "head gradient join kernel", g, ctas)
                   : launch_after(head_grad_join_kernel<16>, grid, 256, 0, s, "head gradient join kernel", g, ctas);
  }
  const int chunks = (d.D + 3) / 4, colblocks = (d.D + 1023) / 1024;
  g.lg = 5;
  while (g.lg < 8 && (1 << g.lg) < chunks) ++g.lg;
  const int splits = std::max(1, std::min((d.V + 31) / 32, 2 * sms / colblocks));
  const size_t nd = (size_t)d.V * 8 * nt * blocks;
  e = mem.alloc(sizeof(float) * (nd + (size_t)splits * (256 >> g.lg) * 8 * d.D), s);
  if (!e.ok()) return e;
  a.dx = r.dx = mem.as<float>();
  if (d.vec_w) e = nt == 1 ? launch_ring<1>(r, kRingScoreGrad, ctas, s) : launch_ring<2>(r, kRingScoreGrad, ctas, s);
  else e = nt == 1 ? launch_rows<1, true>(a, ctas, s) : launch_rows<2, true>(a, ctas, s);
  g.dx = a.dx;
  g.ds = 8 * nt;
  g.part = a.dx + nd;
  const int nr = d.N <= 1 ? 1 : d.N <= 2 ? 2 : d.N <= 4 ? 4 : 8;
  for (g.block = 0; e.ok() && g.block * nr < d.N; ++g.block) {
    g.db = nt == 2 ? 8 * g.block : (int64_t)g.block * d.V * 8;
    e = nr == 1 ? launch_grad<1>(g, splits, s) : nr == 2 ? launch_grad<2>(g, splits, s)
        : nr == 4 ? launch_grad<4>(g, splits, s) : launch_grad<8>(g, splits, s);
  }
  return e;
}

struct HeadCall {
  const char* fn;
  bool distill, backward;
  const trs_view *hidden, *weight, *ids, *logits;
  double smoothing, temperature;
  trs_view *loss, *lse;              // lse: read by the backward
  const trs_view* grad_loss;
  trs_view *grad_hidden, *grad_weight;
};

Error run_head(const HeadCall& c, cudaStream_t stream) {
  const std::string fn = c.fn;
  if (!c.hidden || !c.weight || !c.ids || (c.distill && !c.logits) || (!c.backward && !c.loss) ||
      (c.backward && (!c.grad_loss || !c.lse || (!c.grad_hidden && !c.grad_weight))))
    return make_error(TRS_ERR_ARG, fn + ": null view");
  Error e = validate_view(c.hidden, "hidden");
  if (!e.ok()) return e;
  if (c.hidden->ndim < 2 || c.hidden->ndim > 3)
    return make_error(TRS_ERR_SHAPE, fn + ": hidden must be [tokens, width] or [batch, tokens, width]");
  const Tokens t = tokens_of(c.hidden, c.hidden->ndim - 1);
  e = validate_view(c.weight, "the weight");
  if (!e.ok()) return e;
  if (c.weight->ndim != 2 || c.weight->shape[1] != c.hidden->shape[t.lead])
    return make_error(TRS_ERR_SHAPE, fn + ": the weight must be [vocabulary, width]");
  e = check_tokens(fn, c.ids, t, c.distill ? 1 : 0, c.distill ? "the teacher's ids" : "targets");
  if (e.ok() && c.distill) e = check_tokens(fn, c.logits, t, 1, "the teacher's logits");
  if (e.ok() && c.loss) e = check_tokens(fn, c.loss, t, 0, "the loss");
  if (e.ok() && c.lse) e = check_tokens(fn, c.lse, t, 0, "lse");
  if (e.ok() && c.grad_loss) e = check_tokens(fn, c.grad_loss, t, 0, "the loss gradient");
  if (e.ok() && c.grad_hidden) e = check_tokens(fn, c.grad_hidden, t, 1, "the hidden gradient");
  if (e.ok() && c.grad_weight) e = validate_view(c.grad_weight, "the weight gradient");
  if (!e.ok()) return e;
  if (c.grad_hidden && c.grad_hidden->shape[t.lead] != c.hidden->shape[t.lead])
    return make_error(TRS_ERR_SHAPE, fn + ": the hidden gradient must have the shape of hidden");
  if (c.grad_weight && !same_shape(c.grad_weight, c.weight))
    return make_error(TRS_ERR_SHAPE, fn + ": the weight gradient must have the shape of the weight");
  for (const trs_view* v : {c.hidden, c.weight, c.logits, (const trs_view*)c.loss, (const trs_view*)c.lse, c.grad_loss,
                            (const trs_view*)c.grad_hidden, (const trs_view*)c.grad_weight})
    if (v && v->dtype != TRS_F32) return make_error(TRS_ERR_DTYPE, fn + ": everything but the ids must be f32");
  if (c.ids->dtype != TRS_I32 && c.ids->dtype != TRS_I64)
    return make_error(TRS_ERR_DTYPE, fn + ": ids must be i32 or i64");
  const int64_t V = c.weight->shape[0], D = c.weight->shape[1], N = t.n();
  int64_t K = 1;
  if (c.distill) {
    K = c.ids->shape[t.lead];
    if (c.logits->shape[t.lead] != K)
      return make_error(TRS_ERR_SHAPE, fn + ": the teacher's ids and logits must have one shape");
    if (K < 1 || K > kMaxEntries) return make_error(TRS_ERR_SHAPE, fn + ": a teacher gives 1 to 1024 logits");
  }
  if (V < 1 || D < 1) return make_error(TRS_ERR_SHAPE, fn + ": an empty weight");
  if (!(c.smoothing >= 0.0 && c.smoothing <= 1.0))
    return make_error(TRS_ERR_ARG, fn + ": the smoothing must lie in [0, 1]");
  // its square, its inverse and the products with them stay f32 numbers
  if (!(c.temperature >= 0x1p-40 && c.temperature <= 0x1p40))
    return make_error(TRS_ERR_ARG, fn + ": the temperature must lie in [2^-40, 2^40]");
  const int64_t lim = 1ll << 30;
  if (t.B >= lim || t.T >= lim || N >= lim || V >= lim || D >= lim)
    return make_error(TRS_ERR_SHAPE, fn + ": 2^30 or more tokens, or rows or columns of the weight");
  e = c.backward ? check_outputs(fn, {c.grad_hidden, c.grad_weight},
                                 {c.hidden, c.weight, c.ids, c.logits, c.lse, c.grad_loss})
                 : check_outputs(fn, {c.loss, c.lse}, {c.hidden, c.weight, c.ids, c.logits});
  if (!e.ok()) return e;

  HeadDev d;
  std::memset(static_cast<void*>(&d), 0, sizeof(d));
  d.N = (int)N;
  d.V = (int)V;
  d.D = (int)D;
  d.K = (int)K;
  d.f_T = make_fastdiv((uint32_t)std::max<int64_t>(t.T, 1));
  d.hid = rows_dev(c.hidden, t);
  d.w = static_cast<const float*>(c.weight->data) + c.weight->offset;
  d.wv = c.weight->strides[0];
  d.wd = c.weight->strides[1];
  d.ids = rows_dev(c.ids, t);
  d.ids64 = c.ids->dtype == TRS_I64;
  if (c.distill) d.z = rows_dev(c.logits, t);
  if (c.loss) d.loss = rows_dev(c.loss, t);
  if (c.lse) d.lse = rows_dev(c.lse, t);
  d.distill = c.distill;
  d.temp = (float)c.temperature;
  d.inv_temp = (float)(1.0 / c.temperature);
  d.share = (float)(c.smoothing / (double)V);
  d.weight = (float)(1.0 - c.smoothing);
  d.vec_w = rows_vectors(c.weight);
  if (c.backward) {
    d.gl = rows_dev(c.grad_loss, t);
    if (c.grad_hidden) d.dh = rows_dev(c.grad_hidden, t);
    if (c.grad_weight) {
      d.dw = static_cast<float*>(c.grad_weight->data) + c.grad_weight->offset;
      d.dwv = c.grad_weight->strides[0];
      d.dwd = c.grad_weight->strides[1];
      d.vec_dw = rows_vectors(c.grad_weight);
    }
  }
  d.vec_h = N > 0 && rows_vectors(c.hidden);
  if (N == 0 && !d.dw) return Error{};
  // Up to 16 rows the CUDA cores keep up with HBM, or nearly; without rows the
  // tensor-core path writes the zeros.
  const bool few = N > 0 && N <= 16 && D <= 4096;
  // the rows' targets
  Scratch mem;
  const size_t n = ((size_t)N + 3) / 4 * 4, nk = ((size_t)N * K + 3) / 4 * 4;
  if (!few || c.distill) {
    e = mem.alloc(4 * (n + 4 + 2 * nk + (c.distill ? n : 0)), stream);
    if (!e.ok()) return e;
    d.live = mem.as<int>();
    d.rows = d.live + 4;
    d.eid = d.rows + n;
    d.ew = reinterpret_cast<float*>(d.eid + nk);
    d.ent = d.ew + nk;
  }
  if (c.distill && N > 0) {
    const int smem = 8 * 2 * d.K * 4;
    allow_smem((const void*)head_teacher_kernel, smem);
    head_teacher_kernel<<<(unsigned)((N + 7) / 8), 256, smem, stream>>>(d);
    e = check_launch("head teacher kernel");
    if (!e.ok()) return e;
  }
  if (few) return run_rows(d, c.backward, stream);
  e = launch_after(head_list_kernel, dim3(1), 1024, 0, stream, "head list kernel", d);
  if (!e.ok()) return e;
  if (c.grad_hidden && N > 0) {
    e = launch_after(head_masked_kernel, dim3((unsigned)std::min<int64_t>((N + 7) / 8, 1024)), 256, 0, stream,
                     "head masked rows kernel", d);
    if (!e.ok()) return e;
  }
  return head_tc(d, c.backward, stream);
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
    return TRS_ERR_OOM;
  }
}

}  // namespace
}  // namespace trs

using namespace trs;

extern "C" {

trs_status trs_linear_cross_entropy(const trs_view* hidden, const trs_view* weight, const trs_view* targets,
                                    double smoothing, trs_view* loss, trs_view* lse, trs_stream stream) {
  return guarded([&] {
    return run_head(HeadCall{"linear_cross_entropy", false, false, hidden, weight, targets, nullptr, smoothing, 1.0, loss,
                             lse, nullptr, nullptr, nullptr},
                    static_cast<cudaStream_t>(stream));
  });
}

trs_status trs_linear_cross_entropy_backward(const trs_view* grad_loss, const trs_view* hidden, const trs_view* weight,
                                             const trs_view* targets, const trs_view* lse, double smoothing,
                                             trs_view* grad_hidden, trs_view* grad_weight, trs_stream stream) {
  return guarded([&] {
    return run_head(HeadCall{"linear_cross_entropy_backward", false, true, hidden, weight, targets, nullptr, smoothing, 1.0,
                             nullptr, const_cast<trs_view*>(lse), grad_loss, grad_hidden, grad_weight},
                    static_cast<cudaStream_t>(stream));
  });
}

trs_status trs_linear_distillation(const trs_view* hidden, const trs_view* weight, const trs_view* teacher_ids,
                                   const trs_view* teacher_logits, double temperature, trs_view* loss, trs_view* lse,
                                   trs_stream stream) {
  return guarded([&] {
    return run_head(HeadCall{"linear_distillation", true, false, hidden, weight, teacher_ids, teacher_logits, 0.0,
                             temperature, loss, lse, nullptr, nullptr, nullptr},
                    static_cast<cudaStream_t>(stream));
  });
}

trs_status trs_linear_distillation_backward(const trs_view* grad_loss, const trs_view* hidden, const trs_view* weight,
                                            const trs_view* teacher_ids, const trs_view* teacher_logits,
                                            const trs_view* lse, double temperature, trs_view* grad_hidden,
                                            trs_view* grad_weight, trs_stream stream) {
  return guarded([&] {
    return run_head(HeadCall{"linear_distillation_backward", true, true, hidden, weight, teacher_ids, teacher_logits, 0.0,
                             temperature, nullptr, const_cast<trs_view*>(lse), grad_loss, grad_hidden, grad_weight},
                    static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
