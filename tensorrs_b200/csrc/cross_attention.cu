// cross_attention.cu -- trs_cross_attention and its gradient: the checks, the
// choice of kernel, and the kernels that run on the CUDA cores.
//
//   S = scale q k^T,  P = exp(S - lse),  lse = ln sum exp S,  out = P v
//   backward: delta = sum_d dout out,  dP = dout v^T,  dS = P (dP - delta),
//             dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
//
// with keys at and beyond key_lengths[b] absent (never read); a query without
// keys gives 0, lse = -inf and no gradient.
//
// cross_rows_kernel serves few query rows per key head (single tokens), where
// reading k and v once is all there is to do, and, in blocks of rows, head
// sizes above 128.  A CTA owns (problem, block of NR rows, part of the keys):
// groups of L lanes own one key at a time, each lane 4 (8) elements of the
// head; 4 keys are in flight per group, the dot products fold over the group
// with shuffles, and the running maximum, sum and output stay in registers
// until the CTA's groups are joined in shared memory.  Parts of the keys are
// joined by cross_join_kernel in a fixed order.  One row is bound by the loads
// in flight (8 x 16 heads of 64, 1024 to 2048 keys, 88 MB: 20 us, 4.3 TB/s),
// eight by arithmetic (4 x 16 heads, 2048 keys, 67 MB: 27 us).  Of heads of 256, 256
// queries on 1024 keys, 4 x 8 heads: 500 us (the plain form, products in a library,
// 360): four rows a CTA read k and v 64 times.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "../../include/trs.h"
#include "cross.h"
#include "cross_exact.cuh"

namespace trs {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kRowsMaxHead = 256;

struct RowsDev {
  CrossDev c;
  int blocks;        // blocks of NR rows per problem
  int splits;        // parts of the keys
  int items;         // problems * blocks * splits
  int ld;            // elements per partial row: the head size, rounded up to 4
  float* part;       // [split][problem][M][ld] and then m, l [split][problem][M], when splits > 1
  float* part_m;
  float* part_l;
};

// Four elements of a head as two pairs for the packed f32 operations.
struct Quad {
  uint64_t a, b;
};
template <bool VEC>
__device__ __forceinline__ Quad load4(const float* p, int d, int D, int64_t sd) {
  Quad q;
  if (VEC) {
    const ulonglong2 x = d < D ? *reinterpret_cast<const ulonglong2*>(p + d) : make_ulonglong2(0, 0);
    q.a = x.x;
    q.b = x.y;
  } else {
    q.a = pack2(d < D ? p[d * sd] : 0.f, d + 1 < D ? p[(d + 1) * sd] : 0.f);
    q.b = pack2(d + 2 < D ? p[(d + 2) * sd] : 0.f, d + 3 < D ? p[(d + 3) * sd] : 0.f);
  }
  return q;
}

// N sums over the L lanes of a group: each step a lane hands over the half that
// its partner keeps, so that N dot products take about N + log2 L shuffles
// instead of N log2 L.  Sum i ends in s[i % OWN] of lanes i DUP / OWN .. (OWN =
// N / L where N > L, DUP = L / N where N < L, else 1).
template <int L, int N>
__device__ __forceinline__ void fold_lanes(float (&s)[N], int lane, unsigned mask) {
#pragma unroll
  for (int o = L / 2, w = N / 2; o > 0; o >>= 1, w >>= 1) {
    if (w > 0) {
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < (w > 0 ? w : 1); ++i) {
        const float give = up ? s[i] : s[i + w], keep = up ? s[i + w] : s[i];
        s[i] = keep + __shfl_xor_sync(mask, give, o);
      }
    } else {
      s[0] += __shfl_xor_sync(mask, s[0], o);
    }
  }
}

__device__ __forceinline__ float dot4(const Quad& x, const Quad& y) {
  float lo, hi;
  unpack2(fma2(x.b, y.b, mul2(x.a, y.a)), &lo, &hi);
  return lo + hi;
}

// Two to four CTAs per SM where the rows leave the registers for it: the bytes
// in flight per SM carry this kernel.
template <int NR, int L, int NV, bool VEC>
__global__ void __launch_bounds__(kRowsThreads, NR * NV <= 2 ? 4 : NR * NV <= 4 ? 2 : 1) cross_rows_kernel(const RowsDev d) {
  const CrossDev& c = d.c;
  pdl_launch_dependents();
  constexpr int U = 4;                                  // keys in flight per group
  constexpr int NG = kRowsThreads / L;                  // groups
  constexpr int DP = L * 4 * NV;                        // padded head size
  constexpr int N = NR * U;                             // dot products of a step
  constexpr int OWN = N > L ? N / L : 1;                // of which a lane keeps OWN, from `mine` on
  constexpr int DUP = N < L ? L / N : 1;                // lanes that keep the same one
  constexpr int LPR = L / NR;                           // lanes that keep a row's
  __shared__ float s_m[NG][NR], s_l[NG][NR];
  extern __shared__ float s_acc[];                      // [NG][NR][DP]
  const int gid = threadIdx.x / L, lane = threadIdx.x % L;
  const int mine = lane * OWN / DUP % U;                // this lane's first key of the four
  const unsigned mask = (L == 32 ? 0xffffffffu : (1u << (L & 31)) - 1u) << (threadIdx.x % 32 / L * L);
  for (int item = blockIdx.x; item < d.items; item += gridDim.x) {
    const int sp = item % d.splits, rb = item / d.splits % d.blocks, pr = item / d.splits / d.blocks;
    const int b = pr / c.Hk, hk = pr % c.Hk;
    const int n = key_count(c.len, c.len64, c.len_s, c.Tk, b);
    const int per = (n + d.splits - 1) / d.splits;
    const int k0 = min(n, sp * per), k1 = min(n, k0 + per);
    Quad q[NR][NV], acc[NR][NV];                        // q times the scale and log2 e: a dot product is a score
    float m = -INFINITY, l = 0.f;                       // of this lane's row; l of this lane's keys
    const float f = c.scale * kLog2e;
    const uint64_t f2 = pack2(f, f);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const int row = rb * NR + r;
      const int g = row < c.M ? (int)fdiv((uint32_t)row, c.f_Tq) : 0, t = row < c.M ? row - g * c.Tq : 0;
      const float* qp = static_cast<const float*>(c.q.p) + b * c.q.sb + t * c.q.st + (hk * c.G + g) * c.q.sh;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        acc[r][i] = Quad{0, 0};
        q[r][i] = row < c.M ? load4<VEC>(qp, (lane + i * L) * 4, c.D, c.q.sd) : Quad{0, 0};
        q[r][i] = Quad{mul2(q[r][i].a, f2), mul2(q[r][i].b, f2)};
      }
    }
    const float* kp = static_cast<const float*>(c.k.p) + b * c.k.sb + hk * c.k.sh;
    const float* vp = static_cast<const float*>(c.v.p) + b * c.v.sb + hk * c.v.sh;
    for (int key = k0 + gid * U; key < k1; key += NG * U) {
      Quad kk[U][NV], vv[U][NV];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = key + u;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const bool on = at < k1;
          kk[u][i] = on ? load4<VEC>(kp + at * c.k.st, (lane + i * L) * 4, c.D, c.k.sd) : Quad{0, 0};
          vv[u][i] = on ? load4<VEC>(vp + at * c.v.st, (lane + i * L) * 4, c.D, c.v.sd) : Quad{0, 0};
        }
      }
      float s[N];
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          uint64_t x = 0;
#pragma unroll
          for (int i = 0; i < NV; ++i) x = fma2(q[r][i].b, kk[u][i].b, fma2(q[r][i].a, kk[u][i].a, x));
          float lo, hi;
          unpack2(x, &lo, &hi);
          s[r * U + u] = lo + hi;
        }
      fold_lanes<L, N>(s, lane, mask);
      float mx = m;
#pragma unroll
      for (int e = 0; e < OWN; ++e) {
        s[e] = key + mine + e < k1 ? s[e] : -INFINITY;
        mx = fmaxf(mx, s[e]);
      }
#pragma unroll
      for (int o = LPR / 2; o >= DUP; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(mask, mx, o));
      const float base = mx == -INFINITY ? 0.f : mx;  // all scores -inf so far: every weight stays 0
      const float alpha = ex2(m - base);
      m = mx;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < OWN; ++e) {
        s[e] = ex2(s[e] - base);
        l += s[e];
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float al = NR == 1 ? alpha : __shfl_sync(mask, alpha, r * LPR, L);
        const uint64_t al2 = pack2(al, al);
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[r][i] = Quad{mul2(acc[r][i].a, al2), mul2(acc[r][i].b, al2)};
#pragma unroll
        for (int u = 0; u < U; ++u) {
          constexpr int X = U;  // (r, u) is kept by lane (r U + u) DUP / OWN
          const float p = __shfl_sync(mask, s[(r * X + u) % OWN], (r * X + u) * DUP / OWN, L);
          const uint64_t p2 = pack2(p, p);
#pragma unroll
          for (int i = 0; i < NV; ++i)
            acc[r][i] = Quad{fma2(p2, vv[u][i].a, acc[r][i].a), fma2(p2, vv[u][i].b, acc[r][i].b)};
        }
      }
    }
    // a row's sum over the lanes that keep its keys
#pragma unroll
    for (int o = LPR / 2; o >= DUP; o >>= 1) l += __shfl_xor_sync(mask, l, o);
    // join the CTA's groups
    __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (lane == r * LPR) {
        s_m[gid][r] = m;
        s_l[gid][r] = l;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
        *reinterpret_cast<ulonglong2*>(&s_acc[(gid * NR + r) * DP + (lane + i * L) * 4]) =
            make_ulonglong2(acc[r][i].a, acc[r][i].b);
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < NR * DP; idx += kRowsThreads) {
      const int r = idx / DP, dd = idx % DP, row = rb * NR + r;
      if (row >= c.M || dd >= c.D) continue;
      float mx = -INFINITY;
      for (int g = 0; g < NG; ++g) mx = fmaxf(mx, s_m[g][r]);
      const float base = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, o = 0.f;
      for (int g = 0; g < NG; ++g) {
        const float w = ex2(s_m[g][r] - base);
        sum = __fmaf_rn(w, s_l[g][r], sum);
        o = __fmaf_rn(w, s_acc[(g * NR + r) * DP + dd], o);
      }
      if (d.splits > 1) {
        const int64_t at = ((int64_t)sp * (c.B * c.Hk) + pr) * c.M + row;
        d.part[at * d.ld + dd] = o;
        if (dd == 0) {
          d.part_m[at] = mx;
          d.part_l[at] = sum;
        }
      } else {
        const int gq = (int)fdiv((uint32_t)row, c.f_Tq), t = row - gq * c.Tq, h = hk * c.G + gq;
        float* op = static_cast<float*>(c.out.p) + b * c.out.sb + t * c.out.st + h * c.out.sh;
        op[dd * c.out.sd] = sum == 0.f ? 0.f : o / sum;
        if (dd == 0 && c.lse) c.lse[b * c.ls_b + h * c.ls_h + t * c.ls_t] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
      }
    }
    __syncthreads();
  }
}

// The parts of the keys joined in order: one warp per (problem, row), 4
// elements per lane and step, 8 parts' loads in flight.
struct JoinDev {
  CrossDev c;
  int splits, rows;          // rows per problem in the partials
  int ld;                    // elements per partial row, a multiple of 4
  const float *part, *part_m, *part_l;
};
__global__ void __launch_bounds__(128) cross_join_kernel(const JoinDev d) {
  pdl_wait();
  const CrossDev& c = d.c;
  if (c.nonfinite && *(volatile const int*)c.nonfinite != 0) return;  // the result is there already
  const int64_t w = (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const int np = c.B * c.Hk;
  if (w >= (int64_t)np * c.M) return;
  const int pr = (int)(w / c.M), row = (int)(w % c.M);
  const int64_t step = (int64_t)np * d.rows, first = (int64_t)pr * d.rows + row;
  float mx = -INFINITY;
  for (int s = lane; s < d.splits; s += 32) mx = fmaxf(mx, d.part_m[s * step + first]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float base = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  for (int s = lane; s < d.splits; s += 32) sum = __fmaf_rn(ex2(d.part_m[s * step + first] - base), d.part_l[s * step + first], sum);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int b = pr / c.Hk, hk = pr % c.Hk;
  const int g = (int)fdiv((uint32_t)row, c.f_Tq), t = row - g * c.Tq, h = hk * c.G + g;
  float* op = static_cast<float*>(c.out.p) + b * c.out.sb + t * c.out.st + h * c.out.sh;
  for (int e = lane * 4; e < c.D; e += 128) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < d.splits; s0 += 8) {
      float4 x[8];
      float wt[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool on = s0 + k < d.splits;
        const int64_t at = (s0 + k) * step + first;
        x[k] = on ? *reinterpret_cast<const float4*>(d.part + at * d.ld + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        wt[k] = on ? ex2(d.part_m[at] - base) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        acc.x = __fmaf_rn(wt[k], x[k].x, acc.x);
        acc.y = __fmaf_rn(wt[k], x[k].y, acc.y);
        acc.z = __fmaf_rn(wt[k], x[k].z, acc.z);
        acc.w = __fmaf_rn(wt[k], x[k].w, acc.w);
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    op[e * c.out.sd] = acc.x * inv;
    if (e + 1 < c.D) op[(e + 1) * c.out.sd] = acc.y * inv;
    if (e + 2 < c.D) op[(e + 2) * c.out.sd] = acc.z * inv;
    if (e + 3 < c.D) op[(e + 3) * c.out.sd] = acc.w * inv;
  }
  if (lane == 0 && c.lse) c.lse[b * c.ls_b + h * c.ls_h + t * c.ls_t] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

}  // namespace

Error cross_join(const CrossDev& c, int splits, int rows, int ld, const float* part, const float* part_m,
                 const float* part_l, cudaStream_t stream) {
  JoinDev j;
  j.c = c;
  j.splits = splits;
  j.rows = rows;
  j.ld = ld;
  j.part = part;
  j.part_m = part_m;
  j.part_l = part_l;
  const int64_t warps = (int64_t)c.B * c.Hk * c.M;
  return launch_after(cross_join_kernel, dim3((unsigned)((warps + 3) / 4)), 128, 0, stream, "cross attention join kernel", j);
}

namespace {

// The gradient of up to 8 query rows per key head (head sizes up to 128): k and
// v are read once and dk and dv written once, which bounds it.  Groups of lanes
// own keys as in cross_rows_kernel; a step takes the scores and dP of NR rows
// and U keys, folds both, and adds each pair's dS and P to dq (in registers to
// the end of the CTA's keys) and to the key's dk and dv.  The scale is applied in
// two halves, before and after, so that neither q k nor scale dS has to be an f32
// for the results to be (all of it on the elements of k: 92 -> 94 us for 8 rows
// on 2048 keys, 4 x 16 heads of 64, forward and gradient).
struct RowsGradDev {
  CrossDev c;
  int splits;
  int ld;            // elements per partial row of dq
  float s1, s2;      // the scale, s1 a power of two near its root: S = s1 (s2 q) k, dk = (s1 dS) (s2 q), dq = s2 (s1 dS) k
  float* part;       // [split][problem][M][ld] when splits > 1
};
template <int NR, int L, bool VEC>
__global__ void __launch_bounds__(kRowsThreads, NR <= 4 ? 2 : 1) cross_rows_grad_kernel(const RowsGradDev d) {
  const CrossDev& c = d.c;
  pdl_launch_dependents();
  constexpr int U = NR == 8 ? 2 : 4, NG = kRowsThreads / L, DP = L * 4, N = NR * U;
  constexpr int OWN = N > L ? N / L : 1, DUP = N < L ? L / N : 1, LPR = L / NR;
  extern __shared__ float s_acc[];  // [NG][NR][DP]
  const int gid = threadIdx.x / L, lane = threadIdx.x % L, dd = lane * 4;
  const int mine = lane * OWN / DUP % U, my_row = lane / LPR;
  const unsigned mask = (L == 32 ? 0xffffffffu : (1u << (L & 31)) - 1u) << (threadIdx.x % 32 / L * L);
  const int sp = blockIdx.x % d.splits, pr = blockIdx.x / d.splits, b = pr / c.Hk, hk = pr % c.Hk;
  const int n = key_count(c.len, c.len64, c.len_s, c.Tk, b);
  const int per = (n + d.splits - 1) / d.splits, k0 = min(n, sp * per), k1 = min(n, k0 + per);
  Quad q[NR], go[NR], acc[NR];         // q holds s2 q
  float lse2 = INFINITY, delta = 0.f;  // of this lane's row
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    acc[r] = q[r] = go[r] = Quad{0, 0};
    if (r >= c.M) continue;
    const int g = (int)fdiv((uint32_t)r, c.f_Tq), t = r - g * c.Tq, h = hk * c.G + g;
    auto at = [&](const HeadsDev& x) { return static_cast<const float*>(x.p) + b * x.sb + t * x.st + h * x.sh; };
    q[r] = load4<VEC>(at(c.q), dd, c.D, c.q.sd);
    q[r] = Quad{mul2(q[r].a, pack2(d.s2, d.s2)), mul2(q[r].b, pack2(d.s2, d.s2))};
    go[r] = load4<VEC>(at(c.dout), dd, c.D, c.dout.sd);
    float dl = dot4(go[r], load4<VEC>(at(c.out), dd, c.D, c.out.sd));
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) dl += __shfl_xor_sync(mask, dl, o);
    if (my_row == r) {
      delta = dl;
      const float ls = c.lse[b * c.ls_b + h * c.ls_h + t * c.ls_t];
      lse2 = ls == -INFINITY ? INFINITY : ls * kLog2e;  // scores of -inf alone: no weight
    }
  }
  const float s1 = d.s1, f = s1 * kLog2e;
  // no weight behind the last key, and none for a row that only fills up the block
  // (its score with an infinite key is 0 * inf)
  const int end = my_row < c.M ? k1 - mine : -1;
  auto key_row = [&](const HeadsDev& x, int64_t t) { return static_cast<const float*>(x.p) + b * x.sb + t * x.st + hk * x.sh; };
  auto store = [&](const HeadsDev& x, int64_t t, const Quad& v) {
    float* p = const_cast<float*>(key_row(x, t));
    if (VEC) {
      if (dd < c.D) *reinterpret_cast<ulonglong2*>(p + dd) = make_ulonglong2(v.a, v.b);
    } else {
      float e[4];
      unpack2(v.a, &e[0], &e[1]);
      unpack2(v.b, &e[2], &e[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (dd + i < c.D) p[(dd + i) * x.sd] = e[i];
    }
  };
  for (int key = k0 + gid * U; key < k1; key += NG * U) {
    Quad kk[U], vv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = key + u < k1;
      kk[u] = on ? load4<VEC>(key_row(c.k, key + u), dd, c.D, c.k.sd) : Quad{0, 0};
      vv[u] = on ? load4<VEC>(key_row(c.v, key + u), dd, c.D, c.v.sd) : Quad{0, 0};
    }
    float s[N], dp[N];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[r * U + u] = dot4(q[r], kk[u]);
        dp[r * U + u] = dot4(go[r], vv[u]);
      }
    fold_lanes<L, N>(s, lane, mask);
    fold_lanes<L, N>(dp, lane, mask);
#pragma unroll
    for (int e = 0; e < OWN; ++e) {
      const bool on = key + e < end;
      s[e] = on ? ex2(min_nan(__fmaf_rn(s[e], f, -lse2), 0.f)) : 0.f;  // at most 1: large scores are off from lse
      dp[e] = on ? s[e] * ((dp[e] - delta) * s1) : 0.f;
    }
    Quad dk[U], dv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) dk[u] = dv[u] = Quad{0, 0};
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int from = (r * U + u) * DUP / OWN;
        const float p = __shfl_sync(mask, s[(r * U + u) % OWN], from, L);
        const float ds = __shfl_sync(mask, dp[(r * U + u) % OWN], from, L);
        const uint64_t p2 = pack2(p, p), ds2 = pack2(ds, ds);
        acc[r] = Quad{fma2(ds2, kk[u].a, acc[r].a), fma2(ds2, kk[u].b, acc[r].b)};
        dk[u] = Quad{fma2(ds2, q[r].a, dk[u].a), fma2(ds2, q[r].b, dk[u].b)};
        dv[u] = Quad{fma2(p2, go[r].a, dv[u].a), fma2(p2, go[r].b, dv[u].b)};
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (key + u >= k1) break;
      store(c.dk, key + u, dk[u]);
      store(c.dv, key + u, dv[u]);
    }
  }
  // rows at and behind the key length
  const int tail = c.Tk - n, z1 = n + (int)((int64_t)tail * (sp + 1) / d.splits);
  for (int key = n + (int)((int64_t)tail * sp / d.splits) + gid; key < z1; key += NG) {
    store(c.dk, key, Quad{0, 0});
    store(c.dv, key, Quad{0, 0});
  }
#pragma unroll
  for (int r = 0; r < NR; ++r)
    *reinterpret_cast<ulonglong2*>(&s_acc[(gid * NR + r) * DP + dd]) = make_ulonglong2(acc[r].a, acc[r].b);
  __syncthreads();
  for (int idx = threadIdx.x; idx < NR * DP; idx += kRowsThreads) {
    const int r = idx / DP, e = idx % DP;
    if (r >= c.M || e >= c.D) continue;
    float sum = 0.f;
    for (int g = 0; g < NG; ++g) sum += s_acc[(g * NR + r) * DP + e];
    sum *= d.s2;
    if (d.splits > 1) {
      d.part[(((int64_t)sp * (c.B * c.Hk) + pr) * c.M + r) * d.ld + e] = sum;
    } else {
      const int g = (int)fdiv((uint32_t)r, c.f_Tq), t = r - g * c.Tq, h = hk * c.G + g;
      static_cast<float*>(c.dq.p)[b * c.dq.sb + t * c.dq.st + h * c.dq.sh + e * c.dq.sd] = sum;
    }
  }
}

// dq from the parts, in order: a thread per element.
__global__ void __launch_bounds__(256) cross_rows_sum_kernel(const RowsGradDev d) {
  pdl_wait();
  const CrossDev& c = d.c;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, np = (int64_t)c.B * c.Hk;
  const int e = (int)(i % d.ld);
  const int64_t w = i / d.ld;
  if (w >= np * c.M || e >= c.D) return;
  const int r = (int)(w % c.M), pr = (int)(w / c.M);
  float sum = 0.f;
  for (int s0 = 0; s0 < d.splits; s0 += 8) {
    float x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = s0 + k < d.splits ? d.part[((s0 + k) * np * c.M + w) * d.ld + e] : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += x[k];
  }
  const int b = pr / c.Hk, g = (int)fdiv((uint32_t)r, c.f_Tq), t = r - g * c.Tq, h = pr % c.Hk * c.G + g;
  static_cast<float*>(c.dq.p)[b * c.dq.sb + t * c.dq.st + h * c.dq.sh + e * c.dq.sd] = sum;
}

// The gradient of head sizes above 128 on the CUDA cores, a warp per row: right,
// and slow.  Every pair is walked twice with three dot products folded over the
// warp, one pair at a time: 256 queries on 1024 keys, 4 x 8 heads of 256, take 11.4
// ms, where the plain form takes 0.6.
__global__ void __launch_bounds__(256) cross_grad_rows_kernel(const CrossDev c) {
  const int64_t warps = (int64_t)gridDim.x * 8, w = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  exact_dq_rows(c, w, warps);
  exact_dkv_rows(c, w, warps);
}

// Gradients of no queries or no keys at all.
__global__ void __launch_bounds__(256) cross_zero_kernel(HeadsDev x, int64_t B, int T, int H, int D) {
  const int64_t n = B * T * H * D;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t dd = i % D, h = i / D % H, t = i / D / H % T, b = i / D / H / T;
    static_cast<float*>(x.p)[b * x.sb + t * x.st + h * x.sh + dd * x.sd] = 0.f;
  }
}
__global__ void __launch_bounds__(256) cross_lse_kernel(const CrossDev c) {
  const int64_t n = (int64_t)c.B * c.Hq * c.Tq;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    c.lse[i / c.Tq / c.Hq * c.ls_b + i / c.Tq % c.Hq * c.ls_h + i % c.Tq * c.ls_t] = -INFINITY;
}

Error zero_heads(const HeadsDev& x, int64_t B, int T, int H, int D, cudaStream_t s) {
  const int64_t n = B * T * H * D;
  if (n == 0) return Error{};
  const int64_t g = (n + 255) / 256;
  cross_zero_kernel<<<(unsigned)(g < 4096 ? g : 4096), 256, 0, s>>>(x, B, T, H, D);
  return check_launch("cross attention zero kernel");
}

// ---- host side -------------------------------------------------------------------

// The parts of the keys that leave the fewest CTA places idle in the last wave,
// up to four waves and of 256 keys at least (8 x 16 heads of 64 on 1024 to 2048
// keys, parts of 64, 256 and 1024 at least: 22.6, 20.5 and 24.6 us; one sequence
// of 4 heads on 2048 keys 12.3, 12.3 and 26.6); `base` CTAs without parts.
int64_t key_parts(const void* kernel, int smem, int64_t base, int Tk) {
  const int64_t resident = (int64_t)current_device_info().sm_count * resident_blocks_smem(kernel, kRowsThreads, smem);
  int64_t splits = 1;
  double best = 0.0;
  for (int64_t n = 1; n <= std::max(1, Tk / 256) && (n == 1 || n * base <= 4 * resident); ++n) {
    const int64_t waves = (n * base + resident - 1) / resident;
    const double use = (double)(n * base) / (double)(waves * resident);
    if (use > best + 0.02) {
      best = use;
      splits = n;
    }
  }
  return splits;
}

template <int NR, int L, int NV>
Error launch_rows(RowsDev& d, cudaStream_t s) {
  const CrossDev& c = d.c;
  constexpr int smem = kRowsThreads / L * NR * L * 4 * NV * 4;
  auto k = c.vec ? cross_rows_kernel<NR, L, NV, true> : cross_rows_kernel<NR, L, NV, false>;
  allow_smem((const void*)k, smem);
  const int np = c.B * c.Hk;
  d.blocks = (c.M + NR - 1) / NR;
  const int64_t base = (int64_t)np * d.blocks;
  const int64_t splits = key_parts((const void*)k, smem, base, c.Tk);
  const int64_t items = base * splits;
  if (items >= (1ll << 31)) return make_error(TRS_ERR_SHAPE, "cross_attention: too many query rows");
  d.splits = (int)splits;
  d.items = (int)items;
  Scratch part;
  if (splits > 1) {
    const size_t rows = (size_t)splits * np * c.M;
    d.ld = (c.D + 3) / 4 * 4;
    Error e = part.alloc(sizeof(float) * rows * (d.ld + 2), s);
    if (!e.ok()) return e;
    d.part = part.as<float>();
    d.part_m = d.part + rows * d.ld;
    d.part_l = d.part_m + rows;
  }
  k<<<(unsigned)std::min<int64_t>(items, 1 << 24), kRowsThreads, smem, s>>>(d);
  Error e = check_launch("cross attention rows kernel");
  if (!e.ok() || splits == 1) return e;
  return cross_join(c, d.splits, c.M, d.ld, d.part, d.part_m, d.part_l, s);
}

Error run_rows(const CrossDev& c, cudaStream_t s) {
  RowsDev d;
  std::memset(static_cast<void*>(&d), 0, sizeof(d));
  d.c = c;
  if (c.D <= 32) {
    return c.M == 1 ? launch_rows<1, 8, 1>(d, s) : c.M == 2 ? launch_rows<2, 8, 1>(d, s)
           : c.M <= 4 ? launch_rows<4, 8, 1>(d, s) : launch_rows<8, 8, 1>(d, s);
  }
  if (c.D <= 64) {
    return c.M == 1 ? launch_rows<1, 16, 1>(d, s) : c.M == 2 ? launch_rows<2, 16, 1>(d, s)
           : c.M <= 4 ? launch_rows<4, 16, 1>(d, s) : launch_rows<8, 16, 1>(d, s);
  }
  if (c.D <= 128) {
    return c.M == 1 ? launch_rows<1, 32, 1>(d, s) : c.M == 2 ? launch_rows<2, 32, 1>(d, s)
           : c.M <= 4 ? launch_rows<4, 32, 1>(d, s) : launch_rows<8, 32, 1>(d, s);
  }
  return c.M == 1 ? launch_rows<1, 32, 2>(d, s) : c.M == 2 ? launch_rows<2, 32, 2>(d, s) : launch_rows<4, 32, 2>(d, s);
}

template <int NR, int L>
Error launch_rows_grad(const CrossDev& c, cudaStream_t s) {
  RowsGradDev d;
  std::memset(static_cast<void*>(&d), 0, sizeof(d));
  d.c = c;
  int e2 = 0;
  std::frexp(c.scale, &e2);
  d.s1 = std::ldexp(1.f, e2 / 2);
  d.s2 = c.scale / d.s1;
  constexpr int smem = kRowsThreads / L * NR * L * 4 * 4;
  auto k = c.vec ? cross_rows_grad_kernel<NR, L, true> : cross_rows_grad_kernel<NR, L, false>;
  allow_smem((const void*)k, smem);
  const int64_t np = (int64_t)c.B * c.Hk, splits = key_parts((const void*)k, smem, np, c.Tk);
  d.splits = (int)splits;
  d.ld = (c.D + 3) / 4 * 4;
  Scratch part;
  if (splits > 1) {
    Error e = part.alloc(sizeof(float) * (size_t)(splits * np * c.M) * d.ld, s);
    if (!e.ok()) return e;
    d.part = part.as<float>();
  }
  k<<<(unsigned)(np * splits), kRowsThreads, smem, s>>>(d);
  Error e = check_launch("cross attention rows gradient kernel");
  if (!e.ok() || splits == 1) return e;
  return launch_after(cross_rows_sum_kernel, dim3((unsigned)((np * c.M * d.ld + 255) / 256)), 256, 0, s,
                      "cross attention rows sum kernel", d);
}

template <int L>
Error run_rows_grad(const CrossDev& c, cudaStream_t s) {
  return c.M == 1 ? launch_rows_grad<1, L>(c, s) : c.M == 2 ? launch_rows_grad<2, L>(c, s)
         : c.M <= 4 ? launch_rows_grad<4, L>(c, s) : launch_rows_grad<8, L>(c, s);
}

struct CrossCall {
  const char* fn;
  const trs_view *q, *k, *v, *len;
  double scale;
  trs_view *out, *lse;                // forward outputs; inputs of the backward
  const trs_view* dout;               // backward
  trs_view *dq, *dk, *dv;
};

Error run_cross(const CrossCall& c, bool backward, cudaStream_t stream) {
  const std::string fn = c.fn;
  if (!c.q || !c.k || !c.v || !c.out || (backward && (!c.lse || !c.dout || !c.dq || !c.dk || !c.dv)))
    return make_error(TRS_ERR_ARG, fn + ": null view");
  const trs_view* heads[] = {c.q, c.k, c.v, c.out, c.dout, c.dq, c.dk, c.dv};
  const char* names[] = {"q", "k", "v", "the output", "the output gradient", "the q gradient", "the k gradient",
                         "the v gradient"};
  Error e;
  for (int i = 0; i < (backward ? 8 : 4); ++i) {
    e = check_heads(c.fn, heads[i], TRS_F32, names[i]);
    if (!e.ok()) return e;
  }
  if (!same_shape(c.out, c.q) || (backward && (!same_shape(c.dout, c.q) || !same_shape(c.dq, c.q))))
    return make_error(TRS_ERR_SHAPE, fn + ": the output and its gradient must have the shape of q");
  if (!same_shape(c.k, c.v) || (backward && (!same_shape(c.dk, c.k) || !same_shape(c.dv, c.k))))
    return make_error(TRS_ERR_SHAPE, fn + ": k, v and their gradients must have one shape");
  const int64_t B = c.q->shape[0], Tq = c.q->shape[1], Hq = c.q->shape[2], D = c.q->shape[3];
  const int64_t Tk = c.k->shape[1], Hk = c.k->shape[2];
  if (c.k->shape[0] != B || c.k->shape[3] != D)
    return make_error(TRS_ERR_SHAPE, fn + ": q and k must agree in batch and head size");
  if (Hk == 0 ? Hq != 0 : Hq % Hk != 0)
    return make_error(TRS_ERR_SHAPE, fn + ": the query heads must be a multiple of the key heads");
  if (D > kRowsMaxHead) return make_error(TRS_ERR_SHAPE, fn + ": a head size above 256");
  if (D < 1) return make_error(TRS_ERR_SHAPE, fn + ": an empty head");
  if (!(std::fabs(c.scale) < 0x1p127))  // its product with log2 e is an f32
    return make_error(TRS_ERR_ARG, fn + ": the scale must be below 2^127");
  if (c.lse) {
    e = validate_view(c.lse, "lse");
    if (!e.ok()) return e;
    if (c.lse->dtype != TRS_F32) return make_error(TRS_ERR_DTYPE, fn + ": lse must be f32");
    if (c.lse->ndim != 3 || c.lse->shape[0] != B || c.lse->shape[1] != Hq || c.lse->shape[2] != Tq)
      return make_error(TRS_ERR_SHAPE, fn + ": lse must be [batch, query heads, query tokens]");
  }
  if (c.len) {
    e = validate_view(c.len, "key lengths");
    if (!e.ok()) return e;
    if (c.len->dtype != TRS_I32 && c.len->dtype != TRS_I64)
      return make_error(TRS_ERR_DTYPE, fn + ": key lengths must be i32 or i64");
    if (c.len->ndim != 1 || c.len->shape[0] != B) return make_error(TRS_ERR_SHAPE, fn + ": key lengths must be [batch]");
  }
  // no output may share memory with an input or another output
  const trs_view* reads[] = {c.q, c.k, c.v, c.len, backward ? c.out : nullptr, backward ? c.lse : nullptr, c.dout};
  const trs_view* fw[] = {c.out, c.lse};
  const trs_view* bw[] = {c.dq, c.dk, c.dv};
  const trs_view** writes = backward ? bw : fw;
  const int nw = backward ? 3 : 2;
  for (int i = 0; i < nw; ++i) {
    if (!writes[i]) continue;
    if (writes_collide(writes[i])) return make_error(TRS_ERR_ALIAS, fn + ": two elements of an output share a place");
    for (const trs_view* r : reads)
      if (r && heads_overlap(writes[i], r)) return make_error(TRS_ERR_ALIAS, fn + ": an output overlaps an input");
    for (int j = 0; j < i; ++j)
      if (writes[j] && heads_overlap(writes[i], writes[j]))
        return make_error(TRS_ERR_ALIAS, fn + ": two outputs overlap");
  }
  const int64_t lim = (1ll << 31) - 65536;
  if (B * Hq >= lim || Tq >= lim || Tk >= lim || (Hk && Hq / Hk * Tq >= lim))
    return make_error(TRS_ERR_SHAPE, fn + ": 2^31 or more heads, tokens or rows");
  CrossDev d;
  std::memset(static_cast<void*>(&d), 0, sizeof(d));
  d.B = (int)B;
  d.Hq = (int)Hq;
  d.Hk = (int)Hk;
  d.Tq = (int)Tq;
  d.Tk = (int)Tk;
  d.D = (int)D;
  d.scale = (float)c.scale;
  d.q = heads_dev(c.q);
  d.k = heads_dev(c.k);
  d.v = heads_dev(c.v);
  d.out = heads_dev(c.out);
  if (c.lse) {
    d.lse = static_cast<float*>(c.lse->data) + c.lse->offset;
    d.ls_b = c.lse->strides[0];
    d.ls_h = c.lse->strides[1];
    d.ls_t = c.lse->strides[2];
  }
  if (c.len) {
    d.len64 = c.len->dtype == TRS_I64;
    d.len = static_cast<char*>(c.len->data) + c.len->offset * dtype_size(c.len->dtype);
    d.len_s = c.len->strides[0];
  }
  if (backward) {
    d.dout = heads_dev(c.dout);
    d.dq = heads_dev(c.dq);
    d.dk = heads_dev(c.dk);
    d.dv = heads_dev(c.dv);
  }
  if (B * Hq * Tq == 0 || Tk == 0) {  // no queries, or no keys at all
    if (!backward) {
      e = zero_heads(d.out, B, d.Tq, d.Hq, d.D, stream);
      if (!e.ok() || !c.lse || B * Hq * Tq == 0) return e;
      cross_lse_kernel<<<256, 256, 0, stream>>>(d);
      return check_launch("cross attention lse kernel");
    }
    e = zero_heads(d.dq, B, d.Tq, d.Hq, d.D, stream);
    if (e.ok()) e = zero_heads(d.dk, B, d.Tk, d.Hk, d.D, stream);
    if (e.ok()) e = zero_heads(d.dv, B, d.Tk, d.Hk, d.D, stream);
    return e;
  }
  d.G = (int)(Hq / Hk);
  d.M = d.G * d.Tq;
  d.f_Tq = make_fastdiv((uint32_t)d.Tq);
  auto aligned = [](const trs_view* v) {
    if (((uintptr_t)v->data + (uintptr_t)(v->offset * 4)) % 16 || v->shape[3] % 4) return false;
    if (v->strides[3] != 1) return false;
    for (int i = 0; i < 3; ++i)
      if (v->shape[i] > 1 && v->strides[i] % 4) return false;
    return true;
  };
  d.vec = 1;
  for (int i = 0; i < (backward ? 8 : 4); ++i) d.vec = d.vec && aligned(heads[i]);
  const int sms = current_device_info().sm_count;
  // up to 16 rows (8 of heads above 64) the CUDA cores read k and v faster than
  // the tensor-core path splits them.  4 x 16 heads, 2048 keys, CUDA cores and
  // tensor cores: heads of 64, 16 rows 40 and 58 us, 24 rows 66 and 58; heads
  // of 128, 8 rows 58 and 94, 16 rows 97 and 94
  if (backward && D <= 128 && d.M <= 8)
    return D <= 32 ? run_rows_grad<8>(d, stream) : D <= 64 ? run_rows_grad<16>(d, stream) : run_rows_grad<32>(d, stream);
  const bool tc = D <= 128 && (backward || d.M > (D <= 64 ? 16 : 8));
  if (!tc) {
    if (!backward) return run_rows(d, stream);
    cross_grad_rows_kernel<<<8 * sms, 256, 0, stream>>>(d);
    return check_launch("cross attention gradient rows kernel");
  }
  return backward ? cross_tc_backward(d, stream) : cross_tc_forward(d, stream);
}

trs_status finish(const Error& e) {
  if (!e.ok()) set_last_error(e.msg);
  return e.status;
}

}  // namespace
}  // namespace trs

using namespace trs;

extern "C" {

trs_status trs_cross_attention(const trs_view* q, const trs_view* k, const trs_view* v, const trs_view* key_lengths,
                               double scale, trs_view* out, trs_view* lse, trs_stream stream) {
  CrossCall c = {"cross_attention", q, k, v, key_lengths, scale, out, lse, nullptr, nullptr, nullptr, nullptr};
  return finish(run_cross(c, false, static_cast<cudaStream_t>(stream)));
}

trs_status trs_cross_attention_backward(const trs_view* grad_out, const trs_view* q, const trs_view* k,
                                        const trs_view* v, const trs_view* key_lengths, const trs_view* out,
                                        const trs_view* lse, double scale, trs_view* grad_q, trs_view* grad_k,
                                        trs_view* grad_v, trs_stream stream) {
  CrossCall c = {"cross_attention_backward", q, k, v, key_lengths, scale, const_cast<trs_view*>(out),
                 const_cast<trs_view*>(lse), grad_out, grad_q, grad_k, grad_v};
  return finish(run_cross(c, true, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
