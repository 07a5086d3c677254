// cross_exact.cuh -- cross attention and its gradient row by row in f32, a warp
// per row, each lane holding elements lane, lane + 32, ... of a head: for the
// gradient of head sizes above 128, and for calls whose inputs hold an
// infinity or a NaN, which the tensor-core kernels hand over to this code (a
// split product would turn an infinity times a zero low part into NaN).
#pragma once

#include "cross.h"

namespace trs {

constexpr int kExactE = 8;  // elements per lane: head sizes up to 256

struct HeadRow {
  float x[kExactE];
};
__device__ __forceinline__ HeadRow load_row(const HeadsDev& h, int b, int t, int head, int D) {
  const float* p = static_cast<const float*>(h.p) + b * h.sb + t * h.st + head * h.sh;
  HeadRow r;
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int i = 0; i < kExactE; ++i) r.x[i] = lane + 32 * i < D ? p[(lane + 32 * i) * h.sd] : 0.f;
  return r;
}
__device__ __forceinline__ void store_row(const HeadsDev& h, int b, int t, int head, int D, const HeadRow& r) {
  float* p = static_cast<float*>(h.p) + b * h.sb + t * h.st + head * h.sh;
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int i = 0; i < kExactE; ++i)
    if (lane + 32 * i < D) p[(lane + 32 * i) * h.sd] = r.x[i];
}
__device__ __forceinline__ float dot_row(const HeadRow& a, const HeadRow& b) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kExactE; ++i) s = __fmaf_rn(a.x[i], b.x[i], s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ HeadRow times(HeadRow r, float f) {
#pragma unroll
  for (int i = 0; i < kExactE; ++i) r.x[i] *= f;
  return r;
}
__device__ __forceinline__ HeadRow zero_row() {
  HeadRow r;
#pragma unroll
  for (int i = 0; i < kExactE; ++i) r.x[i] = 0.f;
  return r;
}

// Every query row of the call, warp `w` of `warps`: out and lse.
static __device__ __noinline__ void exact_rows(const CrossDev& c, int64_t w, int64_t warps) {
  const int64_t nq = (int64_t)c.B * c.Hq * c.Tq;
  for (; w < nq; w += warps) {
    const int t = (int)(w % c.Tq), h = (int)(w / c.Tq % c.Hq), b = (int)(w / c.Tq / c.Hq), hk = h / c.G;
    const int n = key_count(c.len, c.len64, c.len_s, c.Tk, b);
    const HeadRow q = times(load_row(c.q, b, t, h, c.D), c.scale * kLog2e);
    HeadRow acc = zero_row();
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < n; ++j) {
      const float s = dot_row(q, load_row(c.k, b, j, hk, c.D));
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
      const float alpha = ex2(m - base), p = ex2(s - base);
      const HeadRow v = load_row(c.v, b, j, hk, c.D);
      m = mn;
      l = __fmaf_rn(l, alpha, p);
#pragma unroll
      for (int i = 0; i < kExactE; ++i) acc.x[i] = __fmaf_rn(p, v.x[i], acc.x[i] * alpha);
    }
#pragma unroll
    for (int i = 0; i < kExactE; ++i) acc.x[i] = l == 0.f ? 0.f : acc.x[i] / l;
    store_row(c.out, b, t, h, c.D, acc);
    if (threadIdx.x % 32 == 0 && c.lse) c.lse[b * c.ls_b + h * c.ls_h + t * c.ls_t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  }
}

// P and dS of one pair, of q times the scale.  P = exp(S - lse) is a weight, at most 1: scores of 1e6
// and more are off by that much from lse, which holds 24 bits of them.
struct PairGrad {
  float p, ds;
};
__device__ __forceinline__ PairGrad pair_grad(const HeadRow& q, const HeadRow& go, const HeadRow& k, const HeadRow& v,
                                              float lse, float delta) {
  PairGrad r;
  const float s = dot_row(q, k);
  r.p = lse == -INFINITY ? 0.f : ex2(min_nan((s - lse) * kLog2e, 0.f));
  r.ds = r.p * (dot_row(go, v) - delta);
  return r;
}

// Every query row: dq.
static __device__ __noinline__ void exact_dq_rows(const CrossDev& c, int64_t w, int64_t warps) {
  const int64_t nq = (int64_t)c.B * c.Hq * c.Tq;
  for (; w < nq; w += warps) {
    const int t = (int)(w % c.Tq), h = (int)(w / c.Tq % c.Hq), b = (int)(w / c.Tq / c.Hq), hk = h / c.G;
    const int n = key_count(c.len, c.len64, c.len_s, c.Tk, b);
    const HeadRow q = times(load_row(c.q, b, t, h, c.D), c.scale), go = load_row(c.dout, b, t, h, c.D);
    const float delta = dot_row(go, load_row(c.out, b, t, h, c.D));
    const float lse = c.lse[b * c.ls_b + h * c.ls_h + t * c.ls_t];
    HeadRow acc = zero_row();
    for (int j = 0; j < n; ++j) {
      const HeadRow k = load_row(c.k, b, j, hk, c.D);
      const PairGrad g = pair_grad(q, go, k, load_row(c.v, b, j, hk, c.D), lse, delta);
#pragma unroll
      for (int i = 0; i < kExactE; ++i) acc.x[i] = __fmaf_rn(g.ds, k.x[i] * c.scale, acc.x[i]);
    }
    store_row(c.dq, b, t, h, c.D, acc);
  }
}

// Every key row: dk and dv, 0 at and behind the key length.
static __device__ __noinline__ void exact_dkv_rows(const CrossDev& c, int64_t w, int64_t warps) {
  const int64_t nk = (int64_t)c.B * c.Hk * c.Tk;
  for (; w < nk; w += warps) {
    const int j = (int)(w % c.Tk), hk = (int)(w / c.Tk % c.Hk), b = (int)(w / c.Tk / c.Hk);
    HeadRow ak = zero_row(), av = zero_row();
    if (j < key_count(c.len, c.len64, c.len_s, c.Tk, b)) {
      const HeadRow k = load_row(c.k, b, j, hk, c.D), v = load_row(c.v, b, j, hk, c.D);
      for (int h = hk * c.G; h < (hk + 1) * c.G; ++h) {
        for (int t = 0; t < c.Tq; ++t) {
          const HeadRow q = times(load_row(c.q, b, t, h, c.D), c.scale), go = load_row(c.dout, b, t, h, c.D);
          const float delta = dot_row(go, load_row(c.out, b, t, h, c.D));
          const PairGrad g = pair_grad(q, go, k, v, c.lse[b * c.ls_b + h * c.ls_h + t * c.ls_t], delta);
#pragma unroll
          for (int i = 0; i < kExactE; ++i) {
            ak.x[i] = __fmaf_rn(g.ds, q.x[i], ak.x[i]);
            av.x[i] = __fmaf_rn(g.p, go.x[i], av.x[i]);
          }
        }
      }
    }
    store_row(c.dk, b, j, hk, c.D, ak);
    store_row(c.dv, b, j, hk, c.D, av);
  }
}

}  // namespace trs
