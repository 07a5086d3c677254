// head.h -- what the translation units of a model's last layer share (head.cu:
// checks, the rows' targets, the join of the vocabulary's parts; head_few.cu: few
// rows; head_tc.cu: more).
//
// Both losses are  lse(x) - sum_v t_v x_v  of the scores x = h w^T / temperature
// against a target distribution t, up to a constant of the row and the factor
// temperature^2; t is a few entries (one for a class, K for a teacher's logits)
// and, for smoothed classes, s / V everywhere.  The gradient of x is softmax(x) - t.
// A row's entries are prepared once per call, sorted by their token; where a token
// comes several times, its first entry has all of its weight and the others 0.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kernels.cuh"
#include "tokens.h"

namespace trs {

constexpr float kHeadLog2e = 1.4426950408889634f;
constexpr double kHeadLn2 = 0.6931471805599453;
constexpr int kNoToken = 0x7fffffff;

struct HeadDev {
  RowsDev hid, dh;               // [.., D]
  const float* w;                // [V, D]
  int64_t wv, wd;
  float* dw;                     // or null
  int64_t dwv, dwd;
  RowsDev ids, z;                // targets [..], or teacher ids and logits [.., K]
  int ids64;
  RowsDev gl, loss, lse;         // [..]
  int N, V, D, K;
  FastDiv f_T;
  int distill;
  float temp, inv_temp;
  float share;                   // s / V
  float weight;                  // 1 - s, a class's entry
  // prepared by head_targets
  int* rows;                     // the rows with a target, in order
  int* live;                     // how many
  int* eid;                      // [N][K] tokens of a row's entries, ascending, kNoToken behind them
  float* ew;                     // [N][K] their weights
  float* ent;                    // [N] sum of w ln w (distillation)
  int vec_h, vec_w, vec_dh, vec_dw;  // 16-byte accesses along D
};

__device__ __forceinline__ float head_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// softmax(x) from the row's lse, the exponent `z` in units of log2: at most 1.  lse is
// rounded to f32, which at scores of 1e7 and more is worth more than the exponential's
// range; a NaN stays one.
__device__ __forceinline__ float head_softmax(float z) {
  asm("min.NaN.f32 %0, %0, 0f00000000;" : "+f"(z));
  return head_ex2(z);
}

template <class T>
__device__ __forceinline__ T* head_row(const HeadDev& d, const RowsDev& r, int i) {
  const uint32_t b = fdiv((uint32_t)i, d.f_T), t = (uint32_t)i - b * d.f_T.d;
  return static_cast<T*>(r.p) + b * r.sb + t * r.st;
}

__device__ __forceinline__ int head_id(const HeadDev& d, const RowsDev& ids, int row, int k) {
  const int64_t at = k * ids.sd;
  const int64_t v = d.ids64 ? head_row<const int64_t>(d, ids, row)[at] : head_row<const int32_t>(d, ids, row)[at];
  return v < 0 || v >= d.V ? kNoToken : (int)v;
}

// The first of a row's tokens in order (kNoToken: the row has no target).
__device__ __forceinline__ int head_first_id(const HeadDev& d, int row) {
  return d.distill ? d.eid[(int64_t)row * d.K] : head_id(d, d.ids, row, 0);
}

// The walk of one row's entries along ascending tokens.
struct Entries {
  const int* id;
  const float* w;
  int left;
  int next;
  __device__ __forceinline__ void begin(const HeadDev& d, int row) {
    id = d.eid + (int64_t)row * d.K;
    w = d.ew + (int64_t)row * d.K;
    left = d.K;
    next = *id;
  }
  __device__ __forceinline__ void step() {
    ++w;
    ++id;
    next = --left > 0 ? *id : kNoToken;
  }
  // skips entries below v, which may be all of them
  __device__ __forceinline__ void skip_to(int v) {
    int lo = 0, hi = left;  // entries before `lo` are below v, those from `hi` on are not
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (id[mid] < v) lo = mid + 1; else hi = mid;
    }
    id += lo;
    w += lo;
    left -= lo;
    next = left > 0 ? *id : kNoToken;
  }
  // the weight of token v, which next may have reached
  __device__ __forceinline__ float take(int v) {
    float s = 0.f;
    while (next == v) {
      s += *w;
      step();
    }
    return s;
  }
};

// Partial statistics of a row over a part of the vocabulary: the largest score
// in units of log2, the sum of 2^(score - largest), sum of weight times score and
// sum of scores in units of log2 too.
struct HeadPart {
  float m, s, dot, sum;
};
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

// part p of live row r (few: of the call's row r) lies at p * sp + r * sr
Error head_join(const HeadDev& d, const HeadPart* part, int parts, int64_t sp, int64_t sr, bool few,
                cudaStream_t stream);

// Few rows (head_few.cu).  8 or 16 of them share a read of the weight, which head_tc.cu
// reads, splits, writes and reads again, for 1 to 256 rows alike: on 32000 x 1024,
// scores of 17 rows 82 us here, of 33 98 there; gradients of 8 rows 88 here, of 16 118,
// of two blocks of rows 257, and 201 there.  Widths up to 4096 (scores of 4 rows
// on 32000: of 4096 103 us here, of 4104 388 there), as shared memory holds; gradients of
// weights whose columns lie apart are walked badly here (8 rows 490 us, 298 there).
inline bool head_few_takes(const HeadDev& d, bool backward) {
  if (d.N < 1 || d.D > 4096) return false;
  if (!backward) return d.N <= 32;
  if (d.wd != 1 && d.D > 1) return false;
  return d.N <= 8 || (d.N <= 16 && d.vec_w && d.D <= 2560);
}
Error head_few(const HeadDev& d, bool backward, cudaStream_t stream);
// More rows, wider ones, or none (head_tc.cu).  How the work is cut, and where its workspaces lie
// in `bytes` of memory, which the call takes before its first launch: its first planes
// are written without waiting for the kernel before them, so the memory must not come
// from anything that was issued, on the same stream by another host thread, after that
// launch.
struct HeadTcPlan {
  int64_t Np, Dp, dtiles;        // rows and width of the planes, tiles along the width
  int64_t Vp, pieces;            // rows of a piece of the vocabulary
  int64_t htiles, wtiles;
  int splits, wsplits;           // parts of dh's and dw's contraction
  size_t wdown, gdown, hdown, h, w, gh, x, part, dh, dw;  // offsets
  size_t bytes;
};
Error head_tc_plan(const HeadDev& d, bool backward, HeadTcPlan* plan);
Error head_tc(const HeadDev& d, bool backward, const HeadTcPlan& plan, char* base, cudaStream_t stream);

}  // namespace trs
