// cross.h -- descriptors shared by the cross-attention translation units
// (cross_attention.cu: checks, the CUDA-core kernels; cross_tc.cu: the tensor
// core kernels).
//
// Heads are grouped: G = Hq / Hk query heads read one key head, so a "problem"
// is one (batch, key head) with the M = G * Tq query rows of its group, row
// r = g * Tq + t, against its batch's keys.  Nothing in the kernels depends on
// the order of the rows, and a key head's gradient is summed over its group by
// the same product that sums it over the tokens.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "heads.h"
#include "kernels.cuh"

namespace trs {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct CrossDev {
  HeadsDev q, k, v, out;         // out: the output (forward), read by the backward
  HeadsDev dout, dq, dk, dv;     // backward
  float* lse;                    // [B, Hq, Tq] through its strides, or null
  int64_t ls_b, ls_h, ls_t;
  const void* len;               // key lengths or null
  int len64;
  int64_t len_s;
  int B, Hq, Hk, G, Tq, Tk, D;
  int M;                         // G * Tq
  FastDiv f_Tq;
  float scale;
  const int* nonfinite;          // tensor-core paths: set when an input holds an infinity or a NaN
  int vec;                       // q, k, v (and the outputs) take 16-byte accesses
};

// The keys of batch b: its length, clamped to [0, Tk].
__device__ __forceinline__ int key_count(const void* len, int len64, int64_t s, int Tk, int b) {
  if (!len) return Tk;
  const int64_t n = len64 ? static_cast<const int64_t*>(len)[b * s] : static_cast<const int32_t*>(len)[b * s];
  return n < 0 ? 0 : n > Tk ? Tk : (int)n;
}

// 2^x.  ex2.approx is off by at most 2 units; arguments here are differences
// to a maximum, and results below 2^-126 flush to 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The smaller of the two, NaN where either is.
__device__ __forceinline__ float min_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

// Two f32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The tensor-core paths (head sizes up to 128).
Error cross_tc_forward(const CrossDev& d, cudaStream_t stream);
Error cross_tc_backward(const CrossDev& d, cudaStream_t stream);

}  // namespace trs
