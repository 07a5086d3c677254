// heads.h -- host-side checks shared by the attention-layer operators
// (rotary.cu, cross_attention.cu): views of the layout [batch, tokens, heads,
// head size], their overlap, and the small tables that go with them.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <string>

#include "plan.h"

namespace trs {

// A [B, T, H, D] operand as the kernels see it: element (0,0,0,0) and the
// four strides in elements.
struct HeadsDev {
  void* p = nullptr;
  int64_t sb = 0, st = 0, sh = 0, sd = 0;
};

inline HeadsDev heads_dev(const trs_view* v) {
  HeadsDev h;
  h.p = static_cast<char*>(v->data) + v->offset * dtype_size(v->dtype);
  h.sb = v->strides[0];
  h.st = v->strides[1];
  h.sh = v->strides[2];
  h.sd = v->strides[3];
  return h;
}

// Valid, rank 4, of `dtype`.
inline Error check_heads(const char* fn, const trs_view* v, int dtype, const char* what) {
  Error e = validate_view(v, what);
  if (!e.ok()) return e;
  if (v->ndim != 4)
    return make_error(TRS_ERR_SHAPE, std::string(fn) + ": " + what + " must be [batch, tokens, heads, head size]");
  if (v->dtype != dtype) return make_error(TRS_ERR_DTYPE, std::string(fn) + ": " + what + " has another dtype");
  return Error{};
}

inline bool same_shape(const trs_view* a, const trs_view* b) {
  if (a->ndim != b->ndim) return false;
  for (int i = 0; i < a->ndim; ++i)
    if (a->shape[i] != b->shape[i]) return false;
  return true;
}

// The very same elements in the same order: an output that is its own input.
inline bool same_elements(const trs_view* a, const trs_view* b) {
  if (!same_shape(a, b) || a->dtype != b->dtype) return false;
  const int64_t es = dtype_size(a->dtype);
  if ((int64_t)(uintptr_t)a->data + a->offset * es != (int64_t)(uintptr_t)b->data + b->offset * es) return false;
  for (int i = 0; i < a->ndim; ++i)
    if (a->shape[i] > 1 && a->strides[i] != b->strides[i]) return false;
  return true;
}

// Whether two elements of an output may share a place (a stride of 0, or
// dimensions that run into one another): every dimension, taken by its
// stride, has to step past all that the smaller ones reach.
inline bool writes_collide(const trs_view* v) {
  int64_t st[kMaxDims], n[kMaxDims];
  int m = 0;
  for (int i = 0; i < v->ndim; ++i) {
    if (v->shape[i] == 0) return false;
    if (v->shape[i] == 1) continue;
    const int64_t s = v->strides[i] < 0 ? -v->strides[i] : v->strides[i];
    int j = m++;
    for (; j > 0 && st[j - 1] > s; --j) {
      st[j] = st[j - 1];
      n[j] = n[j - 1];
    }
    st[j] = s;
    n[j] = v->shape[i];
  }
  int64_t reach = 0;
  for (int i = 0; i < m; ++i) {
    if (st[i] <= reach) return true;
    reach += (n[i] - 1) * st[i];
  }
  return false;
}

// Whether two views may reach a common byte.  They do not when their byte
// ranges are apart, or when they are apart inside a period: of any stride P,
// dimensions of either view that step by multiples of P only move by whole
// periods, and what the others reach, taken modulo P, are two intervals of a
// circle.  That covers slices of one buffer along any of its dimensions (queries,
// keys and values inside one projection's output).
inline bool heads_overlap(const trs_view* a, const trs_view* b) {
  if (numel_of(a->shape, a->ndim) == 0 || numel_of(b->shape, b->ndim) == 0) return false;
  // the bytes reached by the dimensions that do not step by multiples of `period`
  // (0: by all of them)
  auto range = [](const trs_view* v, int64_t period, int64_t* lo, int64_t* hi) {
    const int64_t es = dtype_size(v->dtype);
    int64_t l = v->offset * es, h = l + es;
    for (int i = 0; i < v->ndim; ++i) {
      const int64_t step = v->strides[i] * es, span = (v->shape[i] - 1) * step;
      if (span == 0 || (period > 0 && step % period == 0)) continue;
      if (span > 0) h += span; else l += span;
    }
    *lo = (int64_t)(uintptr_t)v->data + l;
    *hi = (int64_t)(uintptr_t)v->data + h;
  };
  int64_t alo, ahi, blo, bhi;
  range(a, 0, &alo, &ahi);
  range(b, 0, &blo, &bhi);
  if (alo >= bhi || blo >= ahi) return false;
  for (const trs_view* v : {a, b}) {
    for (int i = 0; i < v->ndim; ++i) {
      int64_t period = v->strides[i] * dtype_size(v->dtype);
      if (period < 0) period = -period;
      if (v->shape[i] < 2 || period == 0) continue;
      range(a, period, &alo, &ahi);
      range(b, period, &blo, &bhi);
      int64_t d = (blo - alo) % period;
      if (d < 0) d += period;
      if (d >= ahi - alo && d + (bhi - blo) <= period) return false;
    }
  }
  return true;
}

}  // namespace trs
