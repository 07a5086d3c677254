// tokens.h -- host-side checks shared by the operators on rows of tokens
// (embedding.cu, head.cu): views of the layout [tokens, ...] or
// [batch, tokens, ...] with any strides, and how the kernels see them.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <string>

#include "heads.h"

namespace trs {

// Element (0, 0, 0) and the strides of batch, token and element.
struct RowsDev {
  void* p = nullptr;
  int64_t sb = 0, st = 0, sd = 0;
};

// The leading dimensions that every operand of a call shares.
struct Tokens {
  int lead = 1;          // 1: [tokens, ...], 2: [batch, tokens, ...]
  int64_t B = 1, T = 0;
  int64_t n() const { return B * T; }
};

inline Tokens tokens_of(const trs_view* v, int lead) {
  Tokens t;
  t.lead = lead;
  t.B = lead == 2 ? v->shape[0] : 1;
  t.T = v->shape[lead - 1];
  return t;
}

// Valid, with the leading dimensions of `t` and `inner` (0 or 1) more.
inline Error check_tokens(const std::string& fn, const trs_view* v, const Tokens& t, int inner, const char* what) {
  Error e = validate_view(v, what);
  if (!e.ok()) return e;
  if (v->ndim != t.lead + inner || (t.lead == 2 && v->shape[0] != t.B) || v->shape[t.lead - 1] != t.T)
    return make_error(TRS_ERR_SHAPE, fn + ": " + what + " must be " + (t.lead == 2 ? "[batch, tokens" : "[tokens") +
                                         (inner ? ", ...] like the other operands" : "] like the other operands"));
  return Error{};
}

inline RowsDev rows_dev(const trs_view* v, const Tokens& t) {
  RowsDev r;
  r.p = static_cast<char*>(v->data) + v->offset * dtype_size(v->dtype);
  r.sb = t.lead == 2 ? v->strides[0] : 0;
  r.st = v->strides[t.lead - 1];
  r.sd = v->ndim > t.lead ? v->strides[t.lead] : 0;
  return r;
}

// Whether every row of `v` can be read and written in 16-byte pieces along its
// last dimension.
inline bool rows_vectors(const trs_view* v) {
  const int es = dtype_size(v->dtype), vw = 16 / es, n = v->ndim;
  if (((uintptr_t)v->data + (uintptr_t)(v->offset * es)) % 16) return false;
  if (v->shape[n - 1] % vw || v->strides[n - 1] != 1) return false;
  for (int i = 0; i < n - 1; ++i)
    if (v->shape[i] > 1 && v->strides[i] % vw) return false;
  return true;
}

// No output shares memory with an input or with another output, and no two of
// its own elements share a place.  Null views are left out.
inline Error check_outputs(const std::string& fn, std::initializer_list<const trs_view*> writes,
                           std::initializer_list<const trs_view*> reads) {
  for (const trs_view* const* w = writes.begin(); w != writes.end(); ++w) {
    if (!*w) continue;
    if (writes_collide(*w)) return make_error(TRS_ERR_ALIAS, fn + ": two elements of an output share a place");
    for (const trs_view* r : reads)
      if (r && heads_overlap(*w, r)) return make_error(TRS_ERR_ALIAS, fn + ": an output overlaps an input");
    for (const trs_view* const* o = writes.begin(); o != w; ++o)
      if (*o && heads_overlap(*w, *o)) return make_error(TRS_ERR_ALIAS, fn + ": two outputs overlap");
  }
  return Error{};
}

}  // namespace trs
