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
// head_list_kernel) and the join of the vocabulary's parts.  head_few.cu: few rows,
// which HBM bounds; head_tc.cu: more.
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

// A warp per row: the softmax of the entries that are there, sorted by token.  The
// rank of an entry is counted, K^2 / 32 steps of the warp, which suits the tens of
// entries that are kept in earnest: 8192 rows of 64 entries 27 us, of 128 86, but of
// 1024 4.8 ms (and 7 rows of those 0.86 ms).
__global__ void __launch_bounds__(256) head_teacher_kernel(const HeadDev d) {
  extern __shared__ int s_id[];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int row = blockIdx.x * 8 + warp;
  pdl_wait();  // before the line below: see head_list_kernel
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
      if (p != 0.f) ent += (double)p * (double)(a - ln_sum);  // 0 ln 0 = 0; a may have left f32's range
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
  // What runs next may read the call's inputs and write its workspaces without waiting
  // for this kernel: it must not begin before the call's first kernel has waited for
  // all that came before the call (so the workspaces were taken before that launch).
  // With a teacher's rows that kernel is theirs.
  const bool first = !d.distill || d.N == 0;
  if (!first) pdl_launch_dependents();
  pdl_wait();
  if (first) pdl_launch_dependents();
  constexpr int U = 4;  // consecutive rows of a thread
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int done = 0;
  for (int r0 = 0; r0 < d.N; r0 += 1024 * U) {
    int id[U], mine = 0;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int row = r0 + threadIdx.x * U + j;
      id[j] = row < d.N ? head_first_id(d, row) : kNoToken;
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int row = r0 + threadIdx.x * U + j;
      mine += id[j] != kNoToken;
      if (row >= d.N) continue;
      if (!d.distill) {
        d.eid[row] = id[j];
        d.ew[row] = d.weight;
      }
      if (id[j] == kNoToken && d.loss.p) {
        *head_row<float>(d, d.loss, row) = 0.f;
        if (d.lse.p) *head_row<float>(d, d.lse, row) = 0.f;
      }
    }
    // where this thread's rows begin in the list: the lanes before it, then the warps
    int scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += y;
    }
    if (lane == 31) warps[warp] = scan;
    __syncthreads();
    int at = warps[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += y;
    }
    const int all = __shfl_sync(0xffffffffu, at, 31), before = __shfl_sync(0xffffffffu, at, warp > 0 ? warp - 1 : 0);
    int to = done + (warp > 0 ? before : 0) + scan - mine;
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (id[j] != kNoToken) d.rows[to++] = r0 + threadIdx.x * U + j;
    done += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *d.live = done;
}

// ---- joining the parts of the vocabulary -------------------------------------------

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
  d.vec_dh = N > 0 && c.grad_hidden && rows_vectors(c.grad_hidden);
  if (N == 0 && !d.dw) return Error{};
  // Without rows head_tc.cu writes the zeros.
  const bool few = head_few_takes(d, c.backward);
  // the rows' targets
  Scratch mem;
  const size_t n = ((size_t)N + 3) / 4 * 4, nk = ((size_t)N * K + 3) / 4 * 4;
  HeadTcPlan plan;
  if (!few) {
    e = head_tc_plan(d, c.backward, &plan);
    if (!e.ok()) return e;
  }
  const size_t tc = few ? 0 : plan.bytes;
  if (!few || c.distill) {
    e = mem.alloc(tc + 4 * (n + 4 + 2 * nk + (c.distill ? n : 0)), stream);
    if (!e.ok()) return e;
    d.live = reinterpret_cast<int*>(mem.as<char>() + tc);
    d.rows = d.live + 4;
    d.eid = d.rows + n;
    d.ew = reinterpret_cast<float*>(d.eid + nk);
    d.ent = d.ew + nk;
  }
  if (c.distill && N > 0) {
    const int smem = 8 * 2 * d.K * 4;
    allow_smem((const void*)head_teacher_kernel, smem);
    e = launch_after(head_teacher_kernel, dim3((unsigned)((N + 7) / 8)), 256, smem, stream, "head teacher kernel", d);
    if (!e.ok()) return e;
  }
  if (few) return head_few(d, c.backward, stream);
  e = launch_after(head_list_kernel, dim3(1), 1024, 0, stream, "head list kernel", d);
  if (!e.ok()) return e;
  return head_tc(d, c.backward, plan, mem.as<char>(), stream);
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
    try {
      set_last_error("out of host memory");
    } catch (...) {
    }
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
