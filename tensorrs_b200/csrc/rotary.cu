// rotary.cu -- rotary positions and the per-head norm of queries and keys.
//
//   trs_rotary             y = R(p) x
//   trs_rotary_backward    dx = R(p)^T dy
//   trs_head_norm_rotary   n = x / sqrt(mean(x^2) + eps), y = R(p) (n * gamma)
//   ..._backward           g = R(p)^T dy, dgamma = sum g n, dn = g gamma,
//                          dx = (dn - n mean(dn n)) / sqrt(mean(x^2) + eps)
//
// R(p) turns pair i of the first `rotary` elements of a head by the angle
// p f_i, (a, b) -> m (a cos - b sin, b cos + a sin), and leaves the rest.  The
// pairs are (i, i + rotary / 2) in the half layout and (2i, 2i + 1) in the
// interleaved one.
//
// What bounds it: HBM.  Every element is read once and written once (the
// backward reads x and dy), so the floor is 2 (3) element sizes per element.
// A group of G lanes (a power of two, at most a warp) owns a token: each lane
// keeps its pairs' cos and sin in registers and walks heads with them, so an
// angle is evaluated once per token and chunk of heads instead of once per
// element, and no table of cos and sin is read.  A lane's unit is two 16-byte
// vectors of a head (V pairs); UH heads are loaded before the first is
// used, which keeps 2 UH (4 UH) 16-byte loads of a lane in flight.
// The sums of a row (x^2, dn n) are folded over the group with shuffles.
// Measured, 8192 tokens of 40 heads of 128 in f32 (336 MB): 57 us rotated
// (5.9 TB/s, 0.92 of the copy rate), 62 us normed and rotated (5.4 TB/s), 124
// normed and rotated in f64; the norm's gradient of 4096 tokens of 20 heads of 64
// (63 MB) 21 us and 6 more for the gammas (33 and 6 in f64).  The f64 rotation of
// 2000 tokens of 24 heads of 64 (49 MB) 8.2 us.
//
// Angles: the product p f_i is taken in f64 (positions of a long context times
// a frequency of 1 lose the fraction of a turn in f32); for f32 tensors the
// turns are reduced in f64 and sin and cos taken in f32 of the remainder (off
// by less than 2^-24 of a turn at any position), for f64 tensors all of it is f64.
// The row sums stay in the element type (f32 over at most 512 squares, 32
// lanes' partial sums folded as a tree); dgamma, a sum over all rows, is
// accumulated over the heads of a token (8 at most) in the element type and
// over the tokens in f64, folded over the CTA and then over the CTAs in a fixed
// order, and rounded once.
#include <cmath>
#include <cstring>

#include "../../include/trs.h"
#include "heads.h"
#include "kernels.cuh"

namespace trs {
namespace {

enum RotMode { kRotate = 0, kNormRotate = 1, kNormBackward = 2 };

constexpr int kRotThreads = 256;
constexpr int kRotMaxHead = 512;

struct RotDev {
  HeadsDev x[2], y[2], dy[2];    // queries, keys: input, output, output gradient (backward)
  int64_t blocks0;               // CTAs of the queries; the rest serve the keys
  int H[2];
  int hpc;                       // heads per chunk
  int64_t items[2];              // tokens * chunks, below 2^31
  FastDiv f_chunks[2], f_T;
  const void* pos;
  int pos64;
  int64_t ps_b, ps_t;
  const double* freq;
  int64_t fs;
  const void* gamma[2];          // or null: ones
  int64_t gs[2];
  double* part[2];               // [CTAs][D] partial dgamma, or null
  double magnitude, eps;
  int D, R, NR, NU;              // head size, rotated elements, rotated units, units
  int inverse;
};

template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

template <class T> __device__ __forceinline__ T rfma(T a, T b, T c) {
  if constexpr (sizeof(T) == 4) return __fmaf_rn(a, b, c);
  else return __fma_rn(a, b, c);
}

// 1 / sqrt(mean + eps), both steps rounded to nearest
__device__ __forceinline__ float inv_norm(float ss, float D, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, D), eps)));
}
__device__ __forceinline__ double inv_norm(double ss, double D, double eps) {
  return __ddiv_rn(1.0, __dsqrt_rn(__dadd_rn(__ddiv_rn(ss, D), eps)));
}

// cos and sin of p f(0), .., p f(V - 1), times the magnitude
template <int V, class F>
__device__ __forceinline__ void turn(double p, F f, double magnitude, float (&c)[V], float (&s)[V]) {
  double h[V], t[V];
  int high = 0;  // the upper word of the largest |h|
#pragma unroll
  for (int i = 0; i < V; ++i) {
    h[i] = p * f(i) * 0x1.45f306dc9c883p-3;  // turns
    t[i] = h[i] - rint(h[i]);
    high = max(high, __double2hiint(h[i]) & 0x7fffffff);
  }
  // h is off by 2^-53 of itself twice: past 2^26 turns with what its rounding and
  // that of 1 / (2 pi) left, so that the fraction stays exact to 2^-50
  if (high >= 0x41900000) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double a = p * f(i);
      t[i] += __fma_rn(a, -0x1.6b01ec5417056p-57, __fma_rn(a, 0x1.45f306dc9c883p-3, -h[i]));
      t[i] -= rint(t[i]);
    }
  }
  const float m = (float)magnitude;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float sn, cs;
    sincospif((float)(2.0 * t[i]), &sn, &cs);
    c[i] = cs * m;
    s[i] = sn * m;
  }
}
template <int V, class F>
__device__ __forceinline__ void turn(double p, F f, double magnitude, double (&c)[V], double (&s)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    double sn, cs;
    sincos(p * f(i), &sn, &cs);
    c[i] = cs * magnitude;
    s[i] = sn * magnitude;
  }
}

// (a, b) of a unit turned by its V angles.  IL: the pairs lie inside the
// vectors (a[0],a[1]), ...; else pair i is (a[i], b[i]).
template <class T, int V, bool IL>
__device__ __forceinline__ void rotate(T (&a)[V], T (&b)[V], const T (&c)[V], const T (&s)[V]) {
  if constexpr (IL && V > 1) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const T p = a[2 * i], q = a[2 * i + 1];
      a[2 * i] = rfma(p, c[i], -(q * s[i]));
      a[2 * i + 1] = rfma(q, c[i], p * s[i]);
      const T u = b[2 * i], w = b[2 * i + 1];
      b[2 * i] = rfma(u, c[V / 2 + i], -(w * s[V / 2 + i]));
      b[2 * i + 1] = rfma(w, c[V / 2 + i], u * s[V / 2 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const T p = a[i], q = b[i];
      a[i] = rfma(p, c[i], -(q * s[i]));
      b[i] = rfma(q, c[i], p * s[i]);
    }
  }
}

// One unit's place: the element offsets of its two vectors, whether each
// exists, and whether it is rotated.
struct Unit {
  int o0, o1;
  bool v0, v1, rot;
};
template <int V, bool IL>
__device__ __forceinline__ Unit unit_of(const RotDev& d, int u) {
  Unit n;
  n.rot = u < d.NR;
  if (n.rot) {
    n.o0 = IL ? 2 * V * u : V * u;
    n.o1 = IL ? n.o0 + V : d.R / 2 + V * u;
    n.v0 = n.v1 = true;
  } else {
    n.o0 = d.R + (u - d.NR) * 2 * V;
    n.o1 = n.o0 + V;
    n.v0 = u < d.NU && n.o0 < d.D;
    n.v1 = u < d.NU && n.o1 < d.D;
  }
  return n;
}

template <class T, int V>
__device__ __forceinline__ void load_vec(T (&r)[V], const T* p, int64_t at, int64_t sd, bool ok) {
  if (!ok) {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = T(0);
    return;
  }
  const Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(p + (V == 1 ? at * sd : at));
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = x.v[i];
}
template <class T, int V>
__device__ __forceinline__ void store_vec(T* p, int64_t at, int64_t sd, const T (&r)[V], bool ok) {
  if (!ok) return;
  Vec<T, V> x;
#pragma unroll
  for (int i = 0; i < V; ++i) x.v[i] = r[i];
  *reinterpret_cast<Vec<T, V>*>(p + (V == 1 ? at * sd : at)) = x;
}

template <class T, int G>
__device__ __forceinline__ T group_sum(T x, unsigned mask) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) x += __shfl_xor_sync(mask, x, o, G);
  return x;
}

// V: elements per vector access (1: any strides).  K: units per lane.  UH:
// heads in flight.  G: lanes per token.
// The norm's forward is held to the registers of three CTAs per SM (8192 tokens
// of 40 heads of 128: 66.7 us at the two that it takes by itself, 62.4 at three),
// its gradient to those of three, two in f64 (8192 tokens of 10 heads of 256: 110
// us with the forward, 143 where each takes what it wants); the rotation alone is
// fastest at the two that it takes (118 registers: 56.6 us; 61.1 at three, 68.3 at
// four).
template <class T, int V, bool IL, int MODE, int G, int K, int UH>
__global__ void __launch_bounds__(kRotThreads, MODE == kRotate || K > 1 ? 1 : sizeof(T) == 4 ? 3 : MODE == kNormBackward ? 2 : 1)
rotary_kernel(const RotDev d) {
  const int which = (int64_t)blockIdx.x >= d.blocks0;
  const int64_t blk = which ? (int64_t)blockIdx.x - d.blocks0 : (int64_t)blockIdx.x;
  const int64_t nblk = which ? (int64_t)gridDim.x - d.blocks0 : d.blocks0;
  constexpr int kGroups = kRotThreads / G;
  const int lane = threadIdx.x % G, grp = threadIdx.x / G;
  const unsigned mask = G == 32 ? 0xffffffffu : (((1u << G) - 1u) << ((threadIdx.x & 31) / G * G));
  const HeadsDev X = d.x[which], Y = d.y[which], DY = d.dy[which];
  const T* xp = static_cast<const T*>(X.p);
  T* yp = static_cast<T*>(Y.p);
  const T* dp = static_cast<const T*>(DY.p);
  const T* gam = static_cast<const T*>(d.gamma[which]);
  const int H = d.H[which];

  Unit un[K];
  T ga[K][V], gb[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    un[k] = unit_of<V, IL>(d, lane + k * G);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ga[k][i] = MODE != kRotate && gam && un[k].v0 ? gam[(un[k].o0 + i) * d.gs[which]] : T(1);
      gb[k][i] = MODE != kRotate && gam && un[k].v1 ? gam[(un[k].o1 + i) * d.gs[which]] : T(1);
    }
  }
  // dgamma: f32 (element type) sums over the heads of an item, at most 8, then
  // f64 sums over the items in shared memory, one column per thread
  __shared__ double fold[MODE == kNormBackward ? K * 2 * V : 1][MODE == kNormBackward ? kRotThreads : 1];
  if constexpr (MODE == kNormBackward) {
#pragma unroll
    for (int i = 0; i < K * 2 * V; ++i) fold[i][threadIdx.x] = 0.0;
  }

  for (int64_t it = blk * kGroups + grp; it < d.items[which]; it += nblk * kGroups) {
    const uint32_t tok = fdiv((uint32_t)it, d.f_chunks[which]);
    const int h0 = (int)((uint32_t)it - tok * d.f_chunks[which].d) * d.hpc;
    const int h1 = h0 + d.hpc < H ? h0 + d.hpc : H;
    const int64_t b = fdiv(tok, d.f_T), t = tok - (uint32_t)b * d.f_T.d;
    const T* xt = xp + b * X.sb + t * X.st;
    T* yt = yp + b * Y.sb + t * Y.st;
    const T* dt = dp + b * DY.sb + t * DY.st;
    T a[UH][K][V], c[UH][K][V];
    T ea[MODE == kNormBackward ? UH : 1][K][V], ec[MODE == kNormBackward ? UH : 1][K][V];
    auto load_heads = [&](int h) {
#pragma unroll
      for (int u = 0; u < UH; ++u) {
        const bool on = h + u < h1;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          load_vec<T, V>(a[u][k], xt + (h + u) * X.sh, un[k].o0, X.sd, on && un[k].v0);
          load_vec<T, V>(c[u][k], xt + (h + u) * X.sh, un[k].o1, X.sd, on && un[k].v1);
          if constexpr (MODE == kNormBackward) {
            load_vec<T, V>(ea[u][k], dt + (h + u) * DY.sh, un[k].o0, DY.sd, on && un[k].v0);
            load_vec<T, V>(ec[u][k], dt + (h + u) * DY.sh, un[k].o1, DY.sd, on && un[k].v1);
          }
        }
      }
    };
    // on their way while the angles are evaluated (8192 tokens of 40 heads of 128:
    // rotation 60.4 -> 56.7 us, f64 norm 128.1 -> 124.0); the f32 norm lacks the
    // registers (62.2 -> 62.9)
    constexpr bool kEarly = MODE == kRotate || sizeof(T) == 8;
    if (kEarly) load_heads(h0);
    const int64_t pi = b * d.ps_b + t * d.ps_t;
    const double p = d.pos64 ? (double)static_cast<const int64_t*>(d.pos)[pi]
                             : (double)static_cast<const int32_t*>(d.pos)[pi];
    T cs[K][V], sn[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        cs[k][i] = T(1);
        sn[k][i] = T(0);
      }
      if (un[k].rot) {
        turn<V>(p, [&](int i) { return d.freq[((lane + k * G) * V + i) * d.fs]; }, d.magnitude, cs[k], sn[k]);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (d.inverse) sn[k][i] = -sn[k][i];
      }
    }
    T aa[MODE == kNormBackward ? K : 1][V], ab[MODE == kNormBackward ? K : 1][V];
    if constexpr (MODE == kNormBackward) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) aa[k][i] = ab[k][i] = T(0);
    }
    for (int h = h0; h < h1; h += UH) {
      if (!kEarly || h > h0) load_heads(h);
#pragma unroll
      for (int u = 0; u < UH; ++u) {
        if (h + u >= h1) break;
        if constexpr (MODE != kRotate) {
          T ss = T(0);
#pragma unroll
          for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) {
              ss = rfma(a[u][k][i], a[u][k][i], ss);
              ss = rfma(c[u][k][i], c[u][k][i], ss);
            }
          ss = group_sum<T, G>(ss, mask);
          const T r = inv_norm(ss, (T)d.D, (T)d.eps);
          if constexpr (MODE == kNormRotate) {
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
              for (int i = 0; i < V; ++i) {
                a[u][k][i] = a[u][k][i] * r * ga[k][i];
                c[u][k][i] = c[u][k][i] * r * gb[k][i];
              }
          } else {
            T dot = T(0);
#pragma unroll
            for (int k = 0; k < K; ++k) {
              if (un[k].rot) rotate<T, V, IL>(ea[u][k], ec[u][k], cs[k], sn[k]);
#pragma unroll
              for (int i = 0; i < V; ++i) {
                a[u][k][i] *= r;  // n
                c[u][k][i] *= r;
                aa[k][i] = rfma(ea[u][k][i], a[u][k][i], aa[k][i]);
                ab[k][i] = rfma(ec[u][k][i], c[u][k][i], ab[k][i]);
                ea[u][k][i] *= ga[k][i];  // dn
                ec[u][k][i] *= gb[k][i];
                dot = rfma(ea[u][k][i], a[u][k][i], dot);
                dot = rfma(ec[u][k][i], c[u][k][i], dot);
              }
            }
            dot = group_sum<T, G>(dot, mask) / (T)d.D;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
              for (int i = 0; i < V; ++i) {
                a[u][k][i] = r * rfma(-a[u][k][i], dot, ea[u][k][i]);
                c[u][k][i] = r * rfma(-c[u][k][i], dot, ec[u][k][i]);
              }
          }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if constexpr (MODE != kNormBackward)
            if (un[k].rot) rotate<T, V, IL>(a[u][k], c[u][k], cs[k], sn[k]);
          store_vec<T, V>(yt + (h + u) * Y.sh, un[k].o0, Y.sd, a[u][k], un[k].v0);
          store_vec<T, V>(yt + (h + u) * Y.sh, un[k].o1, Y.sd, c[u][k], un[k].v1);
        }
      }
    }
    if constexpr (MODE == kNormBackward) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          fold[k * 2 * V + i][threadIdx.x] += (double)aa[k][i];
          fold[k * 2 * V + V + i][threadIdx.x] += (double)ab[k][i];
        }
    }
  }

  if constexpr (MODE == kNormBackward) {
    pdl_launch_dependents();
    if (d.part[which] == nullptr) return;
    __syncthreads();
    // column i of unit u is spread over the threads of lane u of every group
    for (int x = threadIdx.x; x < K * 2 * V * G; x += kRotThreads) {
      const int i = x / G, u = x % G, k = i / (2 * V), e = i % (2 * V);
      const Unit n = unit_of<V, IL>(d, u + k * G);
      double s = 0.0;
      for (int g = 0; g < kGroups; ++g) s += fold[i][g * G + u];
      const int at = e < V ? n.o0 + e : n.o1 + e - V;
      if (e < V ? n.v0 : n.v1) d.part[which][blk * d.D + at] = s;
    }
  }
}

// dgamma[d] = the CTAs' partial sums added in a fixed order: 32 columns by 32
// row groups per CTA; blockIdx.y is the tensor.
struct GammaDev {
  const double* part[2];
  int64_t rows[2];
  void* out[2];
  int64_t st[2];
  int D;
};
template <class T>
__global__ void __launch_bounds__(1024) gamma_fold_kernel(const GammaDev d) {
  __shared__ double sm[32][33];
  pdl_wait();
  const int w = blockIdx.y, lane = threadIdx.x % 32, col = blockIdx.x * 32 + lane, g = threadIdx.x / 32;
  if (d.out[w] == nullptr) return;
  double s = 0.0;
  if (col < d.D) {
    for (int64_t r = g; r < d.rows[w]; r += 128) {
      double x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = r + 32 * i < d.rows[w] ? d.part[w][(r + 32 * i) * d.D + col] : 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) s += x[i];
    }
  }
  sm[g][lane] = s;
  __syncthreads();
  // warp g folds column g as a tree
  s = sm[lane][g];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int c = blockIdx.x * 32 + g;
  if (lane == 0 && c < d.D) static_cast<T*>(d.out[w])[c * d.st[w]] = (T)s;
}

template <class T>
__global__ void __launch_bounds__(256) gamma_zero_kernel(const GammaDev d) {
  const int w = blockIdx.y, col = blockIdx.x * 256 + threadIdx.x;
  if (d.out[w] && col < d.D) static_cast<T*>(d.out[w])[col * d.st[w]] = T(0);
}

// ---- host side -------------------------------------------------------------------

struct RotCall {
  const char* fn;
  int mode;
  bool inverse;
  const trs_view *q, *k;          // inputs (k may be null)
  trs_view *yq, *yk;              // outputs
  const trs_view *dq, *dk;        // output gradients (backward of the norm)
  const trs_view *gq, *gk;        // gamma (may be null)
  trs_view *dgq, *dgk;            // gamma gradients (may be null)
  double eps;
  const trs_view *pos, *freqs;
  int layout;
  double magnitude;
};

template <class T, int V, bool IL, int MODE, int G, int K, int UH>
Error launch_rot(RotDev& d, const RotCall& c, cudaStream_t stream) {
  constexpr int kGroups = kRotThreads / G;
  const int sms = current_device_info().sm_count;
  auto kern = rotary_kernel<T, V, IL, MODE, G, K, UH>;
  const int64_t resident = (int64_t)sms * resident_blocks_smem((const void*)kern, kRotThreads, 0);
  // heads per item: 8 that share an angle while the items still fill the GPU.
  // 8192 tokens of 40 heads of 128, 8, 4, 2, 1 heads: rotated 57, 59, 73 and 113
  // us, normed 62, 69, 96 and 149; 64 tokens of them normed: 8 heads 8.2 us, what
  // the rule takes there 4.5
  const int64_t tokens = d.items[0];  // set by the caller: batch * tokens
  int hpc = 8;
  while (hpc > 1 && tokens * ((d.H[0] + d.H[1] + hpc - 1) / hpc) < resident * kGroups) hpc /= 2;
  d.hpc = hpc;
  int64_t blocks[2];
  for (int w = 0; w < 2; ++w) {
    const int64_t chunks = (d.H[w] + hpc - 1) / hpc;
    d.f_chunks[w] = make_fastdiv(chunks ? (uint32_t)chunks : 1u);
    d.items[w] = tokens * chunks;
    if (d.items[w] >= (1ll << 31)) return make_error(TRS_ERR_SHAPE, std::string(c.fn) + ": 2^31 or more tokens");
    blocks[w] = (d.items[w] + kGroups - 1) / kGroups;
  }
  if (MODE == kNormBackward) {
    // one wave: each CTA keeps its dgamma sums to the end
    const int64_t all = blocks[0] + blocks[1];
    if (all > resident) {
      int64_t b1 = blocks[1] ? (blocks[1] * resident + all - 1) / all : 0;
      if (b1 >= resident) b1 = resident - 1;
      blocks[1] = blocks[1] ? (b1 < 1 ? 1 : b1) : 0;
      blocks[0] = resident - blocks[1];
    }
  }
  d.blocks0 = blocks[0];
  Scratch part;
  const bool want = c.dgq || c.dgk;
  if (MODE == kNormBackward && want) {
    Error e = part.alloc(sizeof(double) * (size_t)(blocks[0] + blocks[1]) * d.D, stream);
    if (!e.ok()) return e;
    d.part[0] = c.dgq ? part.as<double>() : nullptr;
    d.part[1] = c.dgk ? part.as<double>() + blocks[0] * d.D : nullptr;
  }
  kern<<<(unsigned)(blocks[0] + blocks[1]), kRotThreads, 0, stream>>>(d);
  Error e = check_launch(c.fn);
  if (!e.ok() || MODE != kNormBackward || !want) return e;
  GammaDev g;
  std::memset(&g, 0, sizeof(g));
  g.D = d.D;
  trs_view* outs[2] = {c.dgq, c.dgk};
  for (int w = 0; w < 2; ++w) {
    if (!outs[w]) continue;
    g.part[w] = d.part[w];
    g.rows[w] = blocks[w];
    g.out[w] = static_cast<T*>(outs[w]->data) + outs[w]->offset;
    g.st[w] = outs[w]->strides[0];
  }
  return launch_after(gamma_fold_kernel<T>, dim3((unsigned)((d.D + 31) / 32), 2), 1024, 0, stream,
                      "gamma gradient fold kernel", g);
}

// lanes per token and units per lane from the number of units
template <class T, int V, bool IL, int MODE>
Error pick_group(RotDev& d, const RotCall& c, cudaStream_t s) {
  constexpr int UH = MODE == kNormBackward ? 2 : 4;
  if constexpr (V > 1) {
    if (d.NU <= 4) return launch_rot<T, V, IL, MODE, 4, 1, UH>(d, c, s);
    if (d.NU <= 8) return launch_rot<T, V, IL, MODE, 8, 1, UH>(d, c, s);
    if (d.NU <= 16) return launch_rot<T, V, IL, MODE, 16, 1, UH>(d, c, s);
    if (d.NU <= 32) return launch_rot<T, V, IL, MODE, 32, 1, UH>(d, c, s);
    return launch_rot<T, V, IL, MODE, 32, 8 / V, 1>(d, c, s);  // a 512-element head: 64 units of 8, 128 of 4
  } else {
    if (d.NU <= 32) return launch_rot<T, V, IL, MODE, 32, 1, UH>(d, c, s);
    if (d.NU <= 128) return launch_rot<T, V, IL, MODE, 32, 4, 1>(d, c, s);
    return launch_rot<T, V, IL, MODE, 32, 8, 1>(d, c, s);
  }
}

template <class T, int MODE>
Error pick_layout(RotDev& d, const RotCall& c, bool vec, cudaStream_t s) {
  constexpr int VW = 16 / (int)sizeof(T);
  const bool il = c.layout == TRS_ROTARY_INTERLEAVED;
  const int V = vec ? VW : 1;
  d.NR = d.R / 2 / V;
  d.NU = d.NR + (d.D - d.R + 2 * V - 1) / (2 * V);
  if (vec) return il ? pick_group<T, VW, true, MODE>(d, c, s) : pick_group<T, VW, false, MODE>(d, c, s);
  return il ? pick_group<T, 1, true, MODE>(d, c, s) : pick_group<T, 1, false, MODE>(d, c, s);
}

template <class T>
Error pick_mode(RotDev& d, const RotCall& c, bool vec, cudaStream_t s) {
  switch (c.mode) {
    case kRotate: return pick_layout<T, kRotate>(d, c, vec, s);
    case kNormRotate: return pick_layout<T, kNormRotate>(d, c, vec, s);
    default: return pick_layout<T, kNormBackward>(d, c, vec, s);
  }
}

Error check_gamma(const char* fn, const trs_view* g, int64_t D, int dt, const char* what) {
  Error e = validate_view(g, what);
  if (!e.ok()) return e;
  if (g->dtype != dt) return make_error(TRS_ERR_DTYPE, std::string(fn) + ": " + what + " has another dtype");
  if (g->ndim != 1 || g->shape[0] != D)
    return make_error(TRS_ERR_SHAPE, std::string(fn) + ": " + what + " must hold the head size's elements");
  return Error{};
}

Error run_rotary(const RotCall& c, cudaStream_t stream) {
  const std::string fn = c.fn;
  if (!c.q || !c.yq || !c.pos || !c.freqs || (c.k == nullptr) != (c.yk == nullptr) ||
      (c.mode == kNormBackward && (!c.dq || (c.k == nullptr) != (c.dk == nullptr))))
    return make_error(TRS_ERR_ARG, fn + ": null view");
  if (c.layout != TRS_ROTARY_HALF && c.layout != TRS_ROTARY_INTERLEAVED)
    return make_error(TRS_ERR_ARG, fn + ": unknown layout");
  if (!c.k && (c.gk || c.dgk)) return make_error(TRS_ERR_ARG, fn + ": a key gamma without keys");
  const trs_view* ins[2] = {c.q, c.k};
  trs_view* outs[2] = {c.yq, c.yk};
  const trs_view* dys[2] = {c.dq, c.dk};
  const trs_view* gammas[2] = {c.gq, c.gk};
  trs_view* dgammas[2] = {c.dgq, c.dgk};
  const char* names[2][5] = {{"q", "q output", "q output gradient", "q gamma", "q gamma gradient"},
                             {"k", "k output", "k output gradient", "k gamma", "k gamma gradient"}};
  const int dt = c.q->dtype;
  Error e = validate_view(c.q, "q");
  if (!e.ok()) return e;
  if (!is_float(dt)) return make_error(TRS_ERR_DTYPE, fn + ": f32 or f64 tensors only");
  RotDev d;
  std::memset(static_cast<void*>(&d), 0, sizeof(d));
  const int nt = c.k ? 2 : 1;
  for (int w = 0; w < nt; ++w) {
    e = check_heads(c.fn, ins[w], dt, names[w][0]);
    if (e.ok()) e = check_heads(c.fn, outs[w], dt, names[w][1]);
    if (e.ok() && c.mode == kNormBackward) e = check_heads(c.fn, dys[w], dt, names[w][2]);
    if (e.ok() && gammas[w]) e = check_gamma(c.fn, gammas[w], c.q->shape[3], dt, names[w][3]);
    if (e.ok() && dgammas[w]) e = check_gamma(c.fn, dgammas[w], c.q->shape[3], dt, names[w][4]);
    if (!e.ok()) return e;
    if (!same_shape(ins[w], outs[w]) || (c.mode == kNormBackward && !same_shape(ins[w], dys[w])))
      return make_error(TRS_ERR_SHAPE, fn + ": " + names[w][1] + " must have the shape of " + names[w][0]);
    if (writes_collide(outs[w]) || (dgammas[w] && writes_collide(dgammas[w])))
      return make_error(TRS_ERR_ALIAS, fn + ": two elements of an output share a place");
  }
  const int64_t B = c.q->shape[0], T = c.q->shape[1], D = c.q->shape[3];
  if (c.k && (c.k->shape[0] != B || c.k->shape[1] != T || c.k->shape[3] != D))
    return make_error(TRS_ERR_SHAPE, fn + ": q and k must agree in batch, tokens and head size");
  // outputs against everything else: an output may be its own tensor's input
  // through the identical layout, nothing more
  const trs_view* reads[10];
  const trs_view* writes[4];
  int owner[10], wowner[4], nr = 0, nw = 0;
  for (int w = 0; w < nt; ++w) {
    reads[nr] = ins[w]; owner[nr++] = w;
    if (c.mode == kNormBackward) { reads[nr] = dys[w]; owner[nr++] = w; }
    if (gammas[w]) { reads[nr] = gammas[w]; owner[nr++] = -1; }
    writes[nw] = outs[w]; wowner[nw++] = w;
    if (dgammas[w]) { writes[nw] = dgammas[w]; wowner[nw++] = -2; }
  }
  reads[nr] = c.pos; owner[nr++] = -1;
  reads[nr] = c.freqs; owner[nr++] = -1;
  e = validate_view(c.pos, "positions");
  if (e.ok()) e = validate_view(c.freqs, "frequencies");
  if (!e.ok()) return e;
  for (int i = 0; i < nw; ++i) {
    for (int j = 0; j < nr; ++j) {
      if (wowner[i] == owner[j] && same_elements(writes[i], reads[j])) continue;
      if (heads_overlap(writes[i], reads[j])) return make_error(TRS_ERR_ALIAS, fn + ": an output overlaps an input");
    }
    for (int j = 0; j < i; ++j)
      if (heads_overlap(writes[i], writes[j])) return make_error(TRS_ERR_ALIAS, fn + ": two outputs overlap");
  }
  // positions [T] or [B, T] (a batch of 1 serves all), frequencies [R / 2]
  if (c.pos->dtype != TRS_I32 && c.pos->dtype != TRS_I64)
    return make_error(TRS_ERR_DTYPE, fn + ": positions must be i32 or i64");
  const int pn = c.pos->ndim;
  if ((pn != 1 && pn != 2) || c.pos->shape[pn - 1] != T || (pn == 2 && c.pos->shape[0] != B && c.pos->shape[0] != 1))
    return make_error(TRS_ERR_SHAPE, fn + ": positions must be [tokens] or [batch, tokens]");
  if (c.freqs->dtype != TRS_F64) return make_error(TRS_ERR_DTYPE, fn + ": frequencies must be f64");
  if (c.freqs->ndim != 1 || c.freqs->shape[0] < 1 || 2 * c.freqs->shape[0] > D)
    return make_error(TRS_ERR_SHAPE, fn + ": frequencies must hold 1 to half the head size's entries");
  if (D > kRotMaxHead) return make_error(TRS_ERR_SHAPE, fn + ": a head size above 512");
  const bool no_rows = B * T * c.q->shape[2] == 0, no_keys = !c.k || B * T * c.k->shape[2] == 0;
  if (no_rows && no_keys) {  // nothing to rotate; a gradient of no rows is zero
    if (!c.dgq && !c.dgk) return Error{};
    GammaDev g;
    std::memset(&g, 0, sizeof(g));
    g.D = (int)D;
    for (int w = 0; w < nt; ++w)
      if (dgammas[w]) {
        g.out[w] = static_cast<char*>(dgammas[w]->data) + dgammas[w]->offset * dtype_size(dt);
        g.st[w] = dgammas[w]->strides[0];
      }
    if (dt == TRS_F32) gamma_zero_kernel<float><<<dim3((unsigned)((D + 255) / 256), 2), 256, 0, stream>>>(g);
    else gamma_zero_kernel<double><<<dim3((unsigned)((D + 255) / 256), 2), 256, 0, stream>>>(g);
    return check_launch("gamma gradient zero kernel");
  }
  const int es = dtype_size(dt), VW = 16 / es;
  d.D = (int)D;
  d.R = (int)(2 * c.freqs->shape[0]);
  if (B * T >= (1ll << 31)) return make_error(TRS_ERR_SHAPE, fn + ": 2^31 or more tokens");
  const int64_t most = (1ll << 31) - 16;  // room for rounding up to whole chunks of heads
  if (c.q->shape[2] >= most || (c.k && (c.k->shape[2] >= most || c.q->shape[2] + c.k->shape[2] >= most)))
    return make_error(TRS_ERR_SHAPE, fn + ": 2^31 or more heads");
  d.f_T = make_fastdiv((uint32_t)T);
  d.inverse = c.inverse || c.mode == kNormBackward;
  d.magnitude = c.magnitude;
  d.eps = c.eps;
  d.pos64 = c.pos->dtype == TRS_I64;
  d.pos = static_cast<char*>(c.pos->data) + c.pos->offset * dtype_size(c.pos->dtype);
  d.ps_t = c.pos->strides[pn - 1];
  d.ps_b = pn == 2 && c.pos->shape[0] == B ? c.pos->strides[0] : 0;
  d.freq = static_cast<double*>(c.freqs->data) + c.freqs->offset;
  d.fs = c.freqs->strides[0];
  d.items[0] = B * T;
  // 16-byte accesses: unit element stride, every row on a 16-byte boundary,
  // and whole vectors on both sides of the pairs' and the rotation's border
  bool vec = d.R % (2 * VW) == 0 && D % VW == 0;
  auto aligned = [&](const trs_view* v) {
    if (((uintptr_t)v->data + (uintptr_t)(v->offset * es)) % 16) return false;
    if (v->strides[3] != 1 && v->shape[3] != 1) return false;
    for (int i = 0; i < 3; ++i)
      if (v->shape[i] > 1 && v->strides[i] % VW) return false;
    return true;
  };
  for (int w = 0; w < nt; ++w) {
    d.H[w] = (int)ins[w]->shape[2];
    d.x[w] = heads_dev(ins[w]);
    d.y[w] = heads_dev(outs[w]);
    vec = vec && aligned(ins[w]) && aligned(outs[w]);
    if (c.mode == kNormBackward) {
      d.dy[w] = heads_dev(dys[w]);
      vec = vec && aligned(dys[w]);
    }
    if (gammas[w]) {
      d.gamma[w] = static_cast<char*>(gammas[w]->data) + gammas[w]->offset * es;
      d.gs[w] = gammas[w]->strides[0];
    }
  }
  return dt == TRS_F32 ? pick_mode<float>(d, c, vec, stream) : pick_mode<double>(d, c, vec, stream);
}

// ---- frequencies -------------------------------------------------------------------

struct FreqDev {
  double* out;
  int64_t st;
  int n, kind;
  double base, factor, lo, hi, context;
};

// f_i = base^(-2i / rotary), then scaled for a context longer than the one
// the model was trained on.
__global__ void __launch_bounds__(128) frequency_kernel(const FreqDev d) {
  for (int i = blockIdx.x * 128 + threadIdx.x; i < d.n; i += gridDim.x * 128) {
    const double e = (double)i / (double)d.n;
    double f = pow(d.base, -e);
    const double turns = d.context * f / 6.283185307179586;  // of this pair over the trained context
    if (d.kind == TRS_SCALING_LINEAR) {
      f /= d.factor;
    } else if (d.kind == TRS_SCALING_BASE) {
      // the base grows so that the slowest pair turns `factor` times slower
      // and the fastest keeps its pace
      const double grow = d.n > 1 ? pow(d.factor, (double)d.n / (double)(d.n - 1)) : d.factor;
      f = pow(d.base * grow, -e);
    } else if (d.kind == TRS_SCALING_BANDS || d.kind == TRS_SCALING_RAMP) {
      // kept where the pair turns at least `hi` times over the trained
      // context, divided by factor below `lo` turns, and between them a mix
      // that runs with the turns (bands) or with the pair's index (ramp)
      double keep;
      if (d.kind == TRS_SCALING_BANDS) {
        keep = (turns - d.lo) / (d.hi - d.lo);
      } else {
        // the index at which a pair makes r turns: n log_base(context / (2 pi r))
        const double step = (double)d.n / log(d.base);
        const double first = fmax(floor(step * log(d.context / (d.hi * 6.283185307179586))), 0.0);
        double last = fmin(ceil(step * log(d.context / (d.lo * 6.283185307179586))), (double)(d.n * 2 - 1));
        if (last <= first) last = first + 0.001;
        keep = 1.0 - ((double)i - first) / (last - first);
      }
      keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
      f = f * keep + f / d.factor * (1.0 - keep);
    }
    d.out[i * d.st] = f;
  }
}

Error run_frequencies(double base, int scaling, double factor, double lo, double hi, double context,
                      const trs_view* out, cudaStream_t stream) {
  if (!out) return make_error(TRS_ERR_ARG, "rotary_frequencies: null view");
  Error e = validate_view(out, "frequencies");
  if (!e.ok()) return e;
  if (out->dtype != TRS_F64) return make_error(TRS_ERR_DTYPE, "rotary_frequencies: frequencies must be f64");
  if (out->ndim != 1 || out->shape[0] < 1)
    return make_error(TRS_ERR_SHAPE, "rotary_frequencies: frequencies must be [rotary / 2]");
  if (out->shape[0] > kRotMaxHead / 2) return make_error(TRS_ERR_SHAPE, "rotary_frequencies: a head size above 512");
  if (writes_collide(out))
    return make_error(TRS_ERR_ALIAS, "rotary_frequencies: two elements of the output share a place");
  if (!(base > 1.0) || !std::isfinite(base)) return make_error(TRS_ERR_ARG, "rotary_frequencies: the base must be above 1");
  if (scaling < TRS_SCALING_NONE || scaling > TRS_SCALING_RAMP)
    return make_error(TRS_ERR_ARG, "rotary_frequencies: unknown scaling");
  if (scaling != TRS_SCALING_NONE && (!(factor > 0.0) || !std::isfinite(factor)))
    return make_error(TRS_ERR_ARG, "rotary_frequencies: the factor must be above 0");
  if ((scaling == TRS_SCALING_BANDS || scaling == TRS_SCALING_RAMP) &&
      (!(lo > 0.0) || !(hi > lo) || !std::isfinite(hi) || !(context > 0.0) || !std::isfinite(context)))
    return make_error(TRS_ERR_ARG, "rotary_frequencies: needs 0 < low < high turns and a trained context");
  FreqDev d;
  d.out = static_cast<double*>(out->data) + out->offset;
  d.st = out->strides[0];
  d.n = (int)out->shape[0];
  d.kind = scaling;
  d.base = base;
  d.factor = factor;
  d.lo = lo;
  d.hi = hi;
  d.context = context;
  frequency_kernel<<<(unsigned)((d.n + 127) / 128), 128, 0, stream>>>(d);
  return check_launch("rotary frequency kernel");
}

trs_status finish(const Error& e) {
  if (!e.ok()) set_last_error(e.msg);
  return e.status;
}

cudaStream_t as_stream(trs_stream s) { return static_cast<cudaStream_t>(s); }

}  // namespace
}  // namespace trs

using namespace trs;

extern "C" {

trs_status trs_rotary_frequencies(double base, int32_t scaling, double factor, double low_turns, double high_turns,
                                  double trained_context, trs_view* freqs, trs_stream stream) {
  return finish(run_frequencies(base, scaling, factor, low_turns, high_turns, trained_context, freqs,
                                as_stream(stream)));
}

trs_status trs_rotary(const trs_view* q, const trs_view* k, const trs_view* positions, const trs_view* freqs,
                      int32_t layout, double magnitude, trs_view* q_out, trs_view* k_out, trs_stream stream) {
  RotCall c = {"rotary", kRotate, false, q, k, q_out, k_out, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
               0.0, positions, freqs, layout, magnitude};
  return finish(run_rotary(c, as_stream(stream)));
}

trs_status trs_rotary_backward(const trs_view* grad_q_out, const trs_view* grad_k_out, const trs_view* positions,
                               const trs_view* freqs, int32_t layout, double magnitude, trs_view* grad_q,
                               trs_view* grad_k, trs_stream stream) {
  RotCall c = {"rotary_backward", kRotate, true, grad_q_out, grad_k_out, grad_q, grad_k, nullptr, nullptr, nullptr,
               nullptr, nullptr, nullptr, 0.0, positions, freqs, layout, magnitude};
  return finish(run_rotary(c, as_stream(stream)));
}

trs_status trs_head_norm_rotary(const trs_view* q, const trs_view* k, const trs_view* q_gamma,
                                const trs_view* k_gamma, double eps, const trs_view* positions,
                                const trs_view* freqs, int32_t layout, double magnitude, trs_view* q_out,
                                trs_view* k_out, trs_stream stream) {
  RotCall c = {"head_norm_rotary", kNormRotate, false, q, k, q_out, k_out, nullptr, nullptr, q_gamma, k_gamma,
               nullptr, nullptr, eps, positions, freqs, layout, magnitude};
  return finish(run_rotary(c, as_stream(stream)));
}

trs_status trs_head_norm_rotary_backward(const trs_view* grad_q_out, const trs_view* grad_k_out, const trs_view* q,
                                         const trs_view* k, const trs_view* q_gamma, const trs_view* k_gamma,
                                         double eps, const trs_view* positions, const trs_view* freqs,
                                         int32_t layout, double magnitude, trs_view* grad_q, trs_view* grad_k,
                                         trs_view* grad_q_gamma, trs_view* grad_k_gamma, trs_stream stream) {
  RotCall c = {"head_norm_rotary_backward", kNormBackward, true, q, k, grad_q, grad_k, grad_q_out, grad_k_out,
               q_gamma, k_gamma, grad_q_gamma, grad_k_gamma, eps, positions, freqs, layout, magnitude};
  return finish(run_rotary(c, as_stream(stream)));
}

}  // extern "C"
