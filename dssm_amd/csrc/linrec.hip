// Gated linear recurrence over sequences, its gradient, and its single-token step.
//
//   u_t = sigmoid(gate_t),  h_t = u_t h_{t-1} + (1 - u_t) cand_t            (TF's GRUCell convention)
//
// per row and channel; a step at or past the row's length carries the state and emits zero
// (tf.nn.dynamic_rnn).  `reverse` walks the row from its last step to its first, as
// bidirectional_dynamic_rnn's backward cell does: time is mirrored by a negative stride, and the steps past
// the length, which the mirrored walk meets first, carry the state all the same.
//
// The gates do not look at the state, so steps compose: a stretch of time is the affine map
// h -> A h + B with A = product of u.  The gradient is the same recurrence from the other end,
//   g_t = dh_t + u_{t+1} g_{t+1},  dcand_t = (1 - u_t) g_t,  dgate_t = g_t (h_{t-1} - cand_t) u_t (1 - u_t),
// with gamma = u g as the value that crosses from step to step (gamma -> P gamma + Q over a stretch).
//
// Layout: a lane owns up to 4 bytes of neighbouring channels of one row (the last lane of an odd number of 16-bit
// channels shares one with its neighbour, and both store the same: 8 x 4365 x 629 bf16 59 + 89 us, 79 + 111 with
// a channel a lane), a wave a piece of kPiece steps whose loads are all in flight at once.  With few channels NW
// waves take NW consecutive pieces: each reduces its piece to (A, B), they meet in LDS once, and each replays its
// piece from registers behind its true state, so the inputs are read once.  With very few channels the time axis
// is also cut into segments of several workgroups: one launch reduces the segments, the next folds the earlier
// segments' (A, B) into its own start; there the inputs are read twice.
//
// The forward keeps the fp32 state in front of every piece (half a byte per element); the
// backward walks a piece forward from it in registers and so needs neither h nor a forward scan.  States,
// gates and sums are fp32 throughout.
//
// Measured: 6144 rows x 32 steps x 128 channels bf16, ragged, 29 us forward and 43 backward (3.9 and 4.3 TB/s of
// the bytes that ragged rows leave); 2 x 65537 x 512 bf16 68 + 74 us, 4 x 16411 x 256 fp32 ragged 32 + 31 forward
// and 29 + 54 backward (the replaying launches 5.0 to 5.5 TB/s, memory; the summing ones read at 4 TB/s).  A
// piece of 16 steps keeps twice the registers and half the waves (backward 51 us, 84 + 101 for the long rows).
// (One launch whose segments wait for each other's sums would read the inputs once; it is not taken: a wait between
// running workgroups for a third of the time of few, very long rows.)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include <type_traits>

#include "seq.h"

namespace dssm {
namespace seq {
namespace {

constexpr int kPiece = DSSM_RECUR_PIECE;
constexpr int kSegWaves = 8;  // the waves of a workgroup where time is cut into segments (cut_of)

// u = sigmoid(f) and v = 1 - u, neither a difference: e = exp(-|f|) never overflows, and whichever of u and v
// is small keeps its relative accuracy down to 2^-126 (|f| = 87.3), below which it is 0.  The hardware's 2^x is off
// by the rounding of its argument, |x| half units: for fp32 gates that rounding and log2 e's own are put back, for
// gates that were rounded to 16 bits (whose own half step moves e by |x| 2^-12 and more) they are not.
template <typename T>
__device__ __forceinline__ void gate_uv(float f, float& u, float& v) {
  const float kL = 1.44269502f, kLlo = 1.92596303e-8f;
  const float hi = -fabsf(f) * kL;
  float e = __builtin_amdgcn_exp2f(hi);
  if constexpr (sizeof(T) == 4) {
    const float x = -fabsf(f), lo = fmaf(x, kL, -hi) + x * kLlo;
    e = hi < -126.f ? 0.f : fmaf(e, lo * 0.693147182f, e);  // (-inf would give inf - inf; NaN stays)
  }
  const float r = __builtin_amdgcn_rcpf(1.f + e), q = e * r;
  u = f >= 0.f ? r : q;
  v = f >= 0.f ? q : r;
}

// A stretch's weight, the product of its u, is 0 only where one of them is: one that underflowed to 0 would make an
// infinite state, which step by step stays infinite, a NaN.  2^-149, the smallest float, takes its place, which is off
// by less than that.  `least`: the smallest of the factors.  All are at least 0 (or NaN, which stays), so they compare
// as their bits do.  The factors' minimum runs beside their product and joins it at the end, off the chain of
// products: 4 x 16411 x 256 fp32 145 us of kernels either way, 148 with the two joined at every factor.
__device__ __forceinline__ unsigned bits_min(unsigned least, float u) { return min(least, __float_as_uint(u)); }
__device__ __forceinline__ float weight_of(float p, unsigned least) {
  return __uint_as_float(max(__float_as_uint(p), min(least, 1u)));
}

struct RecurArgs {
  const void *gate, *cand, *dh;
  int64_t gr, gt, cr, ct, dr, dt;  // row and time strides in elements
  const int* lens;
  const float* h0;     // [R x H], or null: zeros
  const float* dlast;  // backward: [R x H] or null
  void *h, *dgate, *dcand;
  int64_t hr, ht, ogr, ogt, ocr, oct;
  float *last, *dh0;  // forward / backward
  float* states;      // [ceil(T / kPiece)][R x H]
  float* sums;        // [2][S][R x H]: the segments' A and B (P and Q)
  int64_t R;
  int T, H, upr;  // upr: lane units per row
  int reverse, S, L;  // segments and their steps (a multiple of NW * kPiece)
};

template <int V>
struct Unit {  // a lane's channels
  int64_t r, r0, ch;  // row, the wave's first row, first channel in [R x H]
  int c, lo, hi;  // column; active steps [lo, hi) in walking order
  bool in;
};
template <int V>
__device__ __forceinline__ Unit<V> unit_of(const RecurArgs& a, int64_t u) {
  Unit<V> t;
  t.in = u < a.R * a.upr;
  if (!t.in) u = a.R * a.upr - 1;
  t.r = u / a.upr;
  t.c = min((int)(u - t.r * a.upr) * V, a.H - V);
  t.ch = t.r * a.H + t.c;
  int len = a.T;
  if (a.lens) len = min(max(a.lens[t.r], 0), a.T);
  if (!t.in) len = 0;
  t.lo = a.reverse ? a.T - len : 0;
  t.hi = a.reverse ? a.T : len;
  const int64_t r0 = t.r;  // (rows do not fall from lane to lane: the first lane's is the wave's smallest)
  t.r0 = ((int64_t)__builtin_amdgcn_readfirstlane((int)(r0 >> 32)) << 32) |
         (unsigned)__builtin_amdgcn_readfirstlane((int)r0);
  return t;
}
// A tensor as a wave walks it: the address of walking step p is uniform + the lane's offset, which is a
// 32-bit one behind the wave's first row where the rows of a wave lie close enough (W false: any strides),
// so that sixteen loads in flight hold one offset register and not sixteen addresses.
template <typename T, bool W>
struct Walk {
  char* base;
  int64_t step;
  std::conditional_t<W, int64_t, unsigned> off;
  __device__ __forceinline__ Walk(const void* p, const RecurArgs& a, int64_t sr, int64_t st, int64_t r0, int64_t r, int c) {
    base = (char*)p + (r0 * sr + (a.reverse ? (int64_t)(a.T - 1) * st : 0)) * (int64_t)sizeof(T);
    step = (a.reverse ? -st : st) * (int64_t)sizeof(T);
    off = (decltype(off))(((r - r0) * sr + c) * (int64_t)sizeof(T));
  }
  __device__ __forceinline__ T* at(int p) const { return (T*)(base + p * step + off); }
};

// A piece's gates and candidates as they lie in memory.  A step that does not act is not read; where all of
// a wave's steps act, which most pieces are, nothing is compared.
template <typename T, int V, bool W>
struct Piece {
  Pack<T, V> a[kPiece], b[kPiece];
  bool full;
  __device__ __forceinline__ void ask(const Walk<T, W>& g, const Walk<T, W>& c, int q0, int lo, int hi) {
    full = __all(q0 >= lo && q0 + kPiece <= hi);
    if (full) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        a[i] = ldv<T, V>(g.at(q0 + i));
        b[i] = ldv<T, V>(c.at(q0 + i));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        const int p = q0 + i;
        if (p >= lo && p < hi) {
          a[i] = ldv<T, V>(g.at(p));
          b[i] = ldv<T, V>(c.at(p));
        }
      }
    }
  }
  // u and x = (1 - u) cand; steps that do not act are u = 1, x = 0
  __device__ __forceinline__ void take(int q0, int lo, int hi, float (&u)[kPiece][V], float (&x)[kPiece][V]) const {
#pragma unroll
    for (int i = 0; i < kPiece; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float vv;
        gate_uv<T>(ld1(a[i].v[k]), u[i][k], vv);
        x[i][k] = vv * ld1(b[i].v[k]);
      }
    if (!full) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        const bool on = q0 + i >= lo && q0 + i < hi;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          u[i][k] = on ? u[i][k] : 1.f;
          x[i][k] = on ? x[i][k] : 0.f;
        }
      }
    }
  }
};

// The value that enters a segment: `start` carried through the earlier segments' maps.  The waves fold a
// share of the segments each and join through LDS.  dir > 0: segments 0 .. s - 1; dir < 0: S - 1 .. s + 1.
template <int V, int NW>
__device__ __forceinline__ void enter_segment(const RecurArgs& a, const Unit<V>& t, int s, int dir, float (*lds)[64][2 * V],
                                              float (&carry)[V]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = dir > 0 ? s : a.S - 1 - s, per = (n + NW - 1) / NW, k0 = min(w * per, n), k1 = min(k0 + per, n);
  const int64_t C = a.R * a.H;
  float A[V], B[V];
  unsigned least[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    A[k] = 1.f;
    B[k] = 0.f;
    least[k] = ~0u;
  }
  if (t.in)
    for (int j = k0; j < k1; ++j) {
      const int seg = dir > 0 ? j : a.S - 1 - j;
      const Pack<float, V> pa = ldv<float, V>(a.sums + (int64_t)seg * C + t.ch);
      const Pack<float, V> pb = ldv<float, V>(a.sums + (int64_t)(a.S + seg) * C + t.ch);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        B[k] = fmaf(pa.v[k], B[k], pb.v[k]);
        A[k] *= pa.v[k];
        least[k] = bits_min(least[k], pa.v[k]);
      }
    }
#pragma unroll
  for (int k = 0; k < V; ++k) {
    lds[w][lane][k] = weight_of(A[k], least[k]);
    lds[w][lane][V + k] = B[k];
  }
  __syncthreads();
  for (int j = 0; j < NW; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) carry[k] = fmaf(lds[j][lane][k], carry[k], lds[j][lane][V + k]);
  __syncthreads();
}

// ---- forward -----------------------------------------------------------------------------------
// SUM: only the segment's (A, B).
template <typename T, int V, int NW, bool SUM, bool W>
__global__ __launch_bounds__(NW * 64) void k_recur_fwd(RecurArgs a) {
  __shared__ float lds[2][NW][64][2 * V];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the replay walks the segments from the last: what the summing launch read last is what caches hold
  const int s = SUM ? (int)blockIdx.y : a.S - 1 - (int)blockIdx.y;
  const Unit<V> t = unit_of<V>(a, (int64_t)blockIdx.x * 64 + lane);
  const Walk<T, W> g(a.gate, a, a.gr, a.gt, t.r0, t.r, t.c), c(a.cand, a, a.cr, a.ct, t.r0, t.r, t.c);
  const Walk<T, W> ho(a.h, a, a.hr, a.ht, t.r0, t.r, t.c);
  float carry[V], span[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    carry[k] = !SUM && a.h0 && t.in ? a.h0[t.ch + k] : 0.f;
    span[k] = 1.f;
  }
  Piece<T, V, W> in;
  in.ask(g, c, s * a.L + w * kPiece, t.lo, min(t.hi, min(s * a.L + a.L, a.T)));
  if constexpr (!SUM && NW == kSegWaves)
    if (a.S > 1) enter_segment<V, NW>(a, t, s, 1, lds[0], carry);
  const int end = min(s * a.L + a.L, a.T), hi = min(t.hi, end);
  int buf = 0;
  for (int p0 = s * a.L; p0 < end; p0 += NW * kPiece, buf ^= 1) {
    const int q0 = p0 + w * kPiece;
    float u[kPiece][V], x[kPiece][V], h[V];
    in.take(q0, t.lo, hi, u, x);
    const bool full = in.full;
    in.ask(g, c, q0 + NW * kPiece, t.lo, hi);  // the next round's, behind this one's arithmetic
    if constexpr (NW > 1) {
      float A[V], B[V];
      unsigned least[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A[k] = 1.f;
        B[k] = 0.f;
        least[k] = ~0u;
      }
#pragma unroll
      for (int i = 0; i < kPiece; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          B[k] = fmaf(u[i][k], B[k], x[i][k]);
          A[k] *= u[i][k];
          least[k] = bits_min(least[k], u[i][k]);
        }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        lds[buf][w][lane][k] = weight_of(A[k], least[k]);
        lds[buf][w][lane][V + k] = B[k];
      }
      // one barrier a round: the other half of lds is written next, and a wave that writes this half
      // again has passed the next round's barrier, behind every wave's reads here
      __syncthreads();
#pragma unroll
      for (int k = 0; k < V; ++k) least[k] = __float_as_uint(span[k]);
#pragma unroll
      for (int j = 0; j < NW; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if (j == w) h[k] = carry[k];
          carry[k] = fmaf(lds[buf][j][lane][k], carry[k], lds[buf][j][lane][V + k]);
          if constexpr (SUM) {
            span[k] *= lds[buf][j][lane][k];
            least[k] = bits_min(least[k], lds[buf][j][lane][k]);
          }
        }
#pragma unroll
      for (int k = 0; k < V; ++k) span[k] = weight_of(span[k], least[k]);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) h[k] = carry[k];
    }
    if constexpr (!SUM) {
      if (t.in && q0 < a.T) {
        if (a.states) {
          Pack<float, V> st;
#pragma unroll
          for (int k = 0; k < V; ++k) st.v[k] = h[k];
          stv<float, V>(a.states + (int64_t)(q0 / kPiece) * a.R * a.H + t.ch, st);
        }
#pragma unroll
        for (int i = 0; i < kPiece; ++i) {
          const int p = q0 + i;
          const bool on = full || (p >= t.lo && p < t.hi);
          Pack<T, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            h[k] = fmaf(u[i][k], h[k], x[i][k]);
            o.v[k] = st1<T>(on ? h[k] : 0.f);
          }
          if (p < a.T) stv<T, V>(ho.at(p), o);
        }
      }
      if constexpr (NW == 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) carry[k] = h[k];
      }
    }
  }
  if (!t.in || w) return;
  if constexpr (SUM) {
    const int64_t C = a.R * a.H;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      a.sums[(int64_t)s * C + t.ch + k] = span[k];
      a.sums[(int64_t)(a.S + s) * C + t.ch + k] = carry[k];
    }
  } else if (end == a.T) {
#pragma unroll
    for (int k = 0; k < V; ++k) a.last[t.ch + k] = carry[k];
  }
}

// ---- backward ----------------------------------------------------------------------------------
// SUM: only the segment's (P, Q).
template <typename T, int V, int NW, bool SUM, bool W>
__global__ __launch_bounds__(NW * 64) void k_recur_bwd(RecurArgs a) {
  __shared__ float lds[2][NW][64][2 * V];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int s = SUM ? a.S - 1 - (int)blockIdx.y : (int)blockIdx.y;
  const Unit<V> t = unit_of<V>(a, (int64_t)blockIdx.x * 64 + lane);
  const Walk<T, W> g(a.gate, a, a.gr, a.gt, t.r0, t.r, t.c), c(a.cand, a, a.cr, a.ct, t.r0, t.r, t.c);
  const Walk<T, W> d(a.dh, a, a.dr, a.dt, t.r0, t.r, t.c);
  const Walk<T, W> og(a.dgate, a, a.ogr, a.ogt, t.r0, t.r, t.c), oc(a.dcand, a, a.ocr, a.oct, t.r0, t.r, t.c);
  float carry[V], span[V];  // carry: gamma, the gradient that reaches the state behind the current stretch
#pragma unroll
  for (int k = 0; k < V; ++k) {
    carry[k] = !SUM && a.dlast && t.in ? a.dlast[t.ch + k] : 0.f;
    span[k] = 1.f;
  }
  const int begin = s * a.L, end = min(begin + a.L, a.T), lo = max(t.lo, begin);
  const int top = begin + (end - begin - 1) / (NW * kPiece) * (NW * kPiece);
  Pack<T, V> ra[kPiece], rb[kPiece], rd[kPiece];
  Pack<float, V> st;
  bool asked;  // all of the wave's steps act
  auto ask = [&](int q0) {
    asked = __all(q0 >= lo && q0 + kPiece <= t.hi);
    if (asked) {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        ra[i] = ldv<T, V>(g.at(q0 + i));
        if constexpr (!SUM) rb[i] = ldv<T, V>(c.at(q0 + i));
        if (a.dh) rd[i] = ldv<T, V>(d.at(q0 + i));
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPiece; ++i) {
        const int p = q0 + i;
        if (p >= lo && p < t.hi) {
          ra[i] = ldv<T, V>(g.at(p));
          if constexpr (!SUM) rb[i] = ldv<T, V>(c.at(p));
          if (a.dh) rd[i] = ldv<T, V>(d.at(p));
        }
      }
    }
    if constexpr (!SUM)
      if (t.in && q0 >= begin && q0 < a.T) st = ldv<float, V>(a.states + (int64_t)(q0 / kPiece) * a.R * a.H + t.ch);
  };
  ask(top + w * kPiece);
  if constexpr (!SUM && NW == kSegWaves)
    if (a.S > 1) enter_segment<V, NW>(a, t, s, -1, lds[0], carry);
  int buf = 0;
  for (int p0 = top; p0 >= begin; p0 -= NW * kPiece, buf ^= 1) {
    const int q0 = p0 + w * kPiece;
    float hp[V];
#pragma unroll
    for (int k = 0; k < V; ++k) hp[k] = st.v[k];
    float u[kPiece][V], e[kPiece][V], dgf[kPiece][V], vv[kPiece][V];  // e: dh; dgf: (h_{t-1} - c) u v
    const bool full = asked;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
      const bool on = full || (q0 + i >= t.lo && q0 + i < t.hi);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float uu, v1;
        gate_uv<T>(ld1(ra[i].v[k]), uu, v1);
        u[i][k] = on ? uu : 1.f;
        e[i][k] = on && a.dh ? ld1(rd[i].v[k]) : 0.f;
        if constexpr (!SUM) {
          const float cc = ld1(rb[i].v[k]);
          dgf[i][k] = on ? (hp[k] - cc) * (uu * v1) : 0.f;
          vv[i][k] = on ? v1 : 0.f;
          hp[k] = on ? fmaf(uu, hp[k], v1 * cc) : hp[k];
        }
      }
    }
    ask(q0 - NW * kPiece);  // the next round's, behind this one's arithmetic
    float gam[V];
    if constexpr (NW > 1) {
      float P[V], Q[V];
      unsigned least[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        P[k] = 1.f;
        Q[k] = 0.f;
        least[k] = ~0u;
      }
#pragma unroll
      for (int i = kPiece - 1; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          Q[k] = u[i][k] * (e[i][k] + Q[k]);
          P[k] *= u[i][k];
          least[k] = bits_min(least[k], u[i][k]);
        }
      // an active step's dh joins g in front of its u; a step that does not act has u = 1 and dh = 0
#pragma unroll
      for (int k = 0; k < V; ++k) {
        lds[buf][w][lane][k] = weight_of(P[k], least[k]);
        lds[buf][w][lane][V + k] = Q[k];
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < V; ++k) least[k] = __float_as_uint(span[k]);
#pragma unroll
      for (int j = NW - 1; j >= 0; --j)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          if (j == w) gam[k] = carry[k];
          carry[k] = fmaf(lds[buf][j][lane][k], carry[k], lds[buf][j][lane][V + k]);
          if constexpr (SUM) {
            span[k] *= lds[buf][j][lane][k];
            least[k] = bits_min(least[k], lds[buf][j][lane][k]);
          }
        }
#pragma unroll
      for (int k = 0; k < V; ++k) span[k] = weight_of(span[k], least[k]);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) gam[k] = carry[k];
    }
    if constexpr (!SUM) {
      if (t.in && q0 < a.T) {
#pragma unroll
        for (int i = kPiece - 1; i >= 0; --i) {
          const int p = q0 + i;
          Pack<T, V> pg, pc;
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float gg = e[i][k] + gam[k];
            // a step that does not act passes gamma on as it is; its own gradients are zero whatever gamma is
            const bool on = full || (p >= t.lo && p < t.hi);
            pg.v[k] = st1<T>(on ? gg * dgf[i][k] : 0.f);
            pc.v[k] = st1<T>(on ? gg * vv[i][k] : 0.f);
            gam[k] = u[i][k] * gg;
          }
          if (p < a.T) {
            stv<T, V>(og.at(p), pg);
            stv<T, V>(oc.at(p), pc);
          }
        }
      }
      if constexpr (NW == 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) carry[k] = gam[k];
      }
    }
  }
  if (!t.in || w) return;
  if constexpr (SUM) {
    const int64_t C = a.R * a.H;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      a.sums[(int64_t)s * C + t.ch + k] = span[k];
      a.sums[(int64_t)(a.S + s) * C + t.ch + k] = carry[k];
    }
  } else if (begin == 0 && a.dh0) {
#pragma unroll
    for (int k = 0; k < V; ++k) a.dh0[t.ch + k] = carry[k];
  }
}

// ---- one token ---------------------------------------------------------------------------------
template <typename T, int V>
__global__ __launch_bounds__(256) void k_recur_step(const T* __restrict__ gate, int64_t gr, const T* __restrict__ cand,
                                                    int64_t cr, float* __restrict__ state, int64_t sr, T* __restrict__ h,
                                                    int64_t hr, int64_t R, int H, int upr) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= R * upr) return;
  const int64_t r = u / upr;
  const int c = (int)(u - r * upr) * V;
  const Pack<T, V> a = ldv<T, V>(gate + r * gr + c), b = ldv<T, V>(cand + r * cr + c);
  Pack<float, V> s = ldv<float, V>(state + r * sr + c);
  Pack<T, V> o;
#pragma unroll
  for (int k = 0; k < V; ++k) {
    float uu, vv;
    gate_uv<T>(ld1(a.v[k]), uu, vv);
    s.v[k] = fmaf(uu, s.v[k], vv * ld1(b.v[k]));
    o.v[k] = st1<T>(s.v[k]);
  }
  stv<float, V>(state + r * sr + c, s);
  stv<T, V>(h + r * hr + c, o);
}

// How the work is cut.  16-bit channels go two a lane (64 x 100 x 512 bf16 16.3 and 22.3 us, 18.3 and 24.1 with one;
// 64 x 256 x 8192 268 and 419, 297 and 466), but one where the work is small and a lane's own time counts (8 x 128 x
// 133 bf16 7.0 and 9.5 us, 8.4 and 11.6 with two; 16 x 256 x 512 11.2 and 14.6, 12.7 and 17.0).
// `waves`: waves of 64 lanes that the channels alone give.  From 1024 on (one for each SIMD) a wave walks its row
// alone; below it, four or eight share the time of a workgroup's channels, and where even that leaves fewer than 2048
// waves, time is cut into segments until there are 4096 (2 x 65537 x 512: 140 us; 181 with 2048, 154 with 8192), of
// two rounds of pieces at least.  Up to four rounds stay one launch, whose rounds cost less than a second launch's
// start (8 x 128 bf16, two channels a lane: 133 steps 8.4 and 11.6 us, 11.8 and 15.4 cut; 256 steps 10.4 and 16.4,
// 12.0 and 15.6 cut; 512 steps 18.4 and 29.7, 12.1 and 15.7 cut).
struct Cut {
  int V, NW, S, L;
};
Cut cut_of(int64_t R, int T, int H, int dtype) {
  Cut c{};
  const bool small = R * H < 64 * 1024 && (double)R * H * T < 3e6;
  c.V = dtype == DSSM_F32 || H < 2 || small ? 1 : 2;
  const int64_t waves = (R * ((H + c.V - 1) / c.V) + 63) / 64;
  const int pieces = (T + kPiece - 1) / kPiece;
  c.NW = 1;
  c.S = 1;
  if (waves < 1024 && pieces > 1) {
    c.NW = pieces >= 5 ? kSegWaves : 4;
    const int64_t want = 4096 / (waves * c.NW);
    if (c.NW == kSegWaves && want >= 2 && pieces > 4 * c.NW) c.S = (int)std::min<int64_t>(want, (pieces + 2 * c.NW - 1) / (2 * c.NW));
  }
  const int round = c.NW * kPiece, per = (T + c.S - 1) / c.S;
  c.L = (per + round - 1) / round * round;
  c.S = (T + c.L - 1) / c.L;
  return c;
}

bool recur_dims_ok(int64_t R, int T, int H) {
  return R >= 0 && T > 0 && H > 0 && T <= (1 << 28) && H <= (1 << 20) && R <= ((int64_t)1 << 31) &&
         R * H <= ((int64_t)1 << 31);  // (a lane a state: a launch has fewer than 2^32 threads)
}

template <typename T, int V, bool FWD, bool W>
void launch(const RecurArgs& a, const Cut& c, hipStream_t s) {
  const dim3 grid((unsigned)((a.R * a.upr + 63) / 64), (unsigned)c.S);
  auto go = [&](auto nw) {
    constexpr int NW = decltype(nw)::value;
    if constexpr (FWD) {
      if constexpr (NW == kSegWaves)
        if (c.S > 1) hipLaunchKernelGGL((k_recur_fwd<T, V, NW, true, W>), grid, dim3(NW * 64), 0, s, a);
      hipLaunchKernelGGL((k_recur_fwd<T, V, NW, false, W>), grid, dim3(NW * 64), 0, s, a);
    } else {
      if constexpr (NW == kSegWaves)
        if (c.S > 1) hipLaunchKernelGGL((k_recur_bwd<T, V, NW, true, W>), grid, dim3(NW * 64), 0, s, a);
      hipLaunchKernelGGL((k_recur_bwd<T, V, NW, false, W>), grid, dim3(NW * 64), 0, s, a);
    }
  };
  if (c.NW == 1) go(std::integral_constant<int, 1>{});
  else if (c.NW == 4) go(std::integral_constant<int, 4>{});
  else go(std::integral_constant<int, 8>{});
}
template <bool FWD>
int run(RecurArgs& a, int dtype, void* stream) {
  const Cut c = cut_of(a.R, a.T, a.H, dtype);
  a.upr = (a.H + c.V - 1) / c.V;
  a.S = c.S;
  a.L = c.L;
  // a wave's 64 units lie in at most 64 / upr + 2 rows: do all their offsets fit 32 bits?
  int64_t far = 0;
  for (int64_t sr : {a.gr, a.cr, a.hr, a.dr, a.ogr, a.ocr}) far = std::max(far, sr < 0 ? INT64_MAX / 256 : sr);
  const bool wide = (double)far * (64 / a.upr + 2) + a.H >= 1e9;
  by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    auto go = [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      if (wide) launch<T, V, FWD, true>(a, c, (hipStream_t)stream);
      else launch<T, V, FWD, false>(a, c, (hipStream_t)stream);
    };
    if constexpr (sizeof(T) == 4) {
      go(std::integral_constant<int, 1>{});
    } else {
      if (c.V == 2) go(std::integral_constant<int, 2>{});
      else go(std::integral_constant<int, 1>{});
    }
  });
  return seq_status(hipGetLastError());
}

}  // namespace
}  // namespace seq
}  // namespace dssm

using namespace dssm::seq;

extern "C" size_t dssm_linear_recurrence_ws_bytes(int64_t R, int T, int H, int dtype) {
  if (!recur_dims_ok(R, T, H) || !seq_dtype(dtype) || R == 0) return 0;
  const Cut c = cut_of(R, T, H, dtype);
  return c.S > 1 ? (size_t)2 * c.S * R * H * sizeof(float) : 0;
}

extern "C" int dssm_linear_recurrence(const void* gate, int64_t gr, int64_t gt, const void* cand, int64_t cr, int64_t ct,
                                      int dtype, const int32_t* lens, const float* h0, int64_t R, int T, int H,
                                      int reverse, void* h, int64_t hr, int64_t ht, float* last, float* states, void* ws,
                                      size_t ws_bytes, void* stream) {
  if (!seq_dtype(dtype) || !recur_dims_ok(R, T, H) || (R > 0 && (!gate || !cand || !h || !last)))
    return dssm::report_error(DSSM_E_INVALID, "linear_recurrence: bad argument");
  if (R == 0) return DSSM_OK;
  const size_t need = dssm_linear_recurrence_ws_bytes(R, T, H, dtype);
  if (need && (!ws || ws_bytes < need))
    return dssm::report_error(DSSM_E_INVALID, "linear_recurrence: workspace too small (dssm_linear_recurrence_ws_bytes)");
  RecurArgs a{};
  a.gate = gate;
  a.cand = cand;
  a.gr = gr;
  a.gt = gt;
  a.cr = cr;
  a.ct = ct;
  a.lens = lens;
  a.h0 = h0;
  a.h = h;
  a.hr = hr;
  a.ht = ht;
  a.last = last;
  a.states = states;
  a.sums = (float*)ws;
  a.R = R;
  a.T = T;
  a.H = H;
  a.reverse = reverse != 0;
  return run<true>(a, dtype, stream);
}

extern "C" int dssm_linear_recurrence_bwd(const void* gate, int64_t gr, int64_t gt, const void* cand, int64_t cr,
                                          int64_t ct, int dtype, const int32_t* lens, const float* states, const void* dh,
                                          int64_t dr, int64_t dt, const float* dlast, int64_t R, int T, int H, int reverse,
                                          void* dgate, int64_t ogr, int64_t ogt, void* dcand, int64_t ocr, int64_t oct,
                                          float* dh0, void* ws, size_t ws_bytes, void* stream) {
  if (!seq_dtype(dtype) || !recur_dims_ok(R, T, H) || (R > 0 && (!gate || !cand || !states || !dgate || !dcand)))
    return dssm::report_error(DSSM_E_INVALID, "linear_recurrence_bwd: bad argument");
  if (R == 0) return DSSM_OK;
  const size_t need = dssm_linear_recurrence_ws_bytes(R, T, H, dtype);
  if (need && (!ws || ws_bytes < need))
    return dssm::report_error(DSSM_E_INVALID, "linear_recurrence_bwd: workspace too small (dssm_linear_recurrence_ws_bytes)");
  RecurArgs a{};
  a.gate = gate;
  a.cand = cand;
  a.dh = dh;
  a.gr = gr;
  a.gt = gt;
  a.cr = cr;
  a.ct = ct;
  a.dr = dr;
  a.dt = dt;
  a.lens = lens;
  a.dlast = dlast;
  a.states = const_cast<float*>(states);
  a.dgate = dgate;
  a.dcand = dcand;
  a.ogr = ogr;
  a.ogt = ogt;
  a.ocr = ocr;
  a.oct = oct;
  a.dh0 = dh0;
  a.sums = (float*)ws;
  a.R = R;
  a.T = T;
  a.H = H;
  a.reverse = reverse != 0;
  return run<false>(a, dtype, stream);
}

extern "C" int dssm_linear_recurrence_step(const void* gate, int64_t gr, const void* cand, int64_t cr, int dtype,
                                           float* state, int64_t sr, void* h, int64_t hr, int64_t R, int H, void* stream) {
  if (!seq_dtype(dtype) || !recur_dims_ok(R, 1, H) || (R > 0 && (!gate || !cand || !state || !h)))
    return dssm::report_error(DSSM_E_INVALID, "linear_recurrence_step: bad argument");
  if (R > 1 && (std::abs(sr) < H || std::abs(hr) < H))
    return dssm::report_error(DSSM_E_INVALID, "linear_recurrence_step: rows of state or h overlap");
  if (R == 0) return DSSM_OK;
  by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    auto go = [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const int64_t units = R * (H / V);
      hipLaunchKernelGGL((k_recur_step<T, V>), dim3((unsigned)((units + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                         (const T*)gate, gr, (const T*)cand, cr, state, sr, (T*)h, hr, R, H, H / V);
    };
    if (H % 4 == 0) go(std::integral_constant<int, 4>{});
    else go(std::integral_constant<int, 1>{});
  });
  return seq_status(hipGetLastError());
}
