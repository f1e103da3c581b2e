// Root-mean-square norm with the residual's addition, its output in the input's type or in the 8-bit block
// form, its gradient; and the 8-bit block form of plain rows and back.
//
//   s = round(x + residual),  rstd = 1 / sqrt(mean s^2 + eps),  y = s rstd w
//   n = s rstd:  dx = rstd (w dy - n mean(w dy n)) + ds,   dw = sum over rows of dy n
//
// s is rounded to its storage type before the norm, so that the backward, which reads the stored s, is
// the gradient of exactly this forward.  Sums are fp32, a row's squares 64 bits.
//
// Every kernel here is one pass over its rows, bound by memory.  A row stays in registers: NT threads (a
// quarter wave to a workgroup of 16 waves) hold 8 neighbouring columns each, K times over; 16 lanes hold a
// block of 128 columns, so a block's scale is four DPP steps away.  A workgroup stays for many rows, its weights in
// registers, with the next row's loads behind the current one's arithmetic.
//
// Measured: 196608 x 256 bf16 with a residual 68 us forward, 82 + 5 backward (403 MB each way: 5.9 and 4.6 TB/s, the
// forward's inputs in part still cached; one workgroup for every four rows took 117 and 119); 24571 x 1024 to the
// 8-bit form 34 us (5.1 TB/s), its values back in bf16 13 us (5.8 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "seq.h"

namespace dssm {
namespace seq {
namespace {

constexpr int kMaxCols = 16384;      // 1024 threads x 8 columns x 2: a row of the norm, a stretch of the 8-bit form's
constexpr int kMaxCols8 = 1 << 22;   // a row of the 8-bit form, as the product takes it

// the sum of v over the NT threads that share a row (every thread gets it); s: one value a wave
__device__ __forceinline__ double dpp_add(double v, int stage) {
  const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
  const int lo = (int)(unsigned)u, hi = (int)(u >> 32);
  int a, b;
  if (stage == 0) {
    a = __builtin_amdgcn_update_dpp(0, lo, 0xB1, 0xF, 0xF, false);
    b = __builtin_amdgcn_update_dpp(0, hi, 0xB1, 0xF, 0xF, false);
  } else if (stage == 1) {
    a = __builtin_amdgcn_update_dpp(0, lo, 0x4E, 0xF, 0xF, false);
    b = __builtin_amdgcn_update_dpp(0, hi, 0x4E, 0xF, 0xF, false);
  } else if (stage == 2) {
    a = __builtin_amdgcn_update_dpp(0, lo, 0x141, 0xF, 0xF, false);
    b = __builtin_amdgcn_update_dpp(0, hi, 0x141, 0xF, 0xF, false);
  } else {
    a = __builtin_amdgcn_update_dpp(0, lo, 0x140, 0xF, 0xF, false);
    b = __builtin_amdgcn_update_dpp(0, hi, 0x140, 0xF, 0xF, false);
  }
  return v + __builtin_bit_cast(double, (unsigned long long)(unsigned)a | ((unsigned long long)(unsigned)b << 32));
}
__device__ __forceinline__ float dpp_add(float v, int stage) {
  return stage == 0 ? wave_allsum_step<0>(v) : stage == 1 ? wave_allsum_step<1>(v) : stage == 2 ? wave_allsum_step<2>(v)
                                                                                              : wave_allsum_step<3>(v);
}
template <int NT, typename F>
__device__ __forceinline__ F row_sum(F v, F* s) {
#pragma unroll
  for (int k = 0; k < 4; ++k) v = dpp_add(v, k);
  if constexpr (NT >= 32) v = sum_xor16(v);
  if constexpr (NT >= 64) v = sum_xor32(v);
  if constexpr (NT > 64) {
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) s[w] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) v += s[i];
    __syncthreads();
  }
  return v;
}

struct NormArgs {
  const void *x, *res, *dy, *ds, *s_in;
  int64_t ldx, ldres, lddy, ldds, lds;
  const float *w, *rstd_in;
  void *y, *s, *dx;
  int64_t ldy, lddx;
  float* rstd;
  unsigned char *q, *scale;  // 8-bit form: q [rows x Kp], scale [rows x Kp / 128]
  float* part;               // backward: [blocks x cols]
  int64_t rows;
  int cols, kp;
  float eps;
};

// v becomes y = v up w (rstd + rest) in its first n columns, zeros behind them; up is a power of two.  E4M3: y is going
// to be rounded to e4m3.
template <bool E4M3>
__device__ __forceinline__ void scale8(float (&v)[8], const float (&w)[8], float up, float rstd, float rest, int n) {
  float y[8];
  unsigned tie = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // with the product's rounding error and rstd's rest put back: rounded once
    const float x = v[i] * up, p = x * w[i], e = fmaf(x, w[i], -p);
    y[i] = i < n ? fmaf(p, rstd, fmaf(p, rest, e * rstd)) : 0.f;
    tie |= (__float_as_uint(y[i]) & 0x7ffffu) == 0u;
  }
  if (E4M3 && tie) {
    // y that lies half way between two e4m3 values (these have their last 19 bits clear; so have zeros) may have got
    // there by its own rounding: it moves to the side that the exact value is on
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = v[i] * up, p = x * w[i], e = fmaf(x, w[i], -p);
      const float d = fmaf(p, rstd, -y[i]) + fmaf(p, rest, e * rstd);
      const unsigned u = __float_as_uint(y[i]);
      if (i < n && (u & 0x7ffffu) == 0u && (u << 1) != 0u && (u << 1) < 0xff000000u && d != 0.f)
        y[i] = __uint_as_float((d > 0.f) == (y[i] > 0.f) ? u + 1u : u - 1u);
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = y[i];
}

// MODE 0: y in T; 1: y in the 8-bit form; 2: x itself in the 8-bit form (no norm).
// A workgroup walks rows blockIdx.x * kRows + i * gridDim.x * kRows with the weights in registers and the next
// rows' loads in flight behind the current ones' arithmetic.
// MODE 2, whose blocks of 128 do not know of each other, takes rows of any width: blockIdx.y is a stretch of kMaxCols
// columns (bf16: 24571 x 1024 15 us, 5.1 TB/s; 4096 x 16384 32, 6.2; 4096 x 32768 80, 5.1; 7 x 4194304 17, 5.3).
template <typename T, int NT, int K, int MODE, bool R>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_norm(NormArgs a) {
  constexpr int kRows = NT < 256 ? 256 / NT : 1;
  constexpr bool kBranch = MODE == 1 && sizeof(T) == 2;
  __shared__ double red[16];
  const int l = threadIdx.x % NT;
  const int64_t step = (int64_t)gridDim.x * kRows;
  const bool whole = a.cols >= 8;
  const int64_t ldq = a.kp;
  bool heavy = false;  // one of this thread's weights is 2^64 or more
  if constexpr (MODE == 2 && NT * K * 8 == kMaxCols) {
    const int c0 = blockIdx.y * kMaxCols;
    a.x = (const T*)a.x + c0;
    a.q += c0;
    a.scale += c0 / kBlk;
    a.cols -= c0;
    a.kp = min(a.kp - c0, kMaxCols);
  }
  float w[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * NT + l) * 8, nv = a.cols - c;
    if (MODE != 2 && nv > 0) {
      ld_row<float, 8>(a.w + c, nv, w[k]);
#pragma unroll
      for (int i = 0; i < 8; ++i) heavy |= fabsf(w[k][i]) >= 0x1p64f;
    }
  }
  Ask<T, R> x[K], b[K];
  auto ask = [&](int64_t r) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + l) * 8, nv = r < a.rows ? a.cols - c : 0;
      x[k].ask((const T*)a.x + r * a.ldx + c, nv, whole);
      if (MODE != 2 && a.res) b[k].ask((const T*)a.res + r * a.ldres + c, nv, whole);
    }
  };
  int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / NT;
  ask(r);
  // (the loop's condition is the workgroup's, not the row slot's: its barriers need every thread)
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += step, r += step) {
    const bool in = r < a.rows;
    float v[K][8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + l) * 8, nv = in ? a.cols - c : 0;
      x[k].take((const T*)a.x + r * a.ldx + c, nv, whole, v[k]);
      if (MODE != 2 && a.res) {
        float t[8];
        b[k].take((const T*)a.res + r * a.ldres + c, nv, whole, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] = ld1(st1<T>(v[k][i] + t[i]));
      }
    }
    ask(r + step);
    if constexpr (MODE != 2) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[k][i], v[k][i], sum);
      }
      // A thread's squares in fp32, the row's in 64 bits: what a row's values share costs them no accuracy.  Where fp32
      // does not hold the squares (values above 2^63, or below 2^-50 with an eps as small) they are added up once more.
      double total = row_sum<NT, double>((double)sum, red);
      const bool again = total == __builtin_inf() || (a.eps < 0x1p-100f && total < 0x1p-90);
      if (__any(again)) {  // (a row that a workgroup shares has all its waves here)
        double exact = 0.0;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) exact = fma((double)v[k][i], (double)v[k][i], exact);
        exact = row_sum<NT, double>(exact, red);
        if (again) total = exact;
      }
      const double root = 1.0 / sqrt(total / (double)a.cols + (double)a.eps);
      // v w may be past what fp32 holds where y is not, and rstd below its normal range: a row's size is taken away first,
      // by a power of two, 1 at most (1 for a row with infinities, whose root is 0, or NaN).  For 16-bit rows in the
      // 8-bit form, which wait for their arithmetic, that is a branch of its own, for rows with a mean square of 2^60 and
      // more, or of 1 with a weight of 2^64 and more (196608 x 256 bf16 75 us, 90 without it; 24571 x 1024 31.3 and 36;
      // fp32 rows, whose registers it takes, 4096 x 8192 90 and 86).
      int exponent = (int)(__builtin_bit_cast(unsigned long long, root) >> 52 & 0x7ff) - 1023;
      if (exponent < -200 || exponent >= (kBranch && !heavy ? -30 : 0)) exponent = 0;
      const double mant = __builtin_ldexp(root, -exponent);
      const float rstd = (float)mant, rest = (float)(mant - (double)rstd), up = __builtin_ldexpf(1.f, exponent);
      if (in && l == 0 && a.rstd) a.rstd[r] = (float)root;
      // (s may be x or residual: it is stored behind the row sum, when no thread reads them any more)
      if constexpr (kBranch) {
        auto row = [&](float up) {
#pragma unroll
          for (int k = 0; k < K; ++k) {
            const int c = (k * NT + l) * 8, nv = in ? a.cols - c : 0;
            if (a.s && nv > 0) st_row<T, 8, R>((T*)a.s + r * a.lds + c, nv, v[k]);
            scale8<true>(v[k], w[k], up, rstd, rest, nv);
          }
        };
        if (__any(exponent != 0)) row(up);
        else row(1.f);
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (k * NT + l) * 8, nv = in ? a.cols - c : 0;
          if (a.s && nv > 0) st_row<T, 8, R>((T*)a.s + r * a.lds + c, nv, v[k]);
          scale8<MODE == 1>(v[k], w[k], up, rstd, rest, nv);
          if (MODE == 0 && nv > 0) st_row<T, 8, R>((T*)a.y + r * a.ldy + c, nv, v[k]);
        }
      }
    }
    if constexpr (MODE != 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * NT + l) * 8;
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[k][i]));
        const unsigned e = blk_exp(max16(m));
        if (in && c < a.kp) {
          *reinterpret_cast<uint2*>(a.q + r * ldq + c) = to_e4m3x8(v[k], exp_inv(e));
          if ((l & 15) == 0) a.scale[r * (ldq / kBlk) + c / kBlk] = (unsigned char)e;
        }
      }
    }
  }
}

// Backward.  A workgroup walks rows blockIdx.x * kRows + i * gridDim.x * kRows and keeps its share of dw in
// registers; its rows' slots meet in LDS at the end and the workgroup leaves one partial row.
template <typename T, int NT, int K, bool R>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_norm_bwd(NormArgs a) {
  constexpr int kRows = NT < 256 ? 256 / NT : 1;
  __shared__ float red[16];
  // the next row's loads in flight behind this one's arithmetic, but where 1024 threads hold 16 columns each: their
  // 128 registers take no second row (16384 x 4096 bf16 110 us; 191 with both, which spills).  (More than 8192 columns
  // that are no multiple of 8 spill 8 registers all the same, fp32 14.)
  constexpr bool kAhead = NT * K < 2048;
  __shared__ float slot[kRows > 1 ? kRows : 1][kRows > 1 ? NT * 8 + 4 : 1];
  const int l = threadIdx.x % NT, g = threadIdx.x / NT;
  float w[K][8], dw[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * NT + l) * 8, nv = a.cols - c;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[k][i] = 0.f;
    if (nv > 0) ld_row<float, 8>(a.w + c, nv, w[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[k][i] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * kRows;
  const bool whole = a.cols >= 8;
  Ask<T, R> as[K], ad[K], ax[K];
  float arstd = 0.f;
  auto ask = [&](int64_t r) {
    const bool in = r < a.rows;
    if (in) arstd = a.rstd_in[r];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + l) * 8, nv = in ? a.cols - c : 0;
      as[k].ask((const T*)a.s_in + r * a.lds + c, nv, whole);
      ad[k].ask((const T*)a.dy + r * a.lddy + c, nv, whole);
      if (a.ds) ax[k].ask((const T*)a.ds + r * a.ldds + c, nv, whole);
    }
  };
  int64_t r = (int64_t)blockIdx.x * kRows + g;
  if constexpr (kAhead) ask(r);
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += step, r += step) {
    const bool in = r < a.rows;
    if constexpr (!kAhead) {
#pragma unroll
      for (int k = 0; k < K; ++k) as[k] = ad[k] = ax[k] = Ask<T, R>{};
      ask(r);
    }
    const float rstd = arstd;
    float n[K][8], d[K][8], o[K][8], sum = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + l) * 8, nv = in ? a.cols - c : 0;
      as[k].take((const T*)a.s_in + r * a.lds + c, nv, whole, n[k]);
      ad[k].take((const T*)a.dy + r * a.lddy + c, nv, whole, d[k]);
      if (a.ds) ax[k].take((const T*)a.ds + r * a.ldds + c, nv, whole, o[k]);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) o[k][i] = 0.f;
    }
    // (the tails of an element-by-element read are in hand here too: dx may be dy or ds)
    if constexpr (kAhead) ask(r + step);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n[k][i] = in ? n[k][i] * rstd : 0.f;
        dw[k][i] = fmaf(d[k][i], n[k][i], dw[k][i]);
        d[k][i] *= w[k][i];
        sum = fmaf(d[k][i], n[k][i], sum);
      }
    }
    const float mean = row_sum<NT, float>(sum, red) / (float)a.cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + l) * 8, nv = in ? a.cols - c : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[k][i] = fmaf(rstd, d[k][i] - n[k][i] * mean, o[k][i]);
      if (nv > 0) st_row<T, 8, R>((T*)a.dx + r * a.lddx + c, nv, o[k]);
    }
  }
  float* out = a.part + (int64_t)blockIdx.x * a.cols;
  if constexpr (kRows > 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) slot[g][l * 8 + i] = dw[k][i];
      __syncthreads();
      for (int j = threadIdx.x; j < NT * 8; j += 256) {
        float t = 0.f;
#pragma unroll
        for (int q = 0; q < kRows; ++q) t += slot[q][j];
        const int c = k * NT * 8 + j;
        if (c < a.cols) out[c] = t;
      }
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * NT + l) * 8, nv = a.cols - c;
      if (nv > 0) st_row<float, 8>(out + c, nv, dw[k]);
    }
  }
}

// dw [cols] = the partial rows' sum, in order: 16 columns a workgroup, 64 stretches of the rows each
__global__ __launch_bounds__(1024) void k_norm_dw(const float* __restrict__ part, int blocks, int cols,
                                                  float* __restrict__ dw) {
  __shared__ float red[64][17];
  const int j = threadIdx.x & 15, t = threadIdx.x >> 4, c = blockIdx.x * 16 + j;
  const int per = (blocks + 63) / 64, b0 = min(t * per, blocks), b1 = min(b0 + per, blocks);
  float v = 0.f;
  if (c < cols)
    for (int b = b0; b < b1; b += 8) {  // eight loads in flight
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = b + i < b1 ? part[(int64_t)(b + i) * cols + c] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += x[i];
    }
  red[t][j] = v;
  __syncthreads();
  if (t == 0 && c < cols) {
    float sum = 0.f;
#pragma unroll
    for (int q = 0; q < 64; ++q) sum += red[q][j];
    dw[c] = sum;
  }
}

// the 8-bit form's values: 8 columns a thread
template <typename O>
__global__ __launch_bounds__(256) void k_dequant(const unsigned char* __restrict__ q, const unsigned char* __restrict__ scale,
                                                 int64_t rows, int cols, int kp, O* __restrict__ out, int64_t ldo) {
  const int per = (cols + 7) / 8;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= rows * per) return;
  const int64_t r = u / per;
  const int c = (int)(u - r * per) * 8;
  const uint2 b = *reinterpret_cast<const uint2*>(q + r * kp + c);
  const unsigned e = scale[r * (kp / kBlk) + c / kBlk];
  const float s = e == 255u ? __builtin_nanf("") : exp_val(e);
  float x[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int v = (int)(i ? b.y : b.x);
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
    x[4 * i] = lo[0] * s;
    x[4 * i + 1] = lo[1] * s;
    x[4 * i + 2] = hi[0] * s;
    x[4 * i + 3] = hi[1] * s;
  }
  st_row<O, 8>(out + r * ldo + c, cols - c, x);
}

// Threads a row: the fewest that hold it, but a whole workgroup for wide rows, whose wave would keep too
// few loads in flight.  From 4097 to 8192 columns the forward takes two of 512 threads to a compute unit (8192 x 4100
// bf16 54 us, 70 with 1024 threads of 8 columns; 4096 x 8192 46 either way), the backward, whose registers let only
// one stay, 1024 (58 and 73).
template <bool FWD, typename F>
void by_cols(int cols, F&& f) {
  using std::integral_constant;
  auto go = [&](auto ragged) {
    if (cols <= 128) f(integral_constant<int, 16>{}, integral_constant<int, 1>{}, ragged);
    else if (cols <= 256) f(integral_constant<int, 32>{}, integral_constant<int, 1>{}, ragged);
    else if (cols <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{}, ragged);
    else if (cols <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{}, ragged);
    else if (cols <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 1>{}, ragged);
    else if (cols <= 4096) f(integral_constant<int, 256>{}, integral_constant<int, 2>{}, ragged);
    else if (cols <= 8192) f(integral_constant<int, FWD ? 512 : 1024>{}, integral_constant<int, FWD ? 2 : 1>{}, ragged);
    else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{}, ragged);
  };
  if (cols % 8) go(std::true_type{});
  else go(std::false_type{});
}

bool norm_dims_ok(int64_t rows, int cols) {
  return rows >= 0 && rows <= 0x7fffffff && cols > 0 && cols <= kMaxCols;
}
bool dims8_ok(int64_t rows, int cols) { return rows >= 0 && rows <= 0x7fffffff && cols > 0 && cols <= kMaxCols8; }
bool eps_ok(float eps) { return eps > 0.f && eps < __builtin_inff(); }
int kp_of(int cols) { return (cols + kBlk - 1) / kBlk * kBlk; }

template <int MODE>
void run_norm(const NormArgs& a, int dtype, hipStream_t s) {
  by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    by_cols<true>(a.cols, [&](auto nt, auto kk, auto ragged) {
      constexpr int NT = decltype(nt)::value, K = decltype(kk)::value, rows = NT < 256 ? 256 / NT : 1;
      const int64_t blocks = std::min<int64_t>((a.rows + rows - 1) / rows, NT < 512 ? 2048 : NT < 1024 ? 1024 : 512);
      const unsigned stretches = MODE == 2 ? (a.cols + kMaxCols - 1) / kMaxCols : 1;  // (of the norm: checked)
      hipLaunchKernelGGL((k_norm<T, NT, K, MODE, decltype(ragged)::value>), dim3((unsigned)blocks, stretches),
                         dim3(NT < 256 ? 256 : NT), 0, s, a);
    });
  });
}
// Workgroups of the backward, each of which leaves a partial row of dw.  Above 4096 columns one of 1024 threads fills a
// compute unit: 256 (4096 x 8192 bf16 46 us; 67 with 1024 of them).  Below, 512, whose fewer partial rows are worth
// more than the waves (8192 x 1024 bf16 17.8 us, 20.2 with 1024; 16384 x 4096 107 and 126), but 1024 for narrow
// rows (196608 x 64 bf16 21 us, 23 with 512) and for ragged ones, whose groups take more instructions (16384 x 1191
// 40 and 59).  A row at a time: at least two rows each (512 x 4096 11.8 us, 15.1 with one).
int bwd_blocks(int64_t rows, int cols) {
  const int per = cols <= 128 ? 16 : cols <= 256 ? 8 : cols <= 1024 ? 4 : 2;  // rows a workgroup takes at least
  const int most = cols > 4096 ? 256 : cols <= 128 || cols % 8 ? 1024 : 512;
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, (rows + per - 1) / per));
}

}  // namespace
}  // namespace seq
}  // namespace dssm

using namespace dssm::seq;

extern "C" int dssm_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldres, const float* weight,
                             int64_t rows, int cols, int dtype, float eps, void* y, int64_t ldy, void* s, int64_t lds,
                             float* rstd, void* stream) {
  if (!seq_dtype(dtype) || !norm_dims_ok(rows, cols) || !eps_ok(eps) || !weight || ldx < cols || ldy < cols ||
      (residual && ldres < cols) || (s && lds < cols) || (rows > 0 && (!x || !y)))
    return dssm::report_error(DSSM_E_INVALID, "rms_norm: bad argument (1 to 16384 columns, a positive finite eps)");
  if (rows == 0) return DSSM_OK;
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.res = residual;
  a.ldres = ldres;
  a.w = weight;
  a.rows = rows;
  a.cols = cols;
  a.eps = eps;
  a.y = y;
  a.ldy = ldy;
  a.s = s;
  a.lds = lds;
  a.rstd = rstd;
  run_norm<0>(a, dtype, (hipStream_t)stream);
  return seq_status(hipGetLastError());
}

extern "C" int dssm_rms_norm_blocks8(const void* x, int64_t ldx, const void* residual, int64_t ldres, const float* weight,
                                     int64_t rows, int cols, int dtype, float eps, void* q, void* scale, void* s,
                                     int64_t lds, float* rstd, void* stream) {
  if (!seq_dtype(dtype) || !norm_dims_ok(rows, cols) || !eps_ok(eps) || !weight || ldx < cols || (residual && ldres < cols) ||
      (s && lds < cols) || (rows > 0 && (!x || !q || !scale)) || (uintptr_t)q % 16)
    return dssm::report_error(DSSM_E_INVALID,
                              "rms_norm_blocks8: bad argument (1 to 16384 columns, a positive finite eps, 16-byte aligned values)");
  if (rows == 0) return DSSM_OK;
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.res = residual;
  a.ldres = ldres;
  a.w = weight;
  a.rows = rows;
  a.cols = cols;
  a.kp = kp_of(cols);
  a.eps = eps;
  a.q = (unsigned char*)q;
  a.scale = (unsigned char*)scale;
  a.s = s;
  a.lds = lds;
  a.rstd = rstd;
  run_norm<1>(a, dtype, (hipStream_t)stream);
  return seq_status(hipGetLastError());
}

extern "C" size_t dssm_rms_norm_bwd_ws_bytes(int64_t rows, int cols) {
  return norm_dims_ok(rows, cols) ? (size_t)bwd_blocks(rows, cols) * cols * sizeof(float) + 16 : 0;
}

extern "C" int dssm_rms_norm_bwd(const void* dy, int64_t lddy, const void* s, int64_t lds, const float* weight,
                                 const float* rstd, const void* ds, int64_t ldds, int64_t rows, int cols, int dtype, void* dx,
                                 int64_t lddx, float* dweight, void* ws, size_t ws_bytes, void* stream) {
  if (!seq_dtype(dtype) || !norm_dims_ok(rows, cols) || !weight || !dweight || lddy < cols || lds < cols || lddx < cols ||
      (ds && ldds < cols) || (rows > 0 && (!dy || !s || !rstd || !dx)))
    return dssm::report_error(DSSM_E_INVALID, "rms_norm_bwd: bad argument (1 to 16384 columns)");
  if (!ws || ws_bytes < dssm_rms_norm_bwd_ws_bytes(rows, cols))
    return dssm::report_error(DSSM_E_INVALID, "rms_norm_bwd: workspace too small (dssm_rms_norm_bwd_ws_bytes)");
  hipStream_t st = (hipStream_t)stream;
  NormArgs a{};
  a.dy = dy;
  a.lddy = lddy;
  a.s_in = s;
  a.lds = lds;
  a.w = weight;
  a.rstd_in = rstd;
  a.ds = ds;
  a.ldds = ldds;
  a.rows = rows;
  a.cols = cols;
  a.dx = dx;
  a.lddx = lddx;
  a.part = (float*)ws;
  const int blocks = bwd_blocks(rows, cols);
  by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    by_cols<false>(cols, [&](auto nt, auto kk, auto ragged) {
      constexpr int NT = decltype(nt)::value, K = decltype(kk)::value;
      hipLaunchKernelGGL((k_norm_bwd<T, NT, K, decltype(ragged)::value>), dim3(blocks), dim3(NT < 256 ? 256 : NT), 0, st, a);
    });
  });
  hipLaunchKernelGGL(k_norm_dw, dim3((cols + 15) / 16), dim3(1024), 0, st, (const float*)ws, blocks, cols, dweight);
  return seq_status(hipGetLastError());
}

extern "C" int dssm_quantize_blocks8(const void* x, int64_t ldx, int64_t rows, int cols, int dtype, void* q, void* scale,
                                     void* stream) {
  if (!seq_dtype(dtype) || !dims8_ok(rows, cols) || ldx < cols || (rows > 0 && (!x || !q || !scale)) ||
      (uintptr_t)q % 16)
    return dssm::report_error(DSSM_E_INVALID, "quantize_blocks8: bad argument (1 to 2^22 columns, 16-byte aligned values)");
  if (rows == 0) return DSSM_OK;
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.rows = rows;
  a.cols = cols;
  a.kp = kp_of(cols);
  a.q = (unsigned char*)q;
  a.scale = (unsigned char*)scale;
  run_norm<2>(a, dtype, (hipStream_t)stream);
  return seq_status(hipGetLastError());
}

extern "C" int dssm_dequantize_blocks8(const void* q, const void* scale, int64_t rows, int cols, void* out, int64_t ldo,
                                       int out_dtype, void* stream) {
  if (!seq_dtype(out_dtype) || !dims8_ok(rows, cols) || ldo < cols || (rows > 0 && (!out || !q || !scale)) ||
      (uintptr_t)q % 16)
    return dssm::report_error(DSSM_E_INVALID, "dequantize_blocks8: bad argument (1 to 2^22 columns, 16-byte aligned values)");
  if (rows == 0) return DSSM_OK;
  const int64_t units = rows * ((cols + 7) / 8);
  if ((units + 255) / 256 > kMaxBlocks) return dssm::report_error(DSSM_E_UNSUPPORTED, "dequantize_blocks8: too many values");
  by_dtype(out_dtype, [&](auto tag) {
    using O = decltype(tag);
    hipLaunchKernelGGL(k_dequant<O>, dim3((unsigned)((units + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                       (const unsigned char*)q, (const unsigned char*)scale, rows, cols, kp_of(cols), (O*)out, ldo);
  });
  return seq_status(hipGetLastError());
}
