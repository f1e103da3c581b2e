// Shared pieces of the sequence-tower operators (embed.hip, linrec.hip, rmsnorm.hip, gemm8.hip): the
// three storage types, vector loads of rows of any alignment, and the 8-bit block form's arithmetic.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dssm.h"
#include "common.h"

namespace dssm {
int report_error(int code, const char* msg);
}

namespace dssm {
namespace seq {

struct f16s {  // fp16 storage, a type of its own beside u16 (bf16) and float
  _Float16 v;
};

__device__ __forceinline__ float ld1(float v) { return v; }
__device__ __forceinline__ float ld1(u16 v) { return bf2f(v); }
__device__ __forceinline__ float ld1(f16s v) { return (float)v.v; }
template <typename T> __device__ __forceinline__ T st1(float v);
template <> __device__ __forceinline__ float st1<float>(float v) { return v; }
template <> __device__ __forceinline__ u16 st1<u16>(float v) { return f2bf(v); }
template <> __device__ __forceinline__ f16s st1<f16s>(float v) { return f16s{(_Float16)v}; }

// V consecutive elements.  The type's alignment is one element's: gfx950 global memory takes accesses of
// any alignment (rows of an odd width start anywhere), so one vector access serves every stride.
template <typename T, int V>
struct __attribute__((packed, aligned(alignof(T)))) Pack {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> ldv(const T* p) {
  Pack<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const Pack<T, V>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}
// the first `n` of V elements (zeros behind them), and their store; n < V only at a row's ragged end
template <typename T, int V>
__device__ __forceinline__ void ld_row(const T* p, int n, float (&x)[V]) {
  if (n >= V) {
    const Pack<T, V> r = ldv<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = ld1(r.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = i < n ? ld1(p[i]) : 0.f;
  }
}
// (by value: a choice between two array elements would put the array into memory)
__device__ __forceinline__ float pick(bool c, float a, float b) { return c ? a : b; }
template <typename T, int V, bool R = true>
__device__ __forceinline__ void st_row(T* p, int n, const float (&x)[V]) {
  if (n >= V) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = st1<T>(x[i]);
    stv<T, V>(p, r);
  } else if constexpr (!R) {
  } else if constexpr (V == 8) {  // four, two and one of them: three stores at most
    if (n <= 0) return;
    Pack<T, 4> a;
    Pack<T, 2> b;
#pragma unroll
    for (int i = 0; i < 4; ++i) a.v[i] = st1<T>(x[i]);
    if (n & 4) stv<T, 4>(p, a);
#pragma unroll
    for (int i = 0; i < 2; ++i) b.v[i] = st1<T>(pick(n & 4, x[i + 4], x[i]));
    if (n & 2) stv<T, 2>(p + (n & 4), b);
    if (n & 1) p[n - 1] = st1<T>(pick(n & 4, pick(n & 2, x[6], x[4]), pick(n & 2, x[2], x[0])));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = st1<T>(x[i]);
  }
}

// The same load in two steps, so that a kernel asks for all it needs before it waits for any: ask() issues a
// whole group's access and does not look at it, take() converts.  A ragged group (only the last one of a row whose
// width is no multiple of 8) asks for the row's last eight elements, its neighbour's among them, and take() moves its
// own down: element by element the row's end would wait for memory once more (44295 x 1191 bf16 forward 170 us and
// 106 so, backward 256 and 114).  `whole`: the row has eight elements.  R false: no group is ragged, and the code
// for them, which costs short launches 0.3 us, is left out.
template <typename T, bool R>
struct Ask {
  Pack<T, 8> r;
  __device__ __forceinline__ void ask(const T* p, int n, bool whole) {
    const T* q = !R || n >= 8 ? p : p + n - 8;
    if (n > (R && whole ? 0 : 7)) r = ldv<T, 8>(q);
  }
  __device__ __forceinline__ void take(const T* p, int n, bool whole, float (&x)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = ld1(r.v[i]);
    if (n < 8) {
      if (R && whole && n > 0) {
        const int down = 8 - n;
#pragma unroll
        for (int d = 4; d; d >>= 1)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = down & d ? (i + d < 8 ? x[i + d] : 0.f) : x[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = R && i < n ? ld1(p[i]) : 0.f;
      }
    }
  }
};

// ---- the 8-bit block form ---------------------------------------------------------------------------
// A row's 128 columns share the power of two 2^e, the smallest that brings their largest finite
// magnitude into e4m3's +-448; it is stored as the byte e + 127 (E8M0), which the matrix instruction
// takes as it is.  A power of two costs the values no precision: a float's relative step does not
// depend on its exponent.
constexpr int kBlk = 128;

__device__ __forceinline__ unsigned blk_exp(float amax) {
  // amax = m 2^k, m in [1, 2): 448 = 1.75 * 2^8, so e = k - 8, one more where m > 1.75
  if (!(amax > 0.f)) return 127u;
  const unsigned b = __float_as_uint(amax);
  int k = (int)(b >> 23) - 127;
  unsigned m = b & 0x7fffffu;
  if (k == -127) return 0u;  // below the normal range 2^-127 is small enough
  const int e = k - 8 + (m > 0x600000u ? 1 : 0);
  const int s = e + 127;
  return (unsigned)(s < 0 ? 0 : s > 254 ? 254 : s);
}
// 2^(e - 127) and its reciprocal, exactly (e = 0 and 254 give subnormals, which gfx950's fp32 keeps)
__device__ __forceinline__ float exp_val(unsigned e) {
  return __uint_as_float(e ? e << 23 : 0x400000u);
}
__device__ __forceinline__ float exp_inv(unsigned e) {
  return __uint_as_float(e < 254u ? (254u - e) << 23 : 0x400000u);
}
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < __builtin_inff() ? a : 0.f;  // NaN and infinities do not set a block's scale
}
// eight values times `inv` -> eight e4m3 bytes, ties to even; NaN and infinities become NaN
__device__ __forceinline__ uint2 to_e4m3x8(const float (&x)[8], float inv) {
  float y[8];
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bad |= (fabsf(x[i]) < __builtin_inff() ? 0u : 1u) << i;
    y[i] = (bad >> i) & 1u ? 0.f : x[i] * inv;
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  uint2 r = make_uint2((unsigned)lo, (unsigned)hi);
  if (bad) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((bad >> i) & 1u) r.x |= 0x7fu << (8 * i);
      if ((bad >> (i + 4)) & 1u) r.y |= 0x7fu << (8 * i);
    }
  }
  return r;
}

// the largest of a value over the aligned 16 lanes that hold a block of 128 columns, 8 columns a lane
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_mov<0xB1>(v));
  v = fmaxf(v, dpp_mov<0x4E>(v));
  v = fmaxf(v, dpp_mov<0x141>(v));
  return fmaxf(v, dpp_mov<0x140>(v));
}

constexpr int64_t kMaxBlocks = (1 << 24) - 1;  // workgroups of 256: a launch has fewer than 2^32 threads

inline int seq_status(hipError_t e) {
  return e == hipSuccess ? DSSM_OK : report_error(DSSM_E_HIP, hipGetErrorString(e));
}
inline bool seq_dtype(int d) { return d == DSSM_F32 || d == DSSM_BF16 || d == DSSM_F16; }

// f(type tag): calls with the storage type of dtype code d
template <typename F>
inline void by_dtype(int d, F&& f) {
  if (d == DSSM_F32) f(float{});
  else if (d == DSSM_BF16) f(u16{});
  else f(f16s{});
}

}  // namespace seq
}  // namespace dssm
