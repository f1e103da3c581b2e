// 8-bit floating-point product with a scale for each block of 128:
//
//   out[m, n] = sum over blocks b of 2^(ea[m, b] + ew[n, b] - 254) * sum over k in b of a[m, k] w[n, k]  (+ bias[n])
//
// a [M x Kp], w [N x Kp] e4m3, Kp a multiple of 128 (the form's zero padding stands in for a ragged K).
// v_mfma_scale_f32_16x16x128 multiplies 16 x 16 x 128 and applies an E8M0 scale per row and 32 columns of
// each operand by itself; the block of 128 gives its four groups the same byte, so the scales cost no
// instruction of their own and everything accumulates in fp32 inside one chain per output.
//
// Precision: a product of two e4m3 values is exact, but the matrix unit adds eight neighbouring products on a
// grid of 2^-13 of the largest before they join the fp32 chain (measured: beside a product of 2^8, one of
// 2^-5 among the same eight counts and one of 2^-6 does not; among different eights it counts to fp32's last
// bit; v_mfma_f32_16x16x32_fp8_fp8 does the same).  Against the operands' own rounding of 2^-4 that is
// nothing, and below the half step of the bf16 and fp16 results that are offered (2^-8, 2^-11); an fp32
// result would claim more than the unit gives, and is refused.
//
// The instruction's A operand is w and its B operand is a: a lane then ends with four neighbouring n of
// one m, one 8- or 16-byte store.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "seq.h"

namespace dssm {
namespace seq {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Gemm8Args {
  const unsigned char *a, *ea, *w, *ew;
  const float* bias;
  void* out;
  int64_t ldo;
  int M, N, KB;  // KB: blocks of 128
};

__device__ __forceinline__ f32x4 mfma8(const i32x8& w, const i32x8& a, f32x4 c, int sw, int sa) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 0, sw, 0, sa);
}

// a row's scale bytes of blocks kb .. kb + 3 in one word (bytes behind the row's last block: zero)
__device__ __forceinline__ unsigned scale4(const unsigned char* row, int kb, int KB) {
  unsigned v = 0;
  if (kb + 4 <= KB) {
    __builtin_memcpy(&v, row + kb, 4);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (kb + i < KB) v |= (unsigned)row[kb + i] << (8 * i);
  }
  return v;
}

// four neighbouring outputs n .. n + 3 of row m
template <typename O>
__device__ __forceinline__ void store4(const Gemm8Args& g, int m, int n, f32x4 v) {
  if (m >= g.M || n >= g.N) return;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = v[i] + (g.bias && n + i < g.N ? g.bias[n + i] : 0.f);
  st_row<O, 4>((O*)g.out + (int64_t)m * g.ldo + n, g.N - n, x);
}

// ---- tiles -------------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes (WM MI 16) x (WN NI 16) outputs.  Both operands' blocks of 128
// columns go from memory straight to LDS, 16 bytes a lane, into one half of a double buffer while the
// other is multiplied.  A row's 128 bytes are eight 16-byte pieces; piece p of row r lies at p ^ (r & 7),
// so that the 16 rows a fragment read touches spread over all banks.  The direct load writes LDS in lane
// order, so the permutation is applied to the address each lane loads from.
template <int WM, int WN, int MI, int NI, typename O>
__global__ __launch_bounds__(WM * WN * 64) void k_gemm8(Gemm8Args g) {
  constexpr int BM = WM * MI * 16, BN = WN * NI * 16, NW = WM * WN, kLoads = (BM + BN) / 8 / NW;
  static_assert((BM + BN) / 8 % NW == 0 && BM / 8 % NW == 0, "every wave loads the same number of 8-row stripes");
  __shared__ __attribute__((aligned(16))) unsigned char lds[2][(BM + BN) * kBlk];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, wm = wv % WM, wn = wv / WM;
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  // neighbouring tiles to one XCD, in bands of 8 tile rows whose operands its L2 keeps
  int t = xcd_tile(blockIdx.x, tm * tn);
  constexpr int kBand = 8;
  const int band = t / (kBand * tn), rows = min(kBand, tm - band * kBand);
  t -= band * kBand * tn;
  const int m0 = (band * kBand + t % rows) * BM, n0 = t / rows * BN;
  const int64_t Kp = (int64_t)g.KB * kBlk;

  // stripe i of this wave: rows 8 (wv + i NW) ... of the tile's BM + BN rows, a's first
  const unsigned char* src[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = (wv + i * NW) * 8 + (lane >> 3), p = (lane & 7) ^ (r & 7);
    const bool isa = r < BM;
    const int row = isa ? min(m0 + r, g.M - 1) : min(n0 + r - BM, g.N - 1);
    src[i] = (isa ? g.a : g.w) + (int64_t)row * Kp + p * 16;
  }
  auto load = [&](int kb, int buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(src[i] + (int64_t)kb * kBlk),
                                       (__attribute__((address_space(3))) unsigned*)&lds[buf][(wv + i * NW) * 1024], 16, 0,
                                       0);
  };
  const unsigned char* ea[MI];
  const unsigned char* ew[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) ea[i] = g.ea + (int64_t)min(m0 + (wm * MI + i) * 16 + (lane & 15), g.M - 1) * g.KB;
#pragma unroll
  for (int j = 0; j < NI; ++j) ew[j] = g.ew + (int64_t)min(n0 + (wn * NI + j) * 16 + (lane & 15), g.N - 1) * g.KB;
  unsigned sa[MI], sw[NI];

  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // a fragment: lane l holds 32 of row l % 16's bytes, the pieces l / 16 and l / 16 + 4 (the order of k
  // inside a block is free as long as both operands use the same)
  const int fr = lane & 15, fp = lane >> 4;
  auto frag = [&](const unsigned char* base, int r) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(base + (r + fr) * kBlk + ((fp ^ (fr & 7)) * 16));
    const i32x4 hi = *reinterpret_cast<const i32x4*>(base + (r + fr) * kBlk + (((fp + 4) ^ (fr & 7)) * 16));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  load(0, 0);
  for (int kb = 0; kb < g.KB; ++kb) {
    const int buf = kb & 1;
    if ((kb & 3) == 0) {
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[i] = scale4(ea[i], kb, g.KB);
#pragma unroll
      for (int j = 0; j < NI; ++j) sw[j] = scale4(ew[j], kb, g.KB);
    }
    // this wave's direct loads have landed; behind the barrier all waves' have, and all have finished
    // reading the half that is loaded next
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (kb + 1 < g.KB) load(kb + 1, buf ^ 1);
    const unsigned char* A = lds[buf];
    const unsigned char* W = lds[buf] + BM * kBlk;
    i32x8 fw[NI];
#pragma unroll
    for (int j = 0; j < NI; ++j) fw[j] = frag(W, (wn * NI + j) * 16);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const i32x8 fa = frag(A, (wm * MI + i) * 16);
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = mfma8(fw[j], fa, acc[i][j], (int)sw[j], (int)sa[i]);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) sa[i] >>= 8;
#pragma unroll
    for (int j = 0; j < NI; ++j) sw[j] >>= 8;
  }
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
      store4<O>(g, m0 + (wm * MI + i) * 16 + fr, n0 + (wn * NI + j) * 16 + fp * 4, acc[i][j]);
}

// ---- few rows ----------------------------------------------------------------------------------
// The weights are read once, straight into registers: a workgroup takes 16 of their rows against 16 MT
// rows of a, its eight waves every eighth block of 128 columns, four blocks' loads in flight; the waves'
// sums meet in LDS in wave order.
template <int MT, typename O>
__global__ __launch_bounds__(512) void k_gemm8_rows(Gemm8Args g) {
  constexpr int NW = 8, kDepth = MT > 2 ? 2 : 4;
  __shared__ f32x4 part[NW][MT][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, fr = lane & 15, fp = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int64_t Kp = (int64_t)g.KB * kBlk;
  const int64_t nr = min(n0 + fr, g.N - 1);
  const unsigned char* w = g.w + nr * Kp + fp * 32;
  const unsigned char* ew = g.ew + nr * g.KB;
  const unsigned char* a[MT];
  const unsigned char* ea[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = min(m0 + i * 16 + fr, g.M - 1);
    a[i] = g.a + m * Kp + fp * 32;
    ea[i] = g.ea + m * g.KB;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kb = wv; kb < g.KB; kb += NW * kDepth) {
    i32x8 fw[kDepth], fa[kDepth][MT];
    int sw[kDepth], sa[kDepth][MT];
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const int k = kb + d * NW;
      if (k < g.KB) {
        fw[d] = *reinterpret_cast<const i32x8*>(w + (int64_t)k * kBlk);
        sw[d] = ew[k];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          fa[d][i] = *reinterpret_cast<const i32x8*>(a[i] + (int64_t)k * kBlk);
          sa[d][i] = ea[i][k];
        }
      }
    }
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (kb + d * NW < g.KB) {
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = mfma8(fw[d], fa[d][i], acc[i], sw[d], sa[d][i]);
      }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[wv][i][lane] = acc[i];
  __syncthreads();
  for (int i = wv; i < MT; i += NW) {
    f32x4 v = part[0][i][lane];
#pragma unroll
    for (int k = 1; k < NW; ++k) v += part[k][i][lane];
    store4<O>(g, m0 + i * 16 + fr, n0 + fp * 4, v);
  }
}

template <typename O>
void run_gemm8(const Gemm8Args& g, hipStream_t s) {
  const auto tiles = [&](int bm, int bn) { return (int64_t)((g.M + bm - 1) / bm) * ((g.N + bn - 1) / bn); };
  if (g.M <= 16) {
    hipLaunchKernelGGL((k_gemm8_rows<1, O>), dim3((g.N + 15) / 16, 1), dim3(512), 0, s, g);
  } else if (g.M <= 32) {
    hipLaunchKernelGGL((k_gemm8_rows<2, O>), dim3((g.N + 15) / 16, 1), dim3(512), 0, s, g);
  } else if (g.M <= 64 || tiles(128, 128) < 64) {
    hipLaunchKernelGGL((k_gemm8_rows<4, O>), dim3((g.N + 15) / 16, (g.M + 63) / 64), dim3(512), 0, s, g);
  } else if (tiles(256, 256) < 128) {
    hipLaunchKernelGGL((k_gemm8<2, 2, 4, 4, O>), dim3((unsigned)tiles(128, 128)), dim3(256), 0, s, g);
  } else {
    hipLaunchKernelGGL((k_gemm8<2, 4, 8, 4, O>), dim3((unsigned)tiles(256, 256)), dim3(512), 0, s, g);
  }
}

}  // namespace
}  // namespace seq
}  // namespace dssm

using namespace dssm::seq;

extern "C" int dssm_blocks8_matmul(const void* a, const void* ascale, const void* w, const void* wscale, int64_t M, int64_t N,
                                   int64_t K, const float* bias, void* out, int64_t ldo, int out_dtype, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || M > (1 << 28) || N > (1 << 24) || K > (1 << 28) || ldo < N || (out_dtype != DSSM_BF16 && out_dtype != DSSM_F16) ||
      (M > 0 && N > 0 && (!a || !ascale || !w || !wscale || !out)) || (uintptr_t)a % 16 || (uintptr_t)w % 16)
    return dssm::report_error(DSSM_E_INVALID, "blocks8_matmul: bad argument (16-byte aligned values, bf16 or fp16 result)");
  if (M == 0 || N == 0) return DSSM_OK;
  Gemm8Args g{};
  g.a = (const unsigned char*)a;
  g.ea = (const unsigned char*)ascale;
  g.w = (const unsigned char*)w;
  g.ew = (const unsigned char*)wscale;
  g.bias = bias;
  g.out = out;
  g.ldo = ldo;
  g.M = (int)M;
  g.N = (int)N;
  g.KB = (int)((K + kBlk - 1) / kBlk);
  if (out_dtype == DSSM_BF16) run_gemm8<u16>(g, (hipStream_t)stream);
  else run_gemm8<f16s>(g, (hipStream_t)stream);
  return seq_status(hipGetLastError());
}
