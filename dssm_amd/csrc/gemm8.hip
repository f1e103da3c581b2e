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
typedef float f32x16 __attribute__((ext_vector_type(16)));

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
__device__ __forceinline__ unsigned scale_word(const unsigned char* p) {
  unsigned v;
  __builtin_memcpy(&v, p, 4);
  return v;
}
__device__ __forceinline__ unsigned scale4(const unsigned char* row, int kb, int KB) {
  if (kb + 4 <= KB) return scale_word(row + kb);
  unsigned v = 0;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (kb + i < KB) v |= (unsigned)row[kb + i] << (8 * i);
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
// A workgroup of WM x WN waves computes (WM MI 32) x (WN NI 32) outputs with v_mfma_scale_f32_32x32x64.
//
// Both operands go from memory straight to LDS, 16 bytes a lane, a block of 128 columns at a time into one half of
// a double buffer; whole 128-byte lines, because the two halves of a line that are asked for apart meet as
// one pending line in the vector cache and stall it.  A block is multiplied in two rounds of 64 columns, and a
// round multiplies fragments that are in registers already while it reads the next round's: when a block's
// second round begins, nobody needs its LDS half any more, and the block after the next is asked for, two
// rounds of products (2048 cycles of the matrix units) before its first fragment is read.
//
// A row's 128 bytes are eight 16-byte pieces; piece p of row r lies at p ^ (r >> 1 & 7).  A 16-byte read serves
// sixteen lanes a cycle: lanes 0-3, 12-15, 20-23 and 24-27 of a half wave, then the others (found with the
// conflict counter, which reads zero); of these rows no two of the same parity have the same r >> 1 & 7, so
// they cover all 64 banks.  The direct load writes LDS in lane order, so the permutation is applied to the
// address that each lane loads from.
template <int WM, int WN, int MI, int NI, typename O>
__global__ __launch_bounds__(WM * WN * 64, WM * WN == 8 ? 2 : 1) void k_gemm8(Gemm8Args g) {
  constexpr int BM = WM * MI * 32, BN = WN * NI * 32, NW = WM * WN, kLoads = (BM + BN) / 8 / NW;
  static_assert(kLoads * 8 * NW == BM + BN && BM % 8 == 0, "every wave loads the same number of 8-row stripes");
  constexpr int kScaleRows = (BM + BN) / (NW * 64);  // a thread's
  static_assert(kScaleRows * NW * 64 == BM + BN && BM % 64 == 0, "a row's scales are loaded by one thread");
  // two blocks, then two words of scales a row.  One object: of two the compiler knows that they are two, tells
  // the direct loads apart by that, and puts a wait for all of them in front of every read.
  constexpr int kBuf = (BM + BN) * kBlk;
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * kBuf + 2 * (BM + BN) * 4];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wv % WM, wn = wv / WM;
  const int tm = (g.M + BM - 1) / BM, tn = (g.N + BN - 1) / BN;
  // neighbouring tiles to one XCD, in bands of 8 tile rows whose operands its L2 keeps
  int t = xcd_tile(blockIdx.x, tm * tn);
  constexpr int kBand = 8;
  const int band = t / (kBand * tn), rows = min(kBand, tm - band * kBand);
  t -= band * kBand * tn;
  const int m0 = (band * kBand + t % rows) * BM, n0 = t / rows * BN;
  const unsigned Kp = (unsigned)g.KB * kBlk;  // (a tile's rows span less than 2^32 bytes: checked on the host)

  // stripe i of this wave: rows 8 (wv + i NW) ... of the tile's BM + BN rows, a's first; rows behind the last
  // one read the last one (their outputs are not stored)
  const unsigned char* base[kLoads];
  unsigned off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r0 = (wv + i * NW) * 8, r = r0 + (lane >> 3), p = (lane & 7) ^ (r >> 1 & 7);
    const bool isa = r0 < BM;
    base[i] = isa ? g.a + (int64_t)m0 * Kp : g.w + (int64_t)n0 * Kp;
    off[i] = (unsigned)(isa ? min(r, g.M - 1 - m0) : min(r - BM, g.N - 1 - n0)) * Kp + p * 16;
  }
  // (behind the last block the last one is loaded again, into a half that serves no more: no branch)
  auto load = [&](int kb, int from, int to) {
    const unsigned at = (unsigned)min(kb, g.KB - 1) * kBlk;
#pragma unroll
    for (int i = from; i < to; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(base[i] + at + off[i]),
                                       (__attribute__((address_space(3))) unsigned*)&lds[(kb & 1) * kBuf + (wv + i * NW) * 1024],
                                       16, 0, 0);
  };
  // Scales: a thread holds a row's of four blocks in one word, asked for three blocks ahead and written to LDS
  // two ahead.  (The last word of a row starts at KB - 4 and is shifted down.)
  const unsigned char* srow[kScaleRows];
  unsigned sword[kScaleRows];
#pragma unroll
  for (int i = 0; i < kScaleRows; ++i) {
    const int r = i * NW * 64 + threadIdx.x;
    srow[i] = r < BM ? g.ea + (int64_t)min(m0 + r, g.M - 1) * g.KB : g.ew + (int64_t)min(n0 + r - BM, g.N - 1) * g.KB;
    sword[i] = scale4(srow[i], 0, g.KB);
  }
  auto ask_scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i) sword[i] = scale_word(srow[i] + min(kb, g.KB - 4));
  };
  auto put_scales = [&](int kb) {
    const int behind = g.KB >= 4 ? max(0, kb + 4 - g.KB) : 0;
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i)
      *reinterpret_cast<unsigned*>(&lds[2 * kBuf + ((kb >> 2 & 1) * (BM + BN) + i * NW * 64 + threadIdx.x) * 4]) =
          sword[i] >> (8 * behind);
  };
  const int fr = lane & 31, fg = lane >> 5;

  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x16{};

  // a fragment of half h of a block: lane l holds 32 of row l % 32's bytes, pieces 4 h + 2 (l / 32) and the next (the
  // order of k inside a block is free as long as both operands use the same)
  const int sw0 = fr >> 1 & 7, o0 = ((2 * fg) ^ sw0) * 16, o1 = ((2 * fg + 1) ^ sw0) * 16;
  const int ra = (wm * MI * 32 + fr) * kBlk, rw = (BM + wn * NI * 32 + fr) * kBlk;
  auto frag = [&](int kb, int h, int row) {
    const unsigned char* at = lds + (kb & 1) * kBuf + row;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(at + (o0 ^ h * 64)), hi = *reinterpret_cast<const i32x4*>(at + (o1 ^ h * 64));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  i32x8 fa[MI], w0[NI], w1[NI];
  int sa[MI], sw[NI], na[MI], nw[NI];
  auto fetch_scales = [&](int kb) {
    const unsigned char* at = lds + 2 * kBuf + (kb >> 2 & 1) * (BM + BN) * 4 + (kb & 3);
#pragma unroll
    for (int i = 0; i < MI; ++i) na[i] = at[((wm * MI + i) * 32 + fr) * 4];
#pragma unroll
    for (int j = 0; j < NI; ++j) nw[j] = at[(BM + (wn * NI + j) * 32 + fr) * 4];
  };
  // The products of one round on the fragments fa and w; each one, when it has served, is followed by its place
  // in half h of block kb under the products that follow.  A second round (h = 0: the next block's first
  // fragments) also asks for block kb + 1, a part behind each pair of products: asked for at once the loads
  // fill the vector memory's queue, and the products wait behind them.  The order is kept by hand: left alone,
  // the compiler moves each read down to its use.  (The last round reads fragments that nobody multiplies.)
  auto products = [&](const i32x8 (&w)[NI], i32x8 (&next)[NI], int kb, int h, auto&& meet) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[j], fa[i], acc[i][j], 0, 0, 0, sw[j], 0, sa[i]);
      __builtin_amdgcn_sched_barrier(0);
      if (i == 0) meet();
      if (h == 0) load(kb + 1, i * kLoads / MI, (i + 1) * kLoads / MI);
      fa[i] = frag(kb, h, ra + i * 32 * kBlk);
      if (i == 0) {
#pragma unroll
        for (int j = 0; j < NI; ++j) next[j] = frag(kb, h, rw + j * 32 * kBlk);
      }
      if (i == MI - 2 && h == 0) fetch_scales(kb);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  load(0, 0, kLoads);
  put_scales(0);
  load(1, 0, kLoads);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int j = 0; j < NI; ++j) w0[j] = frag(0, 0, rw + j * 32 * kBlk);
#pragma unroll
  for (int i = 0; i < MI; ++i) fa[i] = frag(0, 0, ra + i * 32 * kBlk);
  fetch_scales(0);
  for (int kb = 0; kb < g.KB; ++kb) {
#pragma unroll
    for (int i = 0; i < MI; ++i) sa[i] = na[i];
#pragma unroll
    for (int j = 0; j < NI; ++j) sw[j] = nw[j];
    // first half; the second's fragments are in the same LDS half
    products(w0, w1, kb, 1, [] {});
    // second half, and under its first products: this wave's loads have landed (block kb + 1's are the youngest)
    // and its reads of block kb are done; behind the barrier all waves' have
    products(w1, w0, kb + 1, 0, [&] {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if ((kb & 3) == 2 && kb + 2 < g.KB) put_scales(kb + 2);
      if ((kb & 3) == 1 && kb + 3 < g.KB) ask_scales(kb + 3);
    });
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS that is another workgroup's by then
  // A lane holds, for output column l % 32 of the instruction (m), rows 8 q + 4 (l / 32) + 0 .. 3 (n): eight bytes of
  // a row of the result.  The tile is put together in LDS, so that its rows leave in whole lines: stored from
  // the registers they cost the L2 twelve times the requests.  Piece c (16 bytes) of row r lies at c ^ (r % kPieces).
  asm volatile("s_barrier" ::: "memory");  // all waves are past their last reads of the operands
  constexpr int kPieces = BN / 8;
  static_assert(BM * BN * 2 <= 2 * kBuf && (kPieces & (kPieces - 1)) == 0, "the tile fits where the operands were");
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = (wn * NI + j) * 32 + 8 * q + 4 * fg;
      float add[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) add[e] = g.bias && n0 + n + e < g.N ? g.bias[n0 + n + e] : 0.f;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = (wm * MI + i) * 32 + fr;
        Pack<O, 4> y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y.v[e] = st1<O>(acc[i][j][4 * q + e] + add[e]);
        *reinterpret_cast<uint2*>(&lds[r * BN * 2 + (((n >> 3) ^ (r & (kPieces - 1))) << 4) + (n & 4) * 2]) =
            __builtin_bit_cast(uint2, y);
      }
    }
  __syncthreads();
  for (int u = threadIdx.x; u < BM * kPieces; u += NW * 64) {
    const int r = u / kPieces, c = u % kPieces, n = n0 + c * 8;
    if (m0 + r >= g.M || n >= g.N) continue;
    const uint4 y = *reinterpret_cast<const uint4*>(&lds[r * BN * 2 + ((c ^ (r & (kPieces - 1))) << 4)]);
    const Pack<O, 8> p = __builtin_bit_cast(Pack<O, 8>, y);
    O* to = (O*)g.out + (int64_t)(m0 + r) * g.ldo + n;
    if (n + 8 <= g.N) {
      stv<O, 8>(to, p);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + e < g.N) to[e] = p.v[e];
    }
  }
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
    hipLaunchKernelGGL((k_gemm8<2, 2, 2, 2, O>), dim3((unsigned)tiles(128, 128)), dim3(256), 0, s, g);
  } else {
    hipLaunchKernelGGL((k_gemm8<2, 4, 4, 2, O>), dim3((unsigned)tiles(256, 256)), dim3(512), 0, s, g);
  }
}

}  // namespace
}  // namespace seq
}  // namespace dssm

using namespace dssm::seq;

extern "C" int dssm_blocks8_matmul(const void* a, const void* ascale, const void* w, const void* wscale, int64_t M, int64_t N,
                                   int64_t K, const float* bias, void* out, int64_t ldo, int out_dtype, void* stream) {
  if (M < 0 || N < 0 || K <= 0 || M > (1 << 28) || N > (1 << 24) || K > (1 << 22) || ldo < N || (out_dtype != DSSM_BF16 && out_dtype != DSSM_F16) ||
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
