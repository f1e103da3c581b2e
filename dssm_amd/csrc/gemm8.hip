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
// A group of WM x WN waves computes (WM MI 32) x (WN NI 32) outputs with v_mfma_scale_f32_32x32x64; SK groups of a
// workgroup take a share of K each, in LDS of their own, and meet at the end.
//
// Both operands go from memory straight to LDS, 16 bytes a lane, a block of 128 columns at a time into one of D
// buffers; whole 128-byte lines, because the two halves of a line that are asked for apart meet as one pending
// line in the vector cache and stall it.  A block is multiplied in two rounds of 64 columns, and a round
// multiplies fragments that are in registers already while it reads the next round's: when a block's second
// round begins, nobody needs its buffer any more, and the block D further on is asked for, 2 (D - 1) rounds of
// products before its first fragment is read.  D is 2 for the large tiles (256 x 256: 128 KB of LDS, 2048 cycles
// of the matrix units ahead); 64 x 64 and 32 x 32, which run where there are few tiles and the memory's latency is
// all there is to a block, take 4.
//
// Measured, 8192 x 4096 x 8192: 227 to 233 us a pass among others (224 to 251 under a trace), 2.4 PFLOP/s, 92 to 94 %
// of the library's rate for one scale a tensor (2.56); the matrix units are busy 62 % of the time at 1.85 GHz, to
// which their power brings the clock down.  Without the loads the same loop takes 184 us, always from the same two
// blocks 217.  8192 x 8192 x 4096: 2.3 PFLOP/s.
//
// A row's 128 bytes are eight 16-byte pieces; piece p of row r lies at p ^ (r >> 1 & 7).  A 16-byte read serves
// sixteen lanes a cycle: lanes 0-3, 12-15, 20-23 and 24-27 of a half wave, then the others (found with the
// conflict counter, which reads zero); of these rows no two of the same parity have the same r >> 1 & 7, so
// they cover all 64 banks.  The direct load writes LDS in lane order, so the permutation is applied to the
// address that each lane loads from.
template <int WM, int WN, int MI, int NI, int D, int SK, typename O>
__global__ __launch_bounds__(WM * WN * SK * 64, WM * WN * SK == 8 ? 2 : 1) void k_gemm8(Gemm8Args g) {
  constexpr int BM = WM * MI * 32, BN = WN * NI * 32, NW = WM * WN, kLoads = (BM + BN) / 8 / NW;  // (of one group)
  static_assert(kLoads * 8 * NW == BM + BN && BM % 8 == 0, "every wave loads the same number of 8-row stripes");
  // Scales.  The large tiles keep a word a row, four blocks' bytes, which a thread loads for a row at a time.  The
  // small ones send a byte a row and block the operands' way (the load widens it to a word): no wait of its own,
  // for more work in the vector cache, which they leave idle.
  constexpr bool kWords = D == 2;
  constexpr int kScaleRows = (BM + BN) / (NW * 64) ? (BM + BN) / (NW * 64) : 1;  // a thread's
  static_assert((BM + BN) % 64 == 0 && (kScaleRows * NW * 64 == BM + BN || !kWords), "a row's scales are loaded by one thread");
  // D blocks, then the scales.  One object: of two the compiler knows that they are two, tells the direct loads
  // apart by that, and puts a wait for all of them in front of every read.
  constexpr int kBuf = (BM + BN) * kBlk, kScale = (BM + BN) * 4, kGroup = D * kBuf + D * kScale;
  static_assert(SK == 1 || !kWords, "the words are put by the whole workgroup");
  __shared__ __attribute__((aligned(16))) unsigned char shared[SK * kGroup];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int grp = SK == 1 ? 0 : wave / NW, wv = SK == 1 ? wave : wave % NW, wm = wv % WM, wn = wv / WM;
  const int thread = SK == 1 ? threadIdx.x : threadIdx.x % (NW * 64);
  unsigned char* const lds = shared + grp * kGroup;
  // this group's blocks: `per` from k0 on, of which the first `own` are its own (the walk is as long for every group)
  const int per = SK == 1 ? g.KB : (g.KB + SK - 1) / SK, k0 = grp * per, own = g.KB - k0;
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
    const unsigned at = (unsigned)min(k0 + kb, g.KB - 1) * kBlk;
#pragma unroll
    for (int i = from; i < to; ++i)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(base[i] + at + off[i]),
                                       (__attribute__((address_space(3))) unsigned*)&lds[(kb & (D - 1)) * kBuf + (wv + i * NW) * 1024],
                                       16, 0, 0);
  };
  // Words: asked for three blocks ahead and written to LDS two ahead (the last word of a row starts at KB - 4 and
  // is shifted down).  Bytes: the waves that have a row load block kb + D's with its operands.
  const unsigned char* srow[kScaleRows];
  unsigned sword[kScaleRows];
#pragma unroll
  for (int i = 0; i < kScaleRows; ++i) {
    const int r = i * NW * 64 + thread;
    srow[i] = r < BM ? g.ea + (int64_t)min(m0 + r, g.M - 1) * g.KB : g.ew + (int64_t)min(n0 + r - BM, g.N - 1) * g.KB;
    if (kWords) sword[i] = scale4(srow[i], 0, g.KB);
  }
  auto ask_scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i) sword[i] = scale_word(srow[i] + min(kb, g.KB - 4));
  };
  auto put_scales = [&](int kb) {
    const int behind = g.KB >= 4 ? max(0, kb + 4 - g.KB) : 0;
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i)
      *reinterpret_cast<unsigned*>(&lds[D * kBuf + (kb >> 2 & 1) * kScale + (i * NW * 64 + thread) * 4]) =
          sword[i] >> (8 * behind);
  };
  auto load_scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < kScaleRows; ++i)
      if ((i * NW + wv) * 64 < BM + BN)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(srow[i] + min(k0 + kb, g.KB - 1)),
                                         (__attribute__((address_space(3))) unsigned*)&lds[D * kBuf + (kb & (D - 1)) * kScale +
                                                                                            (i * NW + wv) * 256],
                                         1, 0, 0);
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
    const unsigned char* at = lds + (kb & (D - 1)) * kBuf + row;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(at + (o0 ^ h * 64)), hi = *reinterpret_cast<const i32x4*>(at + (o1 ^ h * 64));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  i32x8 fa[MI], w0[NI], w1[NI];
  int sa[MI], sw[NI], na[MI], nw[NI];
  int mine = -1;  // 0: the block is behind this group's last and counts as zeros (a NaN in it is in the result anyway)
  auto fetch_scales = [&](int kb) {
    const unsigned char* at = lds + D * kBuf + (kWords ? (kb >> 2 & 1) * kScale + (kb & 3) : (kb & (D - 1)) * kScale);
#pragma unroll
    for (int i = 0; i < MI; ++i) na[i] = at[((wm * MI + i) * 32 + fr) * 4];
#pragma unroll
    for (int j = 0; j < NI; ++j) nw[j] = at[(BM + (wn * NI + j) * 32 + fr) * 4];
  };
  // The products of one round on the fragments fa and w; each one, when it has served, is followed by its place
  // in half h of block kb under the products that follow.  A second round (h = 0: the next block's first
  // fragments) also asks for block kb + D - 1, a part behind each pair of products: asked for at once the loads
  // fill the vector memory's queue, and the products wait behind them.  The order is kept by hand: left alone,
  // the compiler moves each read down to its use.  (The last round reads fragments that nobody multiplies.)
  auto products = [&](const i32x8 (&w)[NI], i32x8 (&next)[NI], int kb, int h, auto&& meet) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      if constexpr (SK > 1) fa[i] &= mine;
#pragma unroll
      for (int j = 0; j < NI; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[j], fa[i], acc[i][j], 0, 0, 0, sw[j], 0, sa[i]);
      __builtin_amdgcn_sched_barrier(0);
      if (i == 0) meet();
      if (h == 0) load(kb + D - 1, i * kLoads / MI, (i + 1) * kLoads / MI);
      fa[i] = frag(kb, h, ra + i * 32 * kBlk);
      if (i == 0) {
#pragma unroll
        for (int j = 0; j < NI; ++j) next[j] = frag(kb, h, rw + j * 32 * kBlk);
      }
      if (i == (MI > 1 ? MI - 2 : 0) && h == 0) fetch_scales(kb);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int kb = 0; kb < D; ++kb) {
    load(kb, 0, kLoads);
    if (!kWords) load_scales(kb);
  }
  if (kWords) put_scales(0);
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int j = 0; j < NI; ++j) w0[j] = frag(0, 0, rw + j * 32 * kBlk);
#pragma unroll
  for (int i = 0; i < MI; ++i) fa[i] = frag(0, 0, ra + i * 32 * kBlk);
  fetch_scales(0);
  for (int kb = 0; kb < per; ++kb) {
    if constexpr (SK > 1) mine = kb < own ? -1 : 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) sa[i] = na[i];
#pragma unroll
    for (int j = 0; j < NI; ++j) sw[j] = nw[j];
    // first half; the second's fragments are in the same LDS half
    products(w0, w1, kb, 1, [] {});
    // second half, and under its first products: this wave's loads of block kb + 1 have landed (all but the D - 2
    // younger blocks'; a wave without scale rows of its own has no more than kLoads of them a block) and its reads
    // of block kb are done; behind the barrier all waves' have
    products(w1, w0, kb + 1, 0, [&] {
      if constexpr (kWords) {
        static_assert(D == 2, "nothing younger is in flight");
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if ((kb & 3) == 2 && kb + 2 < g.KB) put_scales(kb + 2);
        if ((kb & 3) == 1 && kb + 3 < g.KB) ask_scales(kb + 3);
      } else {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((D - 2) * kLoads) : "memory");
        load_scales(kb + D);
      }
    });
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS that is another workgroup's by then
  // A lane holds, for output column l % 32 of the instruction (m), rows 8 q + 4 (l / 32) + 0 .. 3 (n): eight bytes of
  // a row of the result.  The tile is put together in LDS, so that its rows leave in whole lines: stored from
  // the registers they cost the L2 twelve times the requests.  Piece c (16 bytes) of row r lies at c ^ (r % kPieces).
  asm volatile("s_barrier" ::: "memory");  // all waves are past their last reads of the operands
  constexpr int kTile = BM * BN * 2;
  if constexpr (SK > 1) {  // the groups' sums, in their order
    static_assert(kTile + (SK - 1) * BM * BN * 4 <= SK * kGroup, "they fit behind the tile");
    f32x4* const sums = reinterpret_cast<f32x4*>(shared + kTile);
    if (grp) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            sums[((((grp - 1) * NW + wv) * MI * NI + i * NI + j) * 4 + q) * 64 + lane] =
                f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    }
    __syncthreads();
    if (!grp) {
#pragma unroll
      for (int k = 0; k < SK - 1; ++k)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 v = sums[(((k * NW + wv) * MI * NI + i * NI + j) * 4 + q) * 64 + lane];
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += v[e];
            }
    }
  }
  constexpr int kPieces = BN / 8;
  static_assert(kTile <= D * kBuf && (kPieces & (kPieces - 1)) == 0, "the tile fits where the operands were");
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (grp) break;
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
        *reinterpret_cast<uint2*>(&shared[r * BN * 2 + (((n >> 3) ^ (r & (kPieces - 1))) << 4) + (n & 4) * 2]) =
            __builtin_bit_cast(uint2, y);
      }
    }
  __syncthreads();
  for (int u = threadIdx.x; u < BM * kPieces; u += NW * SK * 64) {
    const int r = u / kPieces, c = u % kPieces, n = n0 + c * 8;
    if (m0 + r >= g.M || n >= g.N) continue;
    const uint4 y = *reinterpret_cast<const uint4*>(&shared[r * BN * 2 + ((c ^ (r & (kPieces - 1))) << 4)]);
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
// The weights are read once, straight into registers: a workgroup takes 16 of their rows against 16 MT rows of a,
// its eight waves a stretch of the blocks each, kDepth blocks' loads in flight; the waves' sums meet in LDS in
// wave order.  A lane takes the 16-byte pieces l / 16 and l / 16 + 4 of a row's 128 bytes, so that each load
// instruction reads whole halves of lines.
template <int MT, typename O>
__global__ __launch_bounds__(512) void k_gemm8_rows(Gemm8Args g) {
  constexpr int NW = 8, kDepth = 4;
  __shared__ f32x4 part[NW][MT][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, fr = lane & 15, fp = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
  const int64_t Kp = (int64_t)g.KB * kBlk;
  const int64_t nr = min(n0 + fr, g.N - 1);
  const unsigned char* w = g.w + nr * Kp + fp * 16;
  const unsigned char* ew = g.ew + nr * g.KB;
  const unsigned char* a[MT];
  const unsigned char* ea[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = min(m0 + i * 16 + fr, g.M - 1);
    a[i] = g.a + m * Kp + fp * 16;
    ea[i] = g.ea + m * g.KB;
  }
  auto frag = [](const unsigned char* p) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(p), hi = *reinterpret_cast<const i32x4*>(p + 64);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int per = (g.KB + NW - 1) / NW, k0 = min(wv * per, g.KB), k1 = min(k0 + per, g.KB);
  for (int kb = k0; kb < k1; kb += kDepth) {
    i32x8 fw[kDepth], fa[kDepth][MT];
    unsigned sa[MT];
    unsigned sw = scale4(ew, kb, g.KB);
#pragma unroll
    for (int i = 0; i < MT; ++i) sa[i] = scale4(ea[i], kb, g.KB);
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (kb + d < k1) {
        fw[d] = frag(w + (int64_t)(kb + d) * kBlk);
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[d][i] = frag(a[i] + (int64_t)(kb + d) * kBlk);
      }
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
      if (kb + d < k1) {
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i] = mfma8(fw[d], fa[d][i], acc[i], (int)(sw >> (8 * d)), (int)(sa[i] >> (8 * d)));
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

// Which tile: the least of what each would take for a block of 128 columns, in units of 10 ns, from how many rounds
// of workgroups its tiles fill the 256 compute units.  Measured (N = K = 4096 and neighbours): 64 x 64, two
// workgroups a unit, 0.37 us a block up to one a unit, 0.61 a full round; 128 x 128, two a unit, 0.81 and 1.30;
// 256 x 256, one a unit, 1.85 (8192 x 4096 x 8192 in 64 x 64 tiles takes twice its time, 512 x 4096 x 4096 in
// 256 x 256 tiles 42 us against 20).
int tile_of(int64_t t64, int64_t t128, int64_t t256) {
  const int64_t c64 = t64 <= 256 ? 37 : (t64 + 511) / 512 * 61, c128 = t128 <= 256 ? 81 : (t128 + 511) / 512 * 130,
                c256 = (t256 + 255) / 256 * 185;
  return c64 <= c128 && c64 <= c256 ? 64 : c128 <= c256 ? 128 : 256;
}

template <typename O>
int run_gemm8(const Gemm8Args& g, hipStream_t s) {
  const auto tiles = [&](int b) { return (int64_t)((g.M + b - 1) / b) * ((g.N + b - 1) / b); };
  if (tiles(64) > 0x7fffffff) return dssm::report_error(DSSM_E_UNSUPPORTED, "blocks8_matmul: too many outputs");
  const int tile = tile_of(tiles(64), tiles(128), tiles(256));
  // Rows against rows where that takes a workgroup a compute unit at most: the waves of a workgroup share K (7 x 4096 x
  // 4096: 5.9 us (6.1 to 6.8 traced) against 8.5 in 32 x 32 tiles, 32 x 256 x 8192 10.0 against 11.6, 100 x 300 x 200 2.9 against 4.3);
  // 32 rows at a time for 17 to 32 of them (32 x 4096 x 4096: 8.8 us, 10.7 sixteen at a time, 9.1 in tiles).  With more
  // workgroups, each of which reads its rows of a again, tiles are faster (32 x 8192 x 1024 5.6 us against 8.4, 16 x
  // 12288 x 4096 12.3 against 14.6).
  const int64_t n16 = (g.N + 15) / 16, m16 = (g.M + 15) / 16;
  if (n16 * m16 <= 256) {
    hipLaunchKernelGGL((k_gemm8_rows<1, O>), dim3((unsigned)n16, (unsigned)m16), dim3(512), 0, s, g);
  } else if (g.M <= 32 && n16 <= 256) {
    hipLaunchKernelGGL((k_gemm8_rows<2, O>), dim3((unsigned)n16, 1), dim3(512), 0, s, g);
  } else if (tiles(32) <= 256 && g.KB >= 8) {
    // A tile's time is what its compute unit can load: 32 x 32 while these find a unit each, and two blocks for each
    // of the four groups of waves that share K (64 x 4096 x 4096 9.3 us, 11.8 in 64 x 64 tiles; 256 x 1024 x 8192
    // 13.1 and 19.6; of two rounds 12.0 and 12.1; 64 x 4096 x 384 4.6 and 4.3)
    hipLaunchKernelGGL((k_gemm8<1, 1, 1, 1, 4, 4, O>), dim3((unsigned)tiles(32)), dim3(256), 0, s, g);
  } else if (tile == 64) {
    hipLaunchKernelGGL((k_gemm8<2, 2, 1, 1, 4, 1, O>), dim3((unsigned)tiles(64)), dim3(256), 0, s, g);
  } else if (tile == 128) {
    hipLaunchKernelGGL((k_gemm8<2, 2, 2, 2, 2, 1, O>), dim3((unsigned)tiles(128)), dim3(256), 0, s, g);
  } else {
    hipLaunchKernelGGL((k_gemm8<2, 4, 4, 2, 2, 1, O>), dim3((unsigned)tiles(256)), dim3(512), 0, s, g);
  }
  return seq_status(hipGetLastError());
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
  return out_dtype == DSSM_BF16 ? run_gemm8<u16>(g, (hipStream_t)stream) : run_gemm8<f16s>(g, (hipStream_t)stream);
}
