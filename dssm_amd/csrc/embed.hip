// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
// Lookup: y[i] = scale * table[ids[i]]; an id outside [0, V) reads nothing and gives a row of zeros.
//
// Gradient: dtable[v] = scale * sum over the positions i with ids[i] = v of dy[i].  Atomics into the
// table would add a hot token's rows in any order and one after the other; here the positions are first
// sorted by token (stable, so a token's positions stay in order), and the sorted list is cut into equal
// spans whatever the tokens: a span sums the runs of equal tokens it holds in fp32, stores the runs that
// lie whole inside it, and leaves the (at most two) cut ones as partial rows, which the last launch joins
// in span order.  The result does not depend on timing, and a token that fills half of the list is
// spread over as many workgroups as any other half.
//
// The sort is a least-significant-digit radix sort of (token, position) pairs, digits of at most 10 bits;
// a workgroup ranks a tile of 4096 pairs by wave ballots.  The rows of zeros that untouched tokens need
// are written by extra workgroups of the sort's launches, whose own work is latency.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "seq.h"

namespace dssm {
namespace seq {
namespace {

// ---- lookup ------------------------------------------------------------------------------------
// A row takes G lanes of 8 columns each (G a power of two up to 64, wider rows loop), a wave 64 / G rows;
// each lane has kLookRows rows' loads in flight, since a row is one dependent gather behind its id.
constexpr int kLookRows = 4;

template <typename T, typename O, typename I>
__global__ __launch_bounds__(256) void k_lookup(const T* __restrict__ table, int64_t ldt, const I* __restrict__ ids,
                                                int64_t n, int64_t V, int E, float scale, O* __restrict__ out,
                                                int lg) {
  const int G = 1 << lg, slot = threadIdx.x >> lg, slots = 256 >> lg;
  const int64_t r0 = (int64_t)blockIdx.x * slots * kLookRows + slot;
  for (int c = (threadIdx.x & (G - 1)) * 8; c < E; c += G * 8) {
    const int nv = E - c;
    float x[kLookRows][8];
    bool in[kLookRows];
#pragma unroll
    for (int j = 0; j < kLookRows; ++j) {
      const int64_t r = r0 + (int64_t)j * slots;
      const int64_t id = r < n ? (int64_t)ids[r] : -1;
      in[j] = id >= 0 && id < V;
      if (in[j]) {
        ld_row<T, 8>(table + id * ldt + c, nv, x[j]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[j][i] = 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < kLookRows; ++j) {
      const int64_t r = r0 + (int64_t)j * slots;
      if (r >= n) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[j][i] = in[j] ? x[j][i] * scale : 0.f;
      st_row<O, 8>(out + r * E + c, nv, x[j]);
    }
  }
}

// ---- sort --------------------------------------------------------------------------------------
constexpr int kTile = 4096;     // pairs a workgroup ranks
constexpr int kItems = 4;       // of them a thread's (1024 threads)
constexpr int kMaxBins = 1024;  // digits of at most 10 bits

struct Fill {  // the part of the gradient that a launch's extra workgroups clear
  float* p;
  int64_t n4;   // float4s of the part
  int tail;     // floats behind the last float4 (the last part only)
  int first;    // the first of the extra workgroups
};
__device__ __forceinline__ void fill_role(const Fill& f, int block, int blocks) {
  const int64_t step = (int64_t)blocks * blockDim.x;
  const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t i = (int64_t)block * blockDim.x + threadIdx.x; i < f.n4; i += step) reinterpret_cast<float4*>(f.p)[i] = z;
  if (block == 0 && threadIdx.x < f.tail) f.p[f.n4 * 4 + threadIdx.x] = 0.f;
}

// pair i of the first pass, straight from the ids: a token outside the table sorts behind all others
template <typename I>
__device__ __forceinline__ unsigned key_of(const I* ids, int64_t i, unsigned V) {
  const int64_t id = (int64_t)ids[i];
  return id >= 0 && id < (int64_t)V ? (unsigned)id : V;
}

// Ranks a tile's pairs by digit, stably: hist[w][d] becomes the number of the tile's pairs of digit d in
// waves before w, total[d] the tile's count, and rank[] each pair's place among its wave's pairs of its
// digit.  Wave w holds the pairs [256 w, 256 w + 256), lane-major within each of the four items.  A
// wave's lanes find the lanes of their own digit by one ballot per digit bit.  Every thread calls this.
__device__ __forceinline__ void rank_tile(const unsigned (&dig)[kItems], const bool (&live)[kItems], int bits,
                                          unsigned short (*hist)[kMaxBins], unsigned* total, int (&rank)[kItems]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits;
  for (int i = threadIdx.x; i < 16 * bins; i += 1024) hist[i >> bits][i & (bins - 1)] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    unsigned long long same = __ballot(live[j]);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long m = __ballot((dig[j] >> b) & 1u);
      same &= (dig[j] >> b) & 1u ? m : ~m;
    }
    const int before = __popcll(same & ((1ull << lane) - 1ull));
    volatile unsigned short* cell = &hist[w][dig[j]];
    rank[j] = 0;
    unsigned short base = 0;
    if (live[j]) base = *cell;
    __builtin_amdgcn_wave_barrier();
    if (live[j]) {
      rank[j] = base + before;
      if (before == 0) *cell = (unsigned short)(base + __popcll(same));
    }
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if ((int)threadIdx.x < bins) {
    unsigned run = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const unsigned v = hist[k][threadIdx.x];
      hist[k][threadIdx.x] = (unsigned short)run;
      run += v;
    }
    total[threadIdx.x] = run;
  }
  __syncthreads();
}

// exclusive sum over the workgroup's 1024 threads of one value each; s: 16 unsigneds
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned* s) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  unsigned x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  if (lane == 63) s[w] = x;
  __syncthreads();
  unsigned add = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) add += k < w ? s[k] : 0u;
  __syncthreads();
  return x - v + add;
}

struct SortLds {
  unsigned short hist[16][kMaxBins];
  unsigned total[kMaxBins];
  unsigned scan[16];
};

// The whole sort of one tile (n <= 4096) in one workgroup: the digits' passes move the pairs through LDS.
template <typename I>
__global__ __launch_bounds__(1024) void k_sort_one(const I* __restrict__ ids, int n, unsigned V, int bits, int passes,
                                                   unsigned* __restrict__ key, int* __restrict__ pos, Fill f) {
  __shared__ SortLds s;
  __shared__ unsigned lk[kTile];
  __shared__ unsigned short lp[kTile];
  if ((int)blockIdx.x >= f.first) return fill_role(f, blockIdx.x - f.first, gridDim.x - f.first);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  unsigned k[kItems];
  int p[kItems], rank[kItems];
  bool live[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = w * 256 + j * 64 + lane;
    live[j] = i < n;
    k[j] = live[j] ? key_of(ids, i, V) : 0u;
    p[j] = i;
  }
  for (int q = 0; q < passes; ++q) {
    unsigned dig[kItems];
#pragma unroll
    for (int j = 0; j < kItems; ++j) dig[j] = (k[j] >> (q * bits)) & ((1u << bits) - 1u);
    rank_tile(dig, live, bits, s.hist, s.total, rank);
    const bool bin = (int)threadIdx.x < (1 << bits);
    const unsigned base = block_scan(bin ? s.total[threadIdx.x] : 0u, s.scan);
    if (bin) s.total[threadIdx.x] = base;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j)
      if (live[j]) {
        const unsigned at = s.total[dig[j]] + s.hist[w][dig[j]] + rank[j];
        lk[at] = k[j];
        lp[at] = (unsigned short)p[j];
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kItems; ++j) {
      const int i = w * 256 + j * 64 + lane;
      if (live[j]) {
        k[j] = lk[i];
        p[j] = lp[i];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = w * 256 + j * 64 + lane;
    if (live[j]) {
      key[i] = k[j];
      pos[i] = p[j];
    }
  }
}

// A pass over many tiles: counts per tile and digit (cnt [tiles x 1 << bits]) ...
template <typename I>
__global__ __launch_bounds__(1024) void k_sort_count(const I* __restrict__ ids, const unsigned* __restrict__ kin,
                                                     int64_t n, unsigned V, int shift, int bits,
                                                     unsigned* __restrict__ cnt, Fill f) {
  __shared__ unsigned h[4][kMaxBins];  // four copies, so that a hot digit's adds do not all queue at one word
  if ((int)blockIdx.x >= f.first) return fill_role(f, blockIdx.x - f.first, gridDim.x - f.first);
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < 4 * bins; i += 1024) h[i >> bits][i & (bins - 1)] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = (int64_t)blockIdx.x * kTile + j * 1024 + threadIdx.x;
    if (i < n) {
      const unsigned k = kin ? kin[i] : key_of(ids, i, V);
      atomicAdd(&h[threadIdx.x & 3][(k >> shift) & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += 1024)
    cnt[(int64_t)blockIdx.x * bins + d] = h[0][d] + h[1][d] + h[2][d] + h[3][d];
}

// ... for many tiles (k_sort_place says when) the counts' running sums over the tiles, in place, and each
// digit's total into row `tiles`: one workgroup takes 64 digits, its 16 waves a sixteenth of the tiles each
__global__ __launch_bounds__(1024) void k_sort_sums(unsigned* __restrict__ cnt, int tiles, int bins) {
  __shared__ unsigned part[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
  const int per = (tiles + 15) / 16, t0 = min(w * per, tiles), t1 = min(t0 + per, tiles);
  unsigned sum = 0;
  if (d < bins)
    for (int t = t0; t < t1; ++t) sum += cnt[(int64_t)t * bins + d];
  part[w][lane] = sum;
  __syncthreads();
  unsigned run = 0, all = 0;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    run += k < w ? part[k][lane] : 0u;
    all += part[k][lane];
  }
  if (d < bins) {
    for (int t = t0; t < t1; ++t) {
      const unsigned v = cnt[(int64_t)t * bins + d];
      cnt[(int64_t)t * bins + d] = run;
      run += v;
    }
    if (w == 0) cnt[(int64_t)tiles * bins + d] = all;
  }
}

// ... and each tile's pairs to their places.  `summed`: cnt holds running sums (k_sort_sums); otherwise a
// thread adds up its digit's counts itself, all tiles' for the digit's start and the earlier ones' for the
// tile's place in it.
template <typename I>
__global__ __launch_bounds__(1024) void k_sort_place(const I* __restrict__ ids, const unsigned* __restrict__ kin,
                                                     const int* __restrict__ pin, int64_t n, unsigned V, int shift,
                                                     int bits, const unsigned* __restrict__ cnt, int tiles, int summed,
                                                     unsigned* __restrict__ kout, int* __restrict__ pout, Fill f) {
  __shared__ SortLds s;
  if ((int)blockIdx.x >= f.first) return fill_role(f, blockIdx.x - f.first, gridDim.x - f.first);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits, me = blockIdx.x;
  unsigned k[kItems], dig[kItems];
  int p[kItems], rank[kItems];
  bool live[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = (int64_t)me * kTile + w * 256 + j * 64 + lane;
    live[j] = i < n;
    k[j] = !live[j] ? 0u : kin ? kin[i] : key_of(ids, i, V);
    p[j] = !live[j] ? 0 : kin ? pin[i] : (int)i;
    dig[j] = (k[j] >> shift) & (bins - 1);
  }
  unsigned all = 0, before = 0;
  if ((int)threadIdx.x < bins) {
    const unsigned* c = cnt + threadIdx.x;
    if (summed) {
      before = c[(int64_t)me * bins];
      all = c[(int64_t)tiles * bins];
    } else {
      int t = 0;
      for (; t + 16 <= tiles; t += 16) {
        unsigned v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = c[(t + i) * bins];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          all += v[i];
          before += t + i < me ? v[i] : 0u;
        }
      }
      for (; t < tiles; ++t) {
        const unsigned v = c[t * bins];
        all += v;
        before += t < me ? v : 0u;
      }
    }
  }
  rank_tile(dig, live, bits, s.hist, s.total, rank);
  const unsigned start = block_scan(all, s.scan) + before;
  if ((int)threadIdx.x < bins) s.total[threadIdx.x] = start;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j)
    if (live[j]) {
      const unsigned at = s.total[dig[j]] + s.hist[w][dig[j]] + rank[j];
      kout[at] = k[j];
      pout[at] = p[j];
    }
}

// ---- sums --------------------------------------------------------------------------------------
// Span s of the sorted list is [s S, (s + 1) S).  G lanes of 8 columns walk it, eight rows' loads in
// flight.  part[2 s] takes the run that came in from span s - 1, part[2 s + 1] the run that goes on into
// span s + 1 and starts in s; a run that fills a whole span and goes on both ways counts as incoming.
constexpr int kSpan = 32;

template <typename T>
__global__ __launch_bounds__(256) void k_grad_spans(const unsigned* __restrict__ key, const int* __restrict__ pos,
                                                    int64_t n, unsigned V, const T* __restrict__ dy, int64_t lddy,
                                                    int E, float scale, float* __restrict__ dtable,
                                                    float* __restrict__ part, int lg) {
  const int G = 1 << lg;
  const int64_t s = (int64_t)blockIdx.x * (256 >> lg) + (threadIdx.x >> lg);
  const int64_t i0 = s * kSpan, i1 = min(i0 + kSpan, n);
  if (i0 >= n) return;
  const unsigned none = 0xffffffffu;
  const unsigned prev = i0 ? key[i0 - 1] : none, next = i1 < n ? key[i1] : none;
  for (int c = (threadIdx.x & (G - 1)) * 8; c < E; c += G * 8) {
    const int nv = E - c;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    unsigned cur = key[i0];
    bool incoming = cur == prev;
    auto flush = [&](bool outgoing) {
      if (cur >= V) return;
      if (!incoming && !outgoing) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = acc[i] * scale;
        st_row<float, 8>(dtable + (int64_t)cur * E + c, nv, y);
      } else {
        st_row<float, 8>(part + (2 * s + (incoming ? 0 : 1)) * E + c, nv, acc);
      }
    };
    for (int64_t i = i0; i < i1; i += 8) {
      unsigned k[8];
      float x[8][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        k[j] = i + j < i1 ? key[i + j] : none;
        if (k[j] < V) {
          ld_row<T, 8>(dy + (int64_t)pos[i + j] * lddy + c, nv, x[j]);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) x[j][q] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (k[j] == none) break;
        if (k[j] != cur) {
          flush(false);
          cur = k[j];
          incoming = false;
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] = 0.f;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += x[j][q];
      }
    }
    flush(cur == next);
  }
}

// Joins the runs that cross spans: the lanes of span s own the run that starts in s and goes on.  A run
// of few spans is summed at once; a longer one is left to the whole workgroup, whose groups take equal
// stretches of it and join them through LDS, so that half a list of one token is no chain of loads.
constexpr int kShort = 8;

__global__ __launch_bounds__(256) void k_grad_join(const unsigned* __restrict__ key, int64_t n, int64_t spans,
                                                   unsigned V, int E, float scale, const float* __restrict__ part,
                                                   float* __restrict__ dtable, int lg) {
  const int G = 1 << lg, groups = 256 >> lg, grp = threadIdx.x >> lg, lane = threadIdx.x & (G - 1);
  __shared__ float red[256 * 8];
  __shared__ int64_t longs[256];
  __shared__ int nlong;
  if (threadIdx.x == 0) nlong = 0;
  __syncthreads();
  const int64_t s = (int64_t)blockIdx.x * groups + grp;
  const int64_t end = (s + 1) * kSpan;  // the next span's first entry
  const unsigned cur = end < n ? key[end] : V;
  // the run starts in s: its token is not also the one that came in and fills the span from its start
  const bool head = cur < V && key[end - 1] == cur && (key[s * kSpan] != cur || s == 0 || key[s * kSpan - 1] != cur);
  if (head) {
    // the last span that the run reaches
    int64_t last = s + 1;
    while (last - s <= kShort && (last + 1) * kSpan < n && key[(last + 1) * kSpan] == cur) ++last;
    if (last - s <= kShort) {
      for (int c = lane * 8; c < E; c += G * 8) {
        const int nv = E - c;
        float acc[8], x[8];
        ld_row<float, 8>(part + (2 * s + 1) * E + c, nv, acc);
        for (int64_t t = s + 1; t <= last; ++t) {
          ld_row<float, 8>(part + 2 * t * E + c, nv, x);
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] += x[q];
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] *= scale;
        st_row<float, 8>(dtable + (int64_t)cur * E + c, nv, acc);
      }
    } else if (lane == 0) {
      longs[atomicAdd(&nlong, 1)] = s;
    }
  }
  __syncthreads();
  for (int j = 0; j < nlong; ++j) {
    const int64_t h = longs[j];
    const unsigned tok = key[(h + 1) * kSpan];
    // the run's last span: the last one whose first entry is still this token (the list is sorted)
    int64_t lo = h + 1, hi = spans - 1;
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) / 2;
      if (key[mid * kSpan] == tok) lo = mid;
      else hi = mid - 1;
    }
    const int64_t cnt = lo - h, per = (cnt + groups - 1) / groups;
    const int64_t a = min(h + 1 + grp * per, lo + 1), b = min(a + per, lo + 1);
    for (int c0 = 0; c0 < E; c0 += G * 8) {
      const int c = c0 + lane * 8, nv = E - c;
      float acc[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] = 0.f;
      if (nv > 0) {
        int64_t t = a;
        for (; t + 4 <= b; t += 4) {
          float x[4][8];
#pragma unroll
          for (int u = 0; u < 4; ++u) ld_row<float, 8>(part + 2 * (t + u) * E + c, nv, x[u]);
#pragma unroll
          for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int q = 0; q < 8; ++q) acc[q] += x[u][q];
        }
        for (; t < b; ++t) {
          float x[8];
          ld_row<float, 8>(part + 2 * t * E + c, nv, x);
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[q] += x[q];
        }
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) red[q * 256 + threadIdx.x] = acc[q];
      __syncthreads();
      if (grp == 0 && nv > 0) {
        float x[8];
        ld_row<float, 8>(part + (2 * h + 1) * E + c, nv, x);
        for (int g = 0; g < groups; ++g)
#pragma unroll
          for (int q = 0; q < 8; ++q) x[q] += red[q * 256 + (g << lg) + lane];
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] *= scale;
        st_row<float, 8>(dtable + (int64_t)tok * E + c, nv, x);
      }
      __syncthreads();
    }
  }
}

int lanes_log2(int E) {  // log2 of the lanes a row takes: 8 columns each, at most a wave
  int lg = 0;
  while (lg < 6 && (8 << lg) < E) ++lg;
  return lg;
}

// Workspace of a gradient: pairs twice, the tiles' digit counts, the spans' partial rows.
struct GradWs {
  int bits, passes;
  int64_t tiles, spans;
  size_t key0, pos0, key1, pos1, cnt, part, bytes;
};
GradWs grad_ws(int64_t n, int64_t V, int E) {
  GradWs g{};
  int bits = 1;
  while (((int64_t)1 << bits) <= V) ++bits;  // keys 0 .. V
  g.passes = (bits + 9) / 10;
  g.bits = (bits + g.passes - 1) / g.passes;
  g.tiles = (n + kTile - 1) / kTile;
  g.spans = (n + kSpan - 1) / kSpan;
  size_t at = 0;
  auto take = [&](size_t b) {
    const size_t o = at;
    at += (b + 255) / 256 * 256;
    return o;
  };
  g.key0 = take(4 * n);
  g.pos0 = take(4 * n);
  g.key1 = take(4 * n);
  g.pos1 = take(4 * n);
  g.cnt = take(4 * (size_t)(g.tiles + 1) << g.bits);
  g.part = take((size_t)g.spans * 2 * E * 4);
  g.bytes = at;
  return g;
}
bool grad_dims_ok(int64_t n, int64_t V, int E) {
  return n >= 0 && n < ((int64_t)1 << 31) - kTile && V > 0 && V < ((int64_t)1 << 30) && E > 0 && E <= (1 << 20);
}

// More tiles than this have their counts summed by a launch of their own: a workgroup's own sums read
// tiles x bins counts, 16 loads in flight.
constexpr int kOwnSums = 64;

template <typename I>
int run_grad(const void* dy, int dtype, int64_t lddy, const I* ids, int64_t n, int64_t V, int E, float scale, float* dtable,
             char* ws, hipStream_t s) {
  const GradWs g = grad_ws(n, V, E);
  unsigned* key[2] = {(unsigned*)(ws + g.key0), (unsigned*)(ws + g.key1)};
  int* pos[2] = {(int*)(ws + g.pos0), (int*)(ws + g.pos1)};
  unsigned* cnt = (unsigned*)(ws + g.cnt);
  float* part = (float*)(ws + g.part);
  const bool one = n <= kTile;
  // the table's zeros, an equal share to each of the sort's launches
  const int64_t total = V * E, all4 = total / 4;
  const int shares = one ? 1 : 2 * g.passes;
  int share = 0;
  auto part_of = [&](int own, int* grid) {
    Fill f{};
    const int64_t a = all4 * share / shares, b = all4 * (share + 1) / shares;
    f.p = dtable + a * 4;
    f.n4 = b - a;
    f.tail = share + 1 == shares ? (int)(total - all4 * 4) : 0;
    f.first = own;
    const int extra = f.n4 || f.tail ? (int)std::min<int64_t>(512, (f.n4 + 4095) / 4096 + 1) : 0;
    *grid = own + extra;
    ++share;
    return f;
  };
  int grid = 0, side = 0;
  if (n == 0) {
    return seq_status(zero_bytes_async(dtable, (size_t)total * 4, s));
  } else if (one) {
    const Fill f = part_of(1, &grid);
    hipLaunchKernelGGL(k_sort_one<I>, dim3(grid), dim3(1024), 0, s, ids, (int)n, (unsigned)V, g.bits, g.passes, key[0],
                       pos[0], f);
  } else {
    const int tiles = (int)g.tiles, summed = tiles > kOwnSums;
    for (int q = 0; q < g.passes; ++q) {
      const unsigned* kin = q ? key[side] : nullptr;
      const int* pin = q ? pos[side] : nullptr;
      if (q) side ^= 1;
      Fill f = part_of(tiles, &grid);
      hipLaunchKernelGGL(k_sort_count<I>, dim3(grid), dim3(1024), 0, s, ids, kin, n, (unsigned)V, q * g.bits, g.bits, cnt,
                         f);
      if (summed)
        hipLaunchKernelGGL(k_sort_sums, dim3(((1 << g.bits) + 63) / 64), dim3(1024), 0, s, cnt, tiles, 1 << g.bits);
      f = part_of(tiles, &grid);
      hipLaunchKernelGGL(k_sort_place<I>, dim3(grid), dim3(1024), 0, s, ids, kin, pin, n, (unsigned)V, q * g.bits, g.bits,
                         cnt, tiles, summed, key[side], pos[side], f);
    }
  }
  const int lg = lanes_log2(E), groups = 256 >> lg;
  const unsigned blocks = (unsigned)((g.spans + groups - 1) / groups);
  by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    hipLaunchKernelGGL(k_grad_spans<T>, dim3(blocks), dim3(256), 0, s, key[side], pos[side], n, (unsigned)V, (const T*)dy,
                       lddy, E, scale, dtable, part, lg);
  });
  if (g.spans > 1)
    hipLaunchKernelGGL(k_grad_join, dim3(blocks), dim3(256), 0, s, key[side], n, g.spans, (unsigned)V, E, scale, part,
                       dtable, lg);
  return seq_status(hipGetLastError());
}

}  // namespace
}  // namespace seq
}  // namespace dssm

using namespace dssm::seq;

extern "C" int dssm_embedding_lookup(const void* table, int dtype, int64_t ldt, int64_t V, int E, const void* ids,
                                     int ids64, int64_t n, float scale, void* out, int out_dtype, void* stream) {
  if (!table || !seq_dtype(dtype) || !seq_dtype(out_dtype) || V <= 0 || E <= 0 || ldt < E || n < 0 ||
      (n > 0 && (!ids || !out)))
    return dssm::report_error(DSSM_E_INVALID, "embedding_lookup: bad argument");
  if (n == 0) return DSSM_OK;
  const int lg = lanes_log2(E);
  const int64_t rows = (int64_t)(256 >> lg) * kLookRows, blocks = (n + rows - 1) / rows;
  if (blocks > 0x7fffffff) return dssm::report_error(DSSM_E_UNSUPPORTED, "embedding_lookup: too many ids");
  by_dtype(dtype, [&](auto t) {
    by_dtype(out_dtype, [&](auto o) {
      using T = decltype(t);
      using O = decltype(o);
      if (ids64)
        hipLaunchKernelGGL((k_lookup<T, O, int64_t>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                           (const T*)table, ldt, (const int64_t*)ids, n, V, E, scale, (O*)out, lg);
      else
        hipLaunchKernelGGL((k_lookup<T, O, int32_t>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                           (const T*)table, ldt, (const int32_t*)ids, n, V, E, scale, (O*)out, lg);
    });
  });
  return seq_status(hipGetLastError());
}

extern "C" size_t dssm_embedding_grad_ws_bytes(int64_t n, int64_t V, int E) {
  return grad_dims_ok(n, V, E) ? grad_ws(n, V, E).bytes + 256 : 0;
}

extern "C" int dssm_embedding_grad(const void* dy, int dtype, int64_t lddy, const void* ids, int ids64, int64_t n,
                                   int64_t V, int E, float scale, float* dtable, void* ws, size_t ws_bytes, void* stream) {
  if (!seq_dtype(dtype) || !grad_dims_ok(n, V, E) || lddy < E || !dtable || (n > 0 && (!dy || !ids || !ws)))
    return dssm::report_error(DSSM_E_INVALID, "embedding_grad: bad argument");
  if ((uintptr_t)dtable % 16 || (uintptr_t)ws % 16)
    return dssm::report_error(DSSM_E_INVALID, "embedding_grad: the gradient and the workspace are 16-byte aligned");
  if (n > 0 && ws_bytes < grad_ws(n, V, E).bytes)
    return dssm::report_error(DSSM_E_INVALID, "embedding_grad: workspace too small (dssm_embedding_grad_ws_bytes)");
  return ids64 ? run_grad(dy, dtype, lddy, (const int64_t*)ids, n, V, E, scale, dtable, (char*)ws, (hipStream_t)stream)
               : run_grad(dy, dtype, lddy, (const int32_t*)ids, n, V, E, scale, dtable, (char*)ws, (hipStream_t)stream);
}
