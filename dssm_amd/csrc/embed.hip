// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
// Lookup: y[i] = scale * table[ids[i]]; an id outside [0, V) reads nothing and gives a row of zeros.
//
// Gradient: dtable[v] = scale * sum over the positions i with ids[i] = v of dy[i].  Atomics into the
// table would add a hot token's rows in any order and one after the other; here the positions are first
// sorted by token (stable, so a token's positions stay in order), and the sorted list is cut into equal
// spans whatever the tokens: a span sums the runs of equal tokens it holds in fp32, stores the runs that
// lie whole inside it, and leaves the (at most two) cut ones as partial rows, which the last launch joins.  Eight
// positions are added in their order; their sums, and spans', in a fixed one (one after the other, or by doubling where
// there are many).  The result does not depend on timing, and a token that fills half of the list is
// spread over as many workgroups as any other half.
//
// The sort is a least-significant-digit radix sort of (token, position) pairs, digits of at most 10 bits;
// a workgroup ranks a tile of 1024 or 4096 pairs by wave ballots.  The rows of zeros that untouched tokens need
// are written by extra workgroups of the sort's launches, whose own work is latency.
//
// Measured, 196608 tokens of 128 columns over 21128 words (log-uniform; 62 MB that must move, 12.7 us at the
// rate of a large copy): lookup fp32 -> bf16 14.3 us, 4.3 TB/s; gradient of bf16 rows 47 us in six launches:
// per digit count 3.2 and place 8.8 us (loads, tile sums and ranks one behind the other: latency), spans 18
// (50 MB of gathered rows, every workgroup resident at once: the rows' own time and two latencies), join 6.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "seq.h"

namespace dssm {
namespace seq {
namespace {

// ---- lookup ------------------------------------------------------------------------------------
// A lane owns V neighbouring columns (cols_of; the last lane of a row whose width is no multiple takes the row's last
// V, and both that own a column store the same), a row takes G lanes (a power of two up to 64, wider rows loop) and
// a wave 64 / G rows.  A row is one dependent gather behind its id, so each lane has kLookRows rows in flight: the
// ids first, then the rows as they are, converted only when all have been asked for.
constexpr int kLookRows = 4;

template <typename T, typename O, typename I, int V>
__global__ __launch_bounds__(256) void k_lookup(const T* __restrict__ table, int64_t ldt, const I* __restrict__ ids,
                                                int64_t n, int64_t words, int E, float scale, O* __restrict__ out,
                                                int lg) {
  const int G = 1 << lg, slot = threadIdx.x >> lg, slots = 256 >> lg;
  const int64_t r0 = (int64_t)blockIdx.x * slots * kLookRows + slot;
  int64_t id[kLookRows];
#pragma unroll
  for (int j = 0; j < kLookRows; ++j) {
    const int64_t r = r0 + (int64_t)j * slots;
    id[j] = r < n ? (int64_t)ids[r] : -1;
  }
  for (int c0 = (threadIdx.x & (G - 1)) * V; c0 < E; c0 += G * V) {
    const int c = min(c0, E - V);
    Pack<T, V> x[kLookRows];
#pragma unroll
    for (int j = 0; j < kLookRows; ++j)
      if (id[j] >= 0 && id[j] < words) x[j] = ldv<T, V>(table + id[j] * ldt + c);
#pragma unroll
    for (int j = 0; j < kLookRows; ++j) {
      const int64_t r = r0 + (int64_t)j * slots;
      if (r >= n) continue;
      const bool in = id[j] >= 0 && id[j] < words;
      Pack<O, V> y;
#pragma unroll
      for (int i = 0; i < V; ++i) y.v[i] = st1<O>(in ? ld1(x[j].v[i]) * scale : 0.f);
      stv<O, V>(out + r * E + c, y);
    }
  }
}

// ---- sort --------------------------------------------------------------------------------------
// Pairs a workgroup of 1024 threads ranks: 1 or 4 a thread.  One, so that 192 compute units and not 48 rank
// 196608 pairs, until the tiles' counts, which every workgroup reads, become the larger part (kOwnSums): 8.8 us a
// placing launch there, 10.8 with four a thread.
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
// digit.  Wave w holds 64 kItems pairs in a row, lane-major within each item.  A
// wave's lanes find the lanes of their own digit by one ballot per digit bit.  Every thread calls this.
template <int kItems>
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
  __attribute__((aligned(16))) unsigned short hist[16][kMaxBins];
  unsigned total[kMaxBins];
  unsigned scan[16];
};

// The whole sort of at most 4096 pairs in one workgroup: the digits' passes move the pairs through LDS.
// (4 pairs a thread for 4000 ids: 22 us for the whole gradient, the same as many tiles' 23 for 5000; 16 a thread
// for 16384: 45 us against 27.)
constexpr int kOneSort = 4096;

template <typename I, int kItems>
__global__ __launch_bounds__(1024) void k_sort_one(const I* __restrict__ ids, int n, unsigned V, int bits, int passes,
                                                   uint2* __restrict__ pairs, Fill f) {
  __shared__ SortLds s;
  __shared__ unsigned lk[1024 * kItems];
  __shared__ unsigned short lp[1024 * kItems];
  if ((int)blockIdx.x >= f.first) return fill_role(f, blockIdx.x - f.first, gridDim.x - f.first);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  unsigned k[kItems];
  int p[kItems], rank[kItems];
  bool live[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = w * 64 * kItems + j * 64 + lane;
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
      const int i = w * 64 * kItems + j * 64 + lane;
      if (live[j]) {
        k[j] = lk[i];
        p[j] = lp[i];
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int i = w * 64 * kItems + j * 64 + lane;
    if (live[j]) pairs[i] = make_uint2(k[j], (unsigned)p[j]);
  }
}

// A pass over many tiles: counts per tile and digit (cnt [tiles x 1 << bits]) ...
template <typename I, int kItems>
__global__ __launch_bounds__(1024) void k_sort_count(const I* __restrict__ ids, const uint2* __restrict__ in, int64_t n,
                                                     unsigned V, int shift, int bits, unsigned* __restrict__ cnt,
                                                     Fill f) {
  __shared__ unsigned h[4][kMaxBins];  // four copies, so that a hot digit's adds do not all queue at one word
  if ((int)blockIdx.x >= f.first) return fill_role(f, blockIdx.x - f.first, gridDim.x - f.first);
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < 4 * bins; i += 1024) h[i >> bits][i & (bins - 1)] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = (int64_t)blockIdx.x * 1024 * kItems + j * 1024 + threadIdx.x;
    if (i < n) {
      const unsigned k = in ? in[i].x : key_of(ids, i, V);
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
template <typename I, int kItems>
__global__ __launch_bounds__(1024) void k_sort_place(const I* __restrict__ ids, const uint2* __restrict__ in, int64_t n,
                                                     unsigned V, int shift, int bits,
                                                     const unsigned* __restrict__ cnt, int tiles, int summed,
                                                     uint2* __restrict__ out, Fill f) {
  __shared__ SortLds s;
  if ((int)blockIdx.x >= f.first) return fill_role(f, blockIdx.x - f.first, gridDim.x - f.first);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, bins = 1 << bits, me = blockIdx.x;
  unsigned k[kItems], dig[kItems];
  int p[kItems], rank[kItems];
  bool live[kItems];
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const int64_t i = (int64_t)me * 1024 * kItems + w * 64 * kItems + j * 64 + lane;
    live[j] = i < n;
    uint2 kp = make_uint2(0u, (unsigned)i);
    if (live[j] && in) kp = in[i];
    else if (live[j]) kp.x = key_of(ids, i, V);
    k[j] = kp.x;
    p[j] = (int)kp.y;
    dig[j] = (k[j] >> shift) & (bins - 1);
  }
  unsigned all = 0, before = 0;
  if (summed) {
    if ((int)threadIdx.x < bins) {
      before = cnt[(int64_t)me * bins + threadIdx.x];
      all = cnt[(int64_t)tiles * bins + threadIdx.x];
    }
  } else {
    // a thread adds up four digits (one 16-byte load a tile) over every `share`th tile; the shares meet in
    // LDS: share * bins = 4096 sums of each kind, the 32 KB of s.hist before it ranks
    const int d4 = threadIdx.x & (bins / 4 - 1), q = threadIdx.x >> (bits - 2), share = 4096 >> bits;
    uint4 a4 = make_uint4(0, 0, 0, 0), b4 = a4;
    for (int t = q; t < tiles; t += 8 * share) {
      uint4 v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t + i * share < tiles) v[i] = *reinterpret_cast<const uint4*>(cnt + (t + i * share) * bins + d4 * 4);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = t + i * share;
        if (at < tiles) a4 = make_uint4(a4.x + v[i].x, a4.y + v[i].y, a4.z + v[i].z, a4.w + v[i].w);
        if (at < min(tiles, me)) b4 = make_uint4(b4.x + v[i].x, b4.y + v[i].y, b4.z + v[i].z, b4.w + v[i].w);
      }
    }
    unsigned* sum = reinterpret_cast<unsigned*>(s.hist);
    *reinterpret_cast<uint4*>(sum + q * bins + d4 * 4) = a4;
    *reinterpret_cast<uint4*>(sum + 4096 + q * bins + d4 * 4) = b4;
    __syncthreads();
    if ((int)threadIdx.x < bins)
      for (int i = 0; i < min(share, tiles); ++i) {
        all += sum[i * bins + threadIdx.x];
        before += sum[4096 + i * bins + threadIdx.x];
      }
    __syncthreads();
  }
  rank_tile(dig, live, bits, s.hist, s.total, rank);
  const unsigned start = block_scan(all, s.scan) + before;
  if ((int)threadIdx.x < bins) s.total[threadIdx.x] = start;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kItems; ++j)
    if (live[j]) {
      const unsigned at = s.total[dig[j]] + s.hist[w][dig[j]] + rank[j];
      out[at] = make_uint2(k[j], (unsigned)p[j]);
    }
}

// ---- sums --------------------------------------------------------------------------------------
// A group of G lanes, V columns each, sums a stretch of kStretch entries of the sorted list, all rows in
// flight at once; the workgroup's 256 / G stretches are its span.  A run of one token that lies inside a
// stretch goes to the table at once; the pieces of a run that crosses stretches meet in LDS; one that
// crosses spans leaves part[2 s] (the piece of span s that came in from span s - 1) and part[2 s + 1] (the
// piece that starts in s and goes on) for k_grad_join.  A piece that fills its span counts as incoming.
constexpr int kStretch = 8;

template <typename T, int V, bool TREE>
__global__ __launch_bounds__(256) void k_grad_spans(const uint2* __restrict__ pairs, int64_t n, unsigned words,
                                                    const T* __restrict__ dy, int64_t lddy, int E, float scale,
                                                    float* __restrict__ dtable, float* __restrict__ part, int lg) {
  constexpr int kAt = TREE ? 1 : V == 1 ? 8 : 2;  // pieces of a run that are read at once
  __shared__ __attribute__((aligned(16))) float came[256 * V], goes[256 * V];
  __shared__ unsigned long long through[4];  // bits of the threads whose stretch is one run that goes on into the next
  const int G = 1 << lg, groups = 256 >> lg, g = threadIdx.x >> lg, lane = threadIdx.x & (G - 1);
  const int64_t i0 = ((int64_t)blockIdx.x * groups + g) * kStretch, i1 = min(i0 + kStretch, n);
  const unsigned none = 0xffffffffu;
  uint2 k[kStretch];
#pragma unroll
  for (int j = 0; j < kStretch; ++j) k[j] = i0 + j < n ? pairs[i0 + j] : make_uint2(none, 0u);
  const unsigned prev = i0 && i0 < n ? pairs[i0 - 1].x : none, next = i1 < n ? pairs[i1].x : none;
  unsigned last = k[0].x;
#pragma unroll
  for (int j = 1; j < kStretch; ++j) last = k[j].x != none ? k[j].x : last;
  const bool live = i0 < n, in = live && k[0].x == prev, out = live && last == next;
  const bool one = k[0].x == last;  // the stretch is one run
  const unsigned long long pass = __ballot(one && out);
  if ((threadIdx.x & 63) == 0) through[threadIdx.x >> 6] = pass;
  // the last stretch of the run that comes into stretch `from`: the first from there on that is not passed through
  // (groups: the run goes on behind the span)
  auto first_stop = [&](int from) {
    int e = groups;
    const int t0 = from << lg;
    for (int w = t0 >> 6; w < 4 && e == groups; ++w) {
      const unsigned long long stop = ~through[w] & (w == t0 >> 6 ? ~0ull << (t0 & 63) : ~0ull);
      if (stop) e = (w * 64 + __ffsll(stop) - 1) >> lg;
    }
    return e;
  };
  for (int c0 = 0; c0 < E; c0 += G * V) {
    const bool mine = c0 + lane * V < E;
    const int c = min(c0 + lane * V, E - V);
    Pack<T, V> x[kStretch];
#pragma unroll
    for (int j = 0; j < kStretch; ++j)
      if (mine && k[j].x < words) x[j] = ldv<T, V>(dy + (int64_t)k[j].y * lddy + c);
    float acc[V];
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = 0.f;
    bool incoming = in;
#pragma unroll
    for (int j = 0; j < kStretch; ++j) {
      const unsigned cur = k[j].x, after = j + 1 < kStretch ? k[j + 1 < kStretch ? j + 1 : j].x : none;
      if (mine && cur < words) {
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] += ld1(x[j].v[q]);
        if (after != cur) {  // the run's end in this stretch
          const bool outgoing = after == none && out;
          if (incoming || outgoing) {
            float* to = incoming ? came : goes;
#pragma unroll
            for (int q = 0; q < V; ++q) to[threadIdx.x * V + q] = acc[q];
          } else {
            Pack<float, V> y;
#pragma unroll
            for (int q = 0; q < V; ++q) y.v[q] = acc[q] * scale;
            stv<float, V>(dtable + (int64_t)cur * E + c, y);
          }
#pragma unroll
          for (int q = 0; q < V; ++q) acc[q] = 0.f;
          incoming = false;
        }
      }
    }
    __syncthreads();
    if constexpr (TREE) {
      // came[g] becomes the sum of a run's pieces from stretch g to its last one here, by doubling (but for g = 0).
      // What no run has brought is not used.
      const int end = first_stop(g);
      for (int d = 1; d < groups; d <<= 1) {
        const bool more = g && g + d <= min(end, groups - 1);
        if (!__syncthreads_or(more)) break;
        float x[V];
        if (more && mine) {
#pragma unroll
          for (int q = 0; q < V; ++q) x[q] = came[threadIdx.x * V + q] + came[(threadIdx.x + (d << lg)) * V + q];
        }
        __syncthreads();
        if (more && mine) {
#pragma unroll
          for (int q = 0; q < V; ++q) came[threadIdx.x * V + q] = x[q];
        }
      }
      __syncthreads();
    }
    // Who joins a run's pieces: the group where it starts, or group 0 for the one that came into the span.
    const bool starts = out && !(in && one) && last < words;
    const bool enters = g == 0 && in && k[0].x < words;
#pragma unroll
    for (int role = 0; role < 2; ++role) {
      if (!mine || !(role ? starts : enters)) continue;
      const float* from = role ? goes : came;
      float sum[V];
#pragma unroll
      for (int q = 0; q < V; ++q) sum[q] = from[threadIdx.x * V + q];
      bool on = role || (one && out);  // the run reaches the next stretch
      if (on) {
        const int e = first_stop(g + 1);
        on = e == groups;
        // in order, several pieces' reads at once (more at once take registers that waves need)
        const int n1 = min((TREE ? g + 1 : e) + 1, groups);
        for (int j = g + 1; j < n1; j += kAt) {
          float x[kAt][V];
#pragma unroll
          for (int u = 0; u < kAt; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) x[u][q] = j + u < n1 ? came[((((j + u) << lg) + lane) & 255) * V + q] : 0.f;
#pragma unroll
          for (int u = 0; u < kAt; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) sum[q] += x[u][q];
        }
      }
      if (role && !on) {
        Pack<float, V> y;
#pragma unroll
        for (int q = 0; q < V; ++q) y.v[q] = sum[q] * scale;
        stv<float, V>(dtable + (int64_t)last * E + c, y);
      } else {
        Pack<float, V> y;
#pragma unroll
        for (int q = 0; q < V; ++q) y.v[q] = sum[q];
        stv<float, V>(part + (2 * (int64_t)blockIdx.x + role) * E + c, y);
      }
    }
    __syncthreads();
  }
}

// Joins the runs that cross spans: the lanes of span s own the run that starts in s and goes on.  A run
// of few spans is summed at once; a longer one is left to the whole workgroup, whose groups take equal
// stretches of it and join them through LDS, so that half a list of one token is no chain of loads.
constexpr int kShort = 8;
constexpr int kOwned = 8;  // spans a workgroup looks after: its long runs follow each other

template <int V>
__global__ __launch_bounds__(256) void k_grad_join(const uint2* __restrict__ pairs, int64_t n, int64_t spans, int S,
                                                   unsigned words, int E, float scale, const float* __restrict__ part,
                                                   float* __restrict__ dtable, int lg) {
  const int G = 1 << lg, groups = 256 >> lg, grp = threadIdx.x >> lg, lane = threadIdx.x & (G - 1);
  const int owned = min(groups, kOwned);  // spans of this workgroup
  __shared__ float red[256 * V];
  __shared__ int64_t longs[256];
  __shared__ int nlong;
  if (threadIdx.x == 0) nlong = 0;
  __syncthreads();
  const int64_t s = (int64_t)blockIdx.x * owned + grp;
  const int64_t end = (s + 1) * S;  // the next span's first entry
  if (grp < owned && end < n) {
    // all the keys that decide, asked for together: the span's ends, the entry in front of it, and the
    // first entries of the next spans
    const unsigned cur = pairs[end].x, tail = pairs[end - 1].x, head = pairs[s * S].x;
    const unsigned front = s ? pairs[s * S - 1].x : 0xffffffffu;
    unsigned ahead[kShort];
#pragma unroll
    for (int j = 0; j < kShort; ++j) ahead[j] = (s + 2 + j) * S < n ? pairs[(s + 2 + j) * S].x : 0xffffffffu;
    // the run starts in s: its token is not also the one that came in and fills the span from its start
    if (cur < words && tail == cur && (head != cur || front != cur)) {
      int more = 0;  // spans behind s + 1 that the run reaches
#pragma unroll
      for (int j = 0; j < kShort; ++j) more += more == j && ahead[j] == cur;
      if (more < kShort) {
        for (int c0 = lane * V; c0 < E; c0 += G * V) {
          const int c = min(c0, E - V);
          Pack<float, V> x[kShort + 1];
          x[0] = ldv<float, V>(part + (2 * s + 1) * E + c);
#pragma unroll
          for (int j = 0; j < kShort; ++j)
            if (j <= more) x[j + 1] = ldv<float, V>(part + 2 * (s + 1 + j) * E + c);
          Pack<float, V> y = x[0];
#pragma unroll
          for (int j = 0; j < kShort; ++j)
            if (j <= more) {
#pragma unroll
              for (int q = 0; q < V; ++q) y.v[q] += x[j + 1].v[q];
            }
#pragma unroll
          for (int q = 0; q < V; ++q) y.v[q] *= scale;
          stv<float, V>(dtable + (int64_t)cur * E + c, y);
        }
      } else if (lane == 0) {
        longs[atomicAdd(&nlong, 1)] = s;
      }
    }
  }
  __syncthreads();
  for (int j = 0; j < nlong; ++j) {
    const int64_t h = longs[j];
    const unsigned tok = pairs[(h + 1) * S].x;
    // the run's last span: the last one whose first entry is still this token.  The list is sorted, so of 256
    // probes at equal distances a first few are this token's, and the last of those bounds the next round; the
    // first round looks at the next 256 spans, where nearly every run ends.
    int64_t lo = h + 1, hi = spans - 1;
    for (bool first = true; lo < hi; first = false) {
      const int64_t gap = first ? 1 : (hi - lo + 255) / 256, at = lo + (threadIdx.x + 1) * gap;
      const int hit = __syncthreads_count(at <= hi && pairs[at * S].x == tok);
      if (hit < 256 || !first) hi = min(hi, lo + (hit + 1) * gap - 1);
      lo += hit * gap;
    }
    const int64_t cnt = lo - h, per = (cnt + groups - 1) / groups;
    const int64_t a = min(h + 1 + grp * per, lo + 1), b = min(a + per, lo + 1);
    for (int c0 = 0; c0 < E; c0 += G * V) {
      const bool mine = c0 + lane * V < E;
      const int c = min(c0 + lane * V, E - V);
      float acc[V];
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] = 0.f;
      if (mine) {
        int64_t t = a;
        for (; t + 8 <= b; t += 8) {
          Pack<float, V> x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = ldv<float, V>(part + 2 * (t + u) * E + c);
#pragma unroll
          for (int u = 0; u < 8; ++u)
#pragma unroll
            for (int q = 0; q < V; ++q) acc[q] += x[u].v[q];
        }
        for (; t < b; ++t) {
          const Pack<float, V> x = ldv<float, V>(part + 2 * t * E + c);
#pragma unroll
          for (int q = 0; q < V; ++q) acc[q] += x.v[q];
        }
      }
#pragma unroll
      for (int q = 0; q < V; ++q) red[q * 256 + threadIdx.x] = acc[q];
      const int used = (int)((cnt + per - 1) / per);
      for (int d = 1; d < used; d <<= 1) {
        __syncthreads();
        if (!(grp & (2 * d - 1)) && grp + d < used)
#pragma unroll
          for (int q = 0; q < V; ++q) red[q * 256 + threadIdx.x] += red[q * 256 + threadIdx.x + (d << lg)];
      }
      if (grp == 0 && mine) {
        Pack<float, V> x = ldv<float, V>(part + (2 * h + 1) * E + c);
#pragma unroll
        for (int q = 0; q < V; ++q) x.v[q] = (x.v[q] + red[q * 256 + threadIdx.x]) * scale;
        stv<float, V>(dtable + (int64_t)tok * E + c, x);
      }
      __syncthreads();
    }
  }
}

// ---- few tokens --------------------------------------------------------------------------------
// One launch without a sort: a workgroup owns RR rows of the table, looks through all (at most kFew) ids for its
// own, and adds their rows up in LDS in the order of their positions, the groups of lanes each the rows of its
// residue; a run of one token stays in registers.  Then it writes its RR rows, zeros among them, once.
constexpr int kFew = 32;

template <typename T, typename I, int V>
__global__ __launch_bounds__(256) void k_grad_few(const I* __restrict__ ids, int n, int64_t words, int RR,
                                                  const T* __restrict__ dy, int64_t lddy, int E, float scale,
                                                  float* __restrict__ dtable, int lg) {
  extern __shared__ __attribute__((aligned(16))) float acc[];  // [RR x E]
  __shared__ unsigned list[kFew];                              // row << 16 | position, in the order of positions
  __shared__ int found;
  const int lane = threadIdx.x & 63;
  const int64_t row0 = (int64_t)blockIdx.x * RR;
  const int rows = (int)min((int64_t)RR, words - row0);
  const int64_t r = (int)threadIdx.x < n ? (int64_t)ids[threadIdx.x] - row0 : -1;
  const bool mine = r >= 0 && r < rows;
  float* out = dtable + row0 * E;
  const int total = rows * E;
  if (!__syncthreads_or(mine)) {  // most workgroups
    const float zero[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x * 4; i < total; i += 1024) st_row<float, 4>(out + i, total - i, zero);
    return;
  }
  for (int i = threadIdx.x; i < total; i += 256) acc[i] = 0.f;
  const unsigned long long all = __ballot(mine);  // (all ids are in wave 0)
  if (mine) list[__popcll(all & ((1ull << lane) - 1ull))] = (unsigned)r << 16 | threadIdx.x;
  if (threadIdx.x == 0) found = __popcll(all);
  __syncthreads();
  const int m = found;
  const int G = 1 << lg, groups = 256 >> lg, g = threadIdx.x >> lg;
  for (int c = (threadIdx.x & (G - 1)) * V; c < E; c += G * V) {
    const unsigned none = 0xffffffffu;
    unsigned cur = none;
    float sum[V];
    auto flush = [&] {
      if (cur == none) return;
#pragma unroll
      for (int q = 0; q < V; ++q) acc[(int)cur * E + c + q] += sum[q];
    };
    for (int j0 = 0; j0 < m; j0 += 16) {
      Pack<T, V> x[16];
      unsigned k[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        k[j] = j0 + j < m ? list[j0 + j] : none;
        if ((int)((k[j] >> 16) & (groups - 1)) != g) k[j] = none;
        if (k[j] != none) x[j] = ldv<T, V>(dy + (k[j] & 0xffffu) * lddy + c);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k[j] != none) {
          if (k[j] >> 16 != cur) {
            flush();
            cur = k[j] >> 16;
#pragma unroll
            for (int q = 0; q < V; ++q) sum[q] = 0.f;
          }
#pragma unroll
          for (int q = 0; q < V; ++q) sum[q] += ld1(x[j].v[q]);
        }
    }
    flush();
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += 256) out[i] = acc[i] * scale;
}

// Columns a lane owns: 8, 4 or 1, `most` at most; the widest that divides the row or leaves it four lanes (196608 ids over
// 21128 words: 118 bf16 columns 12.6 us and 49, their gradient, with 8 a lane, 26.6 and 69 with one; 33 fp32 9.9 and 44,
// 16.5 and 53; but 20000 ids, 11 bf16 columns 3.4 and 25.6 with 8 a lane, 2.9 and 23.5 with one).  k_grad_few, which adds
// up in place, takes the widest that divides the row.
int cols_of(int E, int most) {
  if (most >= 8 && (E % 8 == 0 || E >= 32)) return 8;
  return E % 4 == 0 || E >= 16 ? 4 : 1;
}
int divisor_of(int E, int most) { return most >= 8 && E % 8 == 0 ? 8 : E % 4 == 0 ? 4 : 1; }
template <typename F>
void by_cols_of(int v, F&& f) {
  if (v == 8) f(std::integral_constant<int, 8>{});
  else if (v == 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 1>{});
}
int lanes_log2(int E, int v) {  // log2 of the lanes a row takes, at most a wave
  int lg = 0;
  while (lg < 6 && (v << lg) < E) ++lg;
  return lg;
}
// Lanes and columns of the summing launch, and the entries of its workgroups' spans.
template <typename T>
constexpr int kGradCols = sizeof(T) == 4 ? 4 : 8;
int span_of(int E, int dtype) {
  return (256 >> lanes_log2(E, cols_of(E, dtype == DSSM_F32 ? kGradCols<float> : kGradCols<u16>))) * kStretch;
}

// More counts (tiles x bins) than this have their sums made by a launch of their own (k_sort_sums, 3 us); up to
// it every workgroup of k_sort_place adds them up itself, 4096 of them at a time: 2.5 us for 192 x 256.
constexpr int64_t kOwnSums = 64 * 1024;

// Workspace of a gradient: pairs twice, the tiles' digit counts, the spans' partial rows.
struct GradWs {
  int bits, passes, S, items, summed;
  int64_t tiles, spans;
  size_t pairs[2], cnt, part, bytes;
};
GradWs grad_ws(int64_t n, int64_t V, int E, int dtype) {
  GradWs g{};
  int bits = 1;
  while (((int64_t)1 << bits) <= V) ++bits;  // keys 0 .. V
  g.passes = (bits + 9) / 10;
  g.bits = std::max(6, (bits + g.passes - 1) / g.passes);  // (few bins leave k_sort_place long sums for few threads)
  const int64_t t1 = (n + 1023) / 1024;
  g.items = (t1 << g.bits) <= kOwnSums ? 1 : 4;
  g.tiles = (n + 1024 * g.items - 1) / (1024 * g.items);
  g.summed = (g.tiles << g.bits) > kOwnSums;
  g.S = span_of(E, dtype);
  g.spans = (n + g.S - 1) / g.S;
  size_t at = 0;
  auto take = [&](size_t b) {
    const size_t o = at;
    at += (b + 255) / 256 * 256;
    return o;
  };
  g.pairs[0] = take(8 * n);
  g.pairs[1] = take(g.passes > 1 && n > kOneSort ? 8 * n : 0);
  g.cnt = take(4 * (size_t)(g.tiles + 1) << g.bits);
  g.part = take((size_t)g.spans * 2 * E * 4);
  g.bytes = at;
  return g;
}
constexpr int kFewLds = 48 * 1024;
// One launch for few ids and a table of up to 32 MB; a larger one is cleared faster beside the sort's launches.
// Measured (32 ids, all different to all the same): 1000 x 32 4.3 to 9.4 us against the sort's 9.5, 21128 x 128 7.7
// to 12.3 against 11.2; 128 ids, all the same: 30 us against 13; 300007 x 100: 32 us against 20.
bool few(int64_t n, int64_t V, int E) { return n <= kFew && E * 4 <= kFewLds && V * E <= (8 << 20); }
bool grad_dims_ok(int64_t n, int64_t V, int E) {
  return n >= 0 && n < ((int64_t)1 << 31) - 4096 && V > 0 && V < ((int64_t)1 << 30) && E > 0 && E <= (1 << 20);
}

template <typename I>
int run_grad(const void* dy, int dtype, int64_t lddy, const I* ids, int64_t n, int64_t V, int E, float scale, float* dtable,
             char* ws, hipStream_t s) {
  if (n && few(n, V, E)) {
    // rows that fit 48 KB of LDS, fewer where that leaves less than 2048 workgroups
    const int RR = (int)std::max<int64_t>(1, std::min<int64_t>(kFewLds / 4 / E, (V + 2047) / 2048));
    by_dtype(dtype, [&](auto tag) {
      using T = decltype(tag);
      by_cols_of(divisor_of(E, kGradCols<T>), [&](auto vec) {
        constexpr int VEC = decltype(vec)::value;
        if constexpr (VEC <= kGradCols<T>)
          hipLaunchKernelGGL((k_grad_few<T, I, VEC>), dim3((unsigned)((V + RR - 1) / RR)), dim3(256), (size_t)RR * E * 4, s, ids,
                             (int)n, V, RR, (const T*)dy, lddy, E, scale, dtable, lanes_log2(E, VEC));
      });
    });
    return seq_status(hipGetLastError());
  }
  const GradWs g = grad_ws(n, V, E, dtype);
  uint2* pairs[2] = {(uint2*)(ws + g.pairs[0]), (uint2*)(ws + g.pairs[1])};
  unsigned* cnt = (unsigned*)(ws + g.cnt);
  float* part = (float*)(ws + g.part);
  const bool one = n <= kOneSort;
  // the table's zeros, a share to each of the sort's launches: the placing ones take twice as long as the counting ones
  const int64_t total = V * E, all4 = total / 4;
  const int shares = one ? 1 : 3 * g.passes;
  int share = 0;
  auto part_of = [&](int own, int* grid, int weight) {
    Fill f{};
    const int64_t a = all4 * share / shares, b = all4 * (share + weight) / shares;
    f.p = dtable + a * 4;
    f.n4 = b - a;
    f.tail = share + weight == shares ? (int)(total - all4 * 4) : 0;
    f.first = own;
    const int extra = f.n4 || f.tail ? (int)std::min<int64_t>(512, (f.n4 + 4095) / 4096 + 1) : 0;
    *grid = own + extra;
    share += weight;
    return f;
  };
  int grid = 0, side = 0;
  if (g.spans > kMaxBlocks) return dssm::report_error(DSSM_E_UNSUPPORTED, "embedding_grad: too many ids");
  if (n == 0) {
    return seq_status(zero_bytes_async(dtable, (size_t)total * 4, s));
  } else if (one) {
    const Fill f = part_of(1, &grid, 1);
    auto kernel = n <= 1024 ? k_sort_one<I, 1> : k_sort_one<I, kOneSort / 1024>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(1024), 0, s, ids, (int)n, (unsigned)V, g.bits, g.passes, pairs[0], f);
  } else {
    const int tiles = (int)g.tiles;
    for (int q = 0; q < g.passes; ++q) {
      const uint2* in = q ? pairs[side] : nullptr;
      if (q) side ^= 1;
      auto pass = [&](auto items) {
        constexpr int kItems = decltype(items)::value;
        Fill f = part_of(tiles, &grid, 1);
        hipLaunchKernelGGL((k_sort_count<I, kItems>), dim3(grid), dim3(1024), 0, s, ids, in, n, (unsigned)V, q * g.bits,
                           g.bits, cnt, f);
        if (g.summed)
          hipLaunchKernelGGL(k_sort_sums, dim3(((1 << g.bits) + 63) / 64), dim3(1024), 0, s, cnt, tiles, 1 << g.bits);
        f = part_of(tiles, &grid, 2);
        hipLaunchKernelGGL((k_sort_place<I, kItems>), dim3(grid), dim3(1024), 0, s, ids, in, n, (unsigned)V, q * g.bits,
                           g.bits, cnt, tiles, g.summed, pairs[side], f);
      };
      if (g.items == 1) pass(std::integral_constant<int, 1>{});
      else pass(std::integral_constant<int, 4>{});
    }
  }
  auto blocks_of = [&](int lg) { 
    const int owned = std::min(256 >> lg, kOwned);
    return dim3((unsigned)((g.spans + owned - 1) / owned));
  };
  by_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    by_cols_of(cols_of(E, kGradCols<T>), [&](auto vec) {
      constexpr int VEC = decltype(vec)::value;
      if constexpr (VEC <= kGradCols<T>) {
        const int lg = lanes_log2(E, VEC);
        // 64 stretches a span and more add their pieces up by doubling (175517 x 4 bf16 over 25 words 22 us for this
        // launch, 9.6 by doubling; the whole gradient of 196608 x 32 bf16 over 500 words 32.5 and 29.3), fewer one after
        // the other (196608 x 32 fp32 28.5 and 29.1, 196608 x 128 bf16 over 21128 words 18.4 us for this launch and 20.5)
        auto kernel = lg <= 2 ? k_grad_spans<T, VEC, true> : k_grad_spans<T, VEC, false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)g.spans), dim3(256), 0, s, pairs[side], n, (unsigned)V, (const T*)dy, lddy, E,
                           scale, dtable, part, lg);
      }
    });
  });
  if (g.spans > 1) {
    const int v = cols_of(E, 4), lg = lanes_log2(E, v);
    if (v == 4)
      hipLaunchKernelGGL(k_grad_join<4>, blocks_of(lg), dim3(256), 0, s, pairs[side], n, g.spans, g.S, (unsigned)V, E, scale,
                         part, dtable, lg);
    else
      hipLaunchKernelGGL(k_grad_join<1>, blocks_of(lg), dim3(256), 0, s, pairs[side], n, g.spans, g.S, (unsigned)V, E, scale,
                         part, dtable, lg);
  }
  return seq_status(hipGetLastError());
}

}  // namespace
}  // namespace seq
}  // namespace dssm

using namespace dssm::seq;

extern "C" int dssm_embedding_lookup(const void* table, int dtype, int64_t ldt, int64_t V, int E, const void* ids,
                                     int ids64, int64_t n, float scale, void* out, int out_dtype, void* stream) {
  if (!table || !seq_dtype(dtype) || !seq_dtype(out_dtype) || V <= 0 || E <= 0 || E > (1 << 30) || ldt < E || n < 0 ||
      (n > 0 && (!ids || !out)))
    return dssm::report_error(DSSM_E_INVALID, "embedding_lookup: bad argument (1 to 2^30 columns)");
  if (n == 0) return DSSM_OK;
  const int v = cols_of(E, 8), lg = lanes_log2(E, v);
  const int64_t rows = (int64_t)(256 >> lg) * kLookRows, blocks = (n + rows - 1) / rows;
  if (blocks > kMaxBlocks) return dssm::report_error(DSSM_E_UNSUPPORTED, "embedding_lookup: too many ids");
  by_dtype(dtype, [&](auto t) {
    by_dtype(out_dtype, [&](auto o) {
      by_cols_of(v, [&](auto vec) {
        using T = decltype(t);
        using O = decltype(o);
        constexpr int VEC = decltype(vec)::value;
        if (ids64)
          hipLaunchKernelGGL((k_lookup<T, O, int64_t, VEC>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                             (const T*)table, ldt, (const int64_t*)ids, n, V, E, scale, (O*)out, lg);
        else
          hipLaunchKernelGGL((k_lookup<T, O, int32_t, VEC>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream,
                             (const T*)table, ldt, (const int32_t*)ids, n, V, E, scale, (O*)out, lg);
      });
    });
  });
  return seq_status(hipGetLastError());
}

extern "C" size_t dssm_embedding_grad_ws_bytes(int64_t n, int64_t V, int E, int dtype) {
  if (!grad_dims_ok(n, V, E) || !seq_dtype(dtype)) return 0;
  return few(n, V, E) ? 16 : grad_ws(n, V, E, dtype).bytes + 256;
}

extern "C" int dssm_embedding_grad(const void* dy, int dtype, int64_t lddy, const void* ids, int ids64, int64_t n,
                                   int64_t V, int E, float scale, float* dtable, void* ws, size_t ws_bytes, void* stream) {
  if (!seq_dtype(dtype) || !grad_dims_ok(n, V, E) || lddy < E || !dtable || (n > 0 && (!dy || !ids || !ws)))
    return dssm::report_error(DSSM_E_INVALID, "embedding_grad: bad argument");
  if ((uintptr_t)dtable % 16 || (uintptr_t)ws % 16)
    return dssm::report_error(DSSM_E_INVALID, "embedding_grad: the gradient and the workspace are 16-byte aligned");
  if (n > 0 && !few(n, V, E) && ws_bytes < grad_ws(n, V, E, dtype).bytes)
    return dssm::report_error(DSSM_E_INVALID, "embedding_grad: workspace too small (dssm_embedding_grad_ws_bytes)");
  return ids64 ? run_grad(dy, dtype, lddy, (const int64_t*)ids, n, V, E, scale, dtable, (char*)ws, (hipStream_t)stream)
               : run_grad(dy, dtype, lddy, (const int32_t*)ids, n, V, E, scale, dtable, (char*)ws, (hipStream_t)stream);
}
