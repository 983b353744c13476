// sample_rows.cu - a token for every row of logits, by temperature, top-k,
// top-p and min-p from given random numbers.
//
//   w_i = exp((x_i - max) / T), tokens in order of falling x, then rising index;
//   the first n stay: n <= top_k, n the least whose w's sum reaches top_p of the
//   top k's, w >= min_p; the token is the first whose sum passes u times theirs.
//
// All three filters and the draw cut one order, so nothing is sorted but what
// lies around a cut.  A cluster of up to eight CTAs takes a row:
//   max  ->  histogram of (max - x) / T, 123 bins an e-fold down to a weight of
//   2^-24: counts and weights, summed over the cluster  ->  prefix sums give the
//   bins of the cuts  ->  the tokens of the bins down to the last cut, if they are
//   at most kCap, or else of the cuts' bins one after the other, go to the first
//   CTA's shared memory; there a cut's bin is sorted and the cut found in it.
// A bin of more than kCap tokens is cut into 2048 finer ones; one of those that
// still holds too many (ties, all but always) is searched by bisection of the
// values, then of the indexes.
//
// Weights are whole numbers of 2^-S, S = 62 - ceil(log2 n), from 64-bit floats
// (2e-15): sums are exact whatever the order of the atomics, so results do not
// depend on it.  Each is off by half a step, and 0 below that, so a sum by n 2^-(S+1)
// of the largest at most (1.2e-10 for 32,000 tokens, 1.2e-7 for 2^20), and a token
// differs from an exact evaluation's only where u falls as near to a border.
//
// Bound: for few rows the chain of passes and of the cluster's waits (1 x 32000,
// top-k and top-p: 17 us; 16 of them, top-p 22; 33 x 50001 fp16, each with filters of its
// own, 37); for many the histogram's instructions, about half of the time, and the
// collecting (64 x 131072: 63 us, one read of HBM would be 5; the further passes find
// the row in L2).
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "tos_dev.cuh"
#include "tos_kernels.h"

namespace cg = cooperative_groups;

namespace tos {

constexpr int kSmpThreads = 512;
constexpr int kBins = 2048;
constexpr int kCap = 4096;              // tokens that are listed, and sorted, in shared memory
constexpr int kPerThread = kBins / kSmpThreads;
typedef unsigned long long u64;

struct SampleArgs {
  const void* x;
  long long stride;
  int n, vec, shift;                    // shift: S
  const float* temperature;
  const int* top_k;
  const float *top_p, *min_p, *u;
  int* token;
  float* prob;
  int* kept;
};

// What a cut is: the first token at which the count is `count` and the sum of weights
// `sum`, one of them for what the cut asks, the other the least there is.
struct Cut {
  unsigned count;
  u64 sum;
};
__device__ __forceinline__ Cut by_count(unsigned n) { return {n, 0}; }
__device__ __forceinline__ Cut reaches(double w) { return {1, w > 0.0 ? (u64)ceil(w) : 0}; }
__device__ __forceinline__ Cut passes(double w) { return {1, (u64)floor(w) + 1}; }    // w >= 0
__device__ __forceinline__ bool past(const Cut& c, unsigned n, u64 w) { return n >= c.count && w >= c.sum; }
struct Found {
  unsigned n;                           // tokens up to and with it
  u64 w, own;                           // their weight, its own
  int index;
};
struct CutBin {                         // where a cut falls in a histogram
  int bin;
  unsigned n0, count;                   // tokens before the bin, in it
  u64 w0, w;                            // weight before it, up to its end
};

// A histogram: weights in two words, counts; or, in the same place, inclusive sums.
struct Hist {
  union {
    struct {
      alignas(16) unsigned lo[kBins], hi[kBins];
    };
    u64 w[kBins];
  };
  alignas(16) unsigned n[kBins];
};
struct SampleShared {
  Hist hist;                            // this CTA's, then all CTAs' inclusive sums
  union {
    Hist all;                           // a part of the bins, all CTAs' (all_bins)
    u64 sorted[kCap];                   // first CTA: a cut's bin
  };
  union {
    u64 list[kCap];                     // tokens, value over inverted index; first CTA: all CTAs'
    Hist fine;                          // a bin cut finer, as hist
  };
  double pow2[32];
  u64 wsum[kSmpThreads / 32];
  unsigned wcnt[kSmpThreads / 32];
  u64 part_w[2][2];                     // this CTA's sums, two rounds apart
  unsigned part_n[2][2];
  float best[kSmpThreads / 32];
  float top;                            // this CTA's largest logit; NaN: it has one
  unsigned first;                       // its first place
  unsigned listed[4];                   // tokens that this CTA has listed for the first, second .. time
  unsigned pushed[4];                   // first CTA: tokens that the others have, from the list's end on
  unsigned picked, base;
  CutBin cut[3];
  Found found;
};

// Order-preserving bits of a float; -0 as +0.
__device__ __forceinline__ unsigned order_key(float x) {
  const unsigned b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Bins.  The first kBins - 1 are for weights of 2^-24 and more, the last for all
// that are less (and summed apart, without atomics); cut finer, those have 41 bins
// an e-fold.
constexpr float kBinsFold = (kBins - 1) / (24 * 0.69314718f);
constexpr float kFineLast = 41.0f / kBinsFold;

struct Row {
  const void* x;
  int n, vec, shift;
  int rank, ctas;
  float top;                            // the largest logit
  bool inf;                             // that was +infinity: such count as 0, all others as far below (and T as 1)
  double rate;                          // log2(e) / T
  float scale;                          // bins per unit of max - x
  const double* pow2;
  // Rounded before it is used, whatever the compiler may fuse: fine() takes a bin's
  // number, which is this rounded down, from it, and that must not become negative.
  __device__ __forceinline__ float place(float v) const { return __fmul_rn(top - v, scale); }
  __device__ __forceinline__ int bin(float v) const { return min(__float2int_rd(place(v)), kBins - 1); }
  __device__ __forceinline__ int fine(float v, int b) const {
    return min(__float2int_rd((place(v) - (float)b) * (b == kBins - 1 ? kFineLast : (float)kBins)), kBins - 1);
  }
  // 2^(shift - (top - v) rate) to the nearest whole number: 2^(m/32) from a table,
  // 2^r, |r| <= 1/64, by its Taylor sum (next term 2e-15).  Whole numbers come of
  // adding 1.5 2^52, 2^52.  No branches: a warp's lanes would take both sides.
  __device__ __forceinline__ u64 weight(float v) const {
    double y = fma((double)v - (double)top, rate, (double)shift);
    y = y > -2.0 ? y : -2.0;                              // 0, as is NaN (-infinity at T infinite)
    const double big = fma(y, 32.0, 6755399441055744.0);
    const int m = __double2loint(big);
    const double r = fma(big - 6755399441055744.0, -1.0 / 32, y);
    constexpr double c1 = 0.6931471805599453, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6, c4 = c2 * c2 / 6, c5 = c2 * c3 / 10;
    double p = fma(r, c5, c4);
    p = fma(p, r, c3);
    p = fma(p, r, c2);
    p = fma(p, r, c1);
    p = fma(p, r, 1.0) * pow2[m & 31];
    p = __hiloint2double(__double2hiint(p) + ((m >> 5) << 20), __double2loint(p));
    return (u64)__double_as_longlong(p + 4503599627370496.0) & 0xfffffffffffffull;
  }
};

// f(values, index of the first) of this CTA's pieces of 16 bytes; a warp's lanes go
// together; -infinity behind the row's end.
template <typename E, typename F>
__device__ __forceinline__ void sweep(const Row& r, F f) {
  constexpr int P = 16 / sizeof(E), U = 4;
  const int pieces = (r.n + P - 1) / P, lane = threadIdx.x & 31, step = r.ctas * kSmpThreads;
  const E* x = reinterpret_cast<const E*>(r.x);
  for (int p0 = r.rank * kSmpThreads + (threadIdx.x & ~31); p0 < pieces; p0 += U * step) {
    uint4 w[U];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = (p0 + q * step + lane) * P;
      constexpr uint32_t none = sizeof(E) == 4 ? 0xff800000u : 0xfc00fc00u;
      w[q] = make_uint4(none, none, none, none);
      if (r.vec && i + P <= r.n) {
        w[q] = *reinterpret_cast<const uint4*>(x + i);
      } else if (i < r.n) {
        uint32_t h[4] = {none, none, none, none};
#pragma unroll
        for (int e = 0; e < P; ++e)
          if (i + e < r.n) {
            if constexpr (sizeof(E) == 4) h[e] = __float_as_uint((float)x[i + e]);
            else h[e / 2] = e & 1 ? (h[e / 2] & 0xffffu) | (uint32_t)reinterpret_cast<const uint16_t*>(x)[i + e] << 16
                                  : (h[e / 2] & 0xffff0000u) | reinterpret_cast<const uint16_t*>(x)[i + e];
          }
        w[q] = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (p0 + q * step >= pieces) break;
      float v[P];
      const uint32_t h[4] = {w[q].x, w[q].y, w[q].z, w[q].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(E) == 4) {
          v[e] = __uint_as_float(h[e]);
        } else {
          const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
          v[2 * e] = g.x;
          v[2 * e + 1] = g.y;
        }
      }
      if (r.inf) {
#pragma unroll
        for (int e = 0; e < P; ++e) v[e] = v[e] == INFINITY ? 0.0f : fminf(v[e], -1e30f);
      }
      f(v, (p0 + q * step + lane) * P);
    }
  }
}

__device__ __forceinline__ void add_weight(Hist& s, int b, u64 w, unsigned n) {
  atomicAdd(&s.n[b], n);
  const unsigned l = (unsigned)w;
  const unsigned old = l ? atomicAdd(&s.lo[b], l) : 0u;
  const unsigned h = (unsigned)(w >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(&s.hi[b], h);
}

// Inclusive sums over the block of (w, n), thread by thread; the totals come too.
__device__ __forceinline__ void block_scan(SampleShared& s, u64& w, unsigned& n, u64& all_w, unsigned& all_n) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 a = __shfl_up_sync(0xffffffffu, w, o);
    const unsigned b = __shfl_up_sync(0xffffffffu, n, o);
    if (lane >= o) {
      w += a;
      n += b;
    }
  }
  __syncthreads();
  if (lane == 31) {
    s.wsum[warp] = w;
    s.wcnt[warp] = n;
  }
  __syncthreads();
  all_w = 0;
  all_n = 0;
#pragma unroll
  for (int i = 0; i < kSmpThreads / 32; ++i) {
    if (i == warp) {
      w += all_w;
      n += all_n;
    }
    all_w += s.wsum[i];
    all_n += s.wcnt[i];
  }
}
// Sums over the block.
__device__ __forceinline__ void block_sum(SampleShared& s, u64& w, unsigned& n) {
  u64 a;
  unsigned b;
  block_scan(s, w, n, a, b);
  w = a;
  n = b;
}

__device__ __forceinline__ void clear(Hist& s) {
  for (int b = threadIdx.x; b < kBins; b += kSmpThreads) s.lo[b] = s.hi[b] = s.n[b] = 0;
}

// All CTAs' histograms, from (w0, n0) on, as inclusive sums in each one's `h`.  A CTA
// adds up its share of the bins, four of one CTA a thread and the CTAs' by shuffles
// (by remote atomics: 12,000 cycles, so 6,500); then each reads all of them.
__device__ __forceinline__ void all_bins(cg::cluster_group& cl, SampleShared& s, Hist& h, u64 w0, unsigned n0) {
  const int ctas = (int)cl.num_blocks(), each = kBins / ctas, from = (int)threadIdx.x % ctas;
  const int mine = (int)cl.block_rank() * each + (int)threadIdx.x / ctas * kPerThread;
  cl.sync();
  {
    const Hist& g = &h == &s.hist ? cl.map_shared_rank(&s, from)->hist : cl.map_shared_rank(&s, from)->fine;
    const uint4 lo = *reinterpret_cast<const uint4*>(g.lo + mine), hi = *reinterpret_cast<const uint4*>(g.hi + mine);
    const uint4 cn = *reinterpret_cast<const uint4*>(g.n + mine);
    u64 w[4] = {((u64)hi.x << 32) + lo.x, ((u64)hi.y << 32) + lo.y, ((u64)hi.z << 32) + lo.z, ((u64)hi.w << 32) + lo.w};
    unsigned n[4] = {cn.x, cn.y, cn.z, cn.w};
    static_assert(kPerThread == 4, "a uint4 of bins");
    for (int x = 1; x < ctas; x <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] += __shfl_xor_sync(0xffffffffu, w[i], x);
        n[i] += __shfl_xor_sync(0xffffffffu, n[i], x);
      }
    if (from == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s.all.w[mine + i] = w[i];
        s.all.n[mine + i] = n[i];
      }
    }
  }
  cl.sync();
  const int b0 = threadIdx.x * kPerThread;
  const SampleShared* o = cl.map_shared_rank(&s, b0 / each);
  u64 x[kPerThread], all;
  unsigned y[kPerThread], alln;
  {
    const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(o->all.w + b0), q = *reinterpret_cast<const ulonglong2*>(o->all.w + b0 + 2);
    const uint4 c = *reinterpret_cast<const uint4*>(o->all.n + b0);
    x[0] = p.x; x[1] = p.y; x[2] = q.x; x[3] = q.y;
    y[0] = c.x; y[1] = c.y; y[2] = c.z; y[3] = c.w;
  }
#pragma unroll
  for (int i = 1; i < kPerThread; ++i) {
    x[i] += x[i - 1];
    y[i] += y[i - 1];
  }
  u64 sum = x[kPerThread - 1];
  unsigned sn = y[kPerThread - 1];
  block_scan(s, sum, sn, all, alln);
  sum += w0 - x[kPerThread - 1];
  sn += n0 - y[kPerThread - 1];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    h.w[b0 + i] = sum + x[i];
    h.n[b0 + i] = sn + y[i];
  }
  __syncthreads();
}

// The first bin past the cut, of inclusive sums from (w0, n0) on; by all threads,
// to be read behind a barrier.
__device__ __forceinline__ void find_bin(CutBin& to, const Cut& c, const Hist& h, u64 w0, unsigned n0) {
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = threadIdx.x * kPerThread + i;
    const u64 wb = b ? h.w[b - 1] : w0;
    const unsigned nb = b ? h.n[b - 1] : n0;
    if (past(c, h.n[b], h.w[b]) && !past(c, nb, wb)) to = {b, nb, h.n[b] - nb, wb, h.w[b]};
  }
}

// Which values lie in bins from[i] to to[i] for some i, of the fine ones of bin
// from[0] in `f` alone (f < 0: in all).
template <int N>
struct Ranges {
  Row r;
  int from[N], to[N], f;
  bool plain;
  __device__ __forceinline__ Ranges(const Row& row, int fine) : r(row), f(fine), plain(fine < 0 && row.scale > 0.0f) {}
  __device__ __forceinline__ void set(int i, int a, int b) {
    from[i] = a;
    to[i] = b;
    plain &= b < kBins - 1;
  }
  __device__ __forceinline__ bool has(float v) const {
    bool in = false;
    if (plain) {                                          // -infinity, and what lies further than floats go: not in any
      const float x = r.place(v);
#pragma unroll
      for (int i = 0; i < N; ++i) in |= x >= (float)from[i] && x < (float)(to[i] + 1);
      return in;
    }
    const int b = r.bin(v);
#pragma unroll
    for (int i = 0; i < N; ++i) in |= b >= from[i] && b <= to[i];
    return in && v > -INFINITY && (f < 0 || r.fine(v, from[0]) == f);
  }
};

// Tokens of a range go to the first CTA's list, by way of this CTA's: its own from the
// front, the others' from the end.  (An atomic add in another CTA's memory for every
// piece with a token costs 16 x 32000 0.6 us more.)
template <typename E, typename G>
__device__ __forceinline__ void collect(SampleShared& s, SampleShared* lead, const Row& r, const G& g, int time) {
  sweep<E>(r, [&](const auto& v, int i) {
    constexpr int P = 16 / sizeof(E);
    unsigned mine = 0;
#pragma unroll
    for (int e = 0; e < P; ++e) mine |= (g.has(v[e]) ? 1u : 0u) << e;
    if (!mine) return;
    unsigned at = atomicAdd(&s.listed[time], __popc(mine));
#pragma unroll
    for (int e = 0; e < P; ++e)
      if (mine >> e & 1) {
        if (at < kCap) s.list[at] = (u64)order_key(v[e]) << 32 | ~(unsigned)(i + e);
        ++at;
      }
  });
  if (r.rank == 0) return;
  __syncthreads();
  const unsigned n = min(s.listed[time], (unsigned)kCap);
  if (threadIdx.x == 0) s.base = atomicAdd(&lead->pushed[time], n);
  __syncthreads();
  for (unsigned i = threadIdx.x; i < n; i += kSmpThreads)
    if (s.base + i < kCap) lead->list[kCap - 1 - (s.base + i)] = s.list[i];
}

// First CTA: of the list's tokens of a cut's bin (all: it has no others), in falling
// order, the first past the cut.
constexpr int kQuick = 128;
__device__ __noinline__ Found find_listed(SampleShared& s, const Row& r, const Cut& c, const CutBin& at, int time, bool all) {
  const int tid = threadIdx.x, count = (int)at.count, front = (int)s.listed[time], listed = front + (int)s.pushed[time];
  auto token = [&](int i) { return s.list[i < front ? i : kCap - 1 - (i - front)]; };
  if (tid == 0) s.picked = 0;
  if (count <= kQuick) {
    // Each token's place and the weight before it, by comparing it with all: 4 to 32
    // lanes a token.  (As below one token takes 5,000 cycles, so 4,300, a hundred 10,000
    // and 6,700.)
    u64* weights = s.sorted + kCap / 2;
    __syncthreads();
    for (int i = tid; i < listed; i += kSmpThreads) {
      const u64 x = token(i);
      const float v = key_value((unsigned)(x >> 32));
      if (!all && r.bin(v) != at.bin) continue;
      const unsigned to = atomicAdd(&s.picked, 1u);
      s.sorted[to] = x;
      weights[to] = r.weight(v);
    }
    __syncthreads();
    int lg = 5;                                           // of the lanes a token
    while (count << lg > kSmpThreads) --lg;
    const int lanes = 1 << lg, i = tid >> lg;
    u64 w = 0;
    unsigned n = 0;
    if (i < count) {
      const u64 x = s.sorted[i];
      for (int j = tid & (lanes - 1); j < count; j += lanes)
        if (s.sorted[j] > x) {
          w += weights[j];
          ++n;
        }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      w += __shfl_xor_sync(0xffffffffu, w, o);
      n += __shfl_xor_sync(0xffffffffu, n, o);
    }
    w += at.w0;
    n += at.n0;
    if (i < count && (tid & (lanes - 1)) == 0 && past(c, n + 1, w + weights[i]) && !past(c, n, w))
      s.found = {n + 1, w + weights[i], weights[i], (int)~(unsigned)s.sorted[i]};
    __syncthreads();
    return s.found;
  }
  int m = 2 * kQuick;
  while (m < count) m <<= 1;
  for (int i = count + tid; i < m; i += kSmpThreads) s.sorted[i] = 0;
  __syncthreads();
  for (int i = tid; i < listed; i += kSmpThreads) {
    const u64 x = token(i);
    if (all) s.sorted[i] = x;
    else if (r.bin(key_value((unsigned)(x >> 32))) == at.bin) s.sorted[atomicAdd(&s.picked, 1u)] = x;
  }
  __syncthreads();
  auto stage = [&](int k, int j, int i) {
    const int a = 2 * i - (i & (j - 1)), b = a + j;
    const u64 x = s.sorted[a], y = s.sorted[b];
    if ((x < y) == ((a & k) == 0)) {
      s.sorted[a] = y;
      s.sorted[b] = x;
    }
  };
  for (int k = 2; k <= m; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < m / 2; i += kSmpThreads) stage(k, j, i);
      __syncthreads();
    }
  // sums from (w0, n0) on, a run of tokens a thread
  const int run = (count + kSmpThreads - 1) / kSmpThreads, i0 = tid * run, i1 = min(i0 + run, count);
  u64 sum = 0, total;
  unsigned none = 0, nonen;
  for (int i = i0; i < i1; ++i) sum += r.weight(key_value((unsigned)(s.sorted[i] >> 32)));
  u64 w = sum;
  block_scan(s, w, none, total, nonen);
  w += at.w0 - sum;
  for (int i = i0; i < i1; ++i) {
    const u64 own = r.weight(key_value((unsigned)(s.sorted[i] >> 32))), before = w;
    w += own;
    const unsigned n = at.n0 + i;
    if (past(c, n + 1, w) && !past(c, n, before)) s.found = {n + 1, w, own, (int)~(unsigned)s.sorted[i]};
  }
  __syncthreads();
  return s.found;
}

// Count and weight over the row of the tokens for which keep(value, index), the
// same in every CTA.  round: 0, 1 in turn.
template <typename E, typename F>
__device__ __forceinline__ void count_row(cg::cluster_group& cl, SampleShared& s, const Row& r, int round, F keep, u64& w,
                                          unsigned& n) {
  w = 0;
  n = 0;
  sweep<E>(r, [&](const auto& v, int i) {
    constexpr int P = 16 / sizeof(E);
#pragma unroll 1
    for (int e = 0; e < P; ++e)
      if (v[e] > -INFINITY && keep(v[e], i + e)) {
        w += r.weight(v[e]);
        ++n;
      }
  });
  block_sum(s, w, n);
  if (threadIdx.x == 0) {
    s.part_w[round][0] = w;
    s.part_n[round][0] = n;
  }
  cl.sync();
  w = 0;
  n = 0;
  for (unsigned c = 0; c < cl.num_blocks(); ++c) {
    const SampleShared* o = cl.map_shared_rank(&s, c);
    w += o->part_w[round][0];
    n += o->part_n[round][0];
  }
}

// The token at which a cut falls, in the bin where it does; the same in every CTA
// (last: in the first, the others need not know).  time: 0, 1 .. of a row.
template <typename E>
__device__ __noinline__ Found resolve(cg::cluster_group& cl, SampleShared& s, const Row& r, const Cut& c, CutBin at, int time,
                                      bool last) {
  SampleShared* lead = cl.map_shared_rank(&s, 0);
  const int b = at.bin;
  int f = -1;                                             // the finer bin, if any
  if (at.count > kCap) {
    cl.sync();                                            // what was read of `all`, what was sorted there, the list are done with
    clear(s.fine);
    __syncthreads();
    sweep<E>(r, [&](const auto& v, int) {
      constexpr int P = 16 / sizeof(E);
#pragma unroll 1
      for (int e = 0; e < P; ++e)
        if (v[e] > -INFINITY && r.bin(v[e]) == b) add_weight(s.fine, r.fine(v[e], b), r.weight(v[e]), 1);
    });
    all_bins(cl, s, s.fine, at.w0, at.n0);
    find_bin(s.cut[2], c, s.fine, at.w0, at.n0);
    __syncthreads();
    at = s.cut[2];
    f = at.bin;
    cl.sync();                                            // `all` is read, `fine` makes way for the list
  }
  Ranges<1> g(r, f);
  g.set(0, b, b);
  Found got;
  if (at.count <= kCap) {
    collect<E>(s, lead, r, g, time);
    cl.sync();
    if (r.rank == 0) got = find_listed(s, r, c, at, time, true);
    if (last) return got;
    cl.sync();
    return lead->found;
  }
  // bisection: the largest key k such that what is not below it is past the cut
  const u64 w0 = at.w0;
  const unsigned n0 = at.n0;
  unsigned lo = 0, hi = 0xffffffffu;
  int round = 0;
  u64 w;
  unsigned n;
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2 + 1;
    count_row<E>(cl, s, r, round ^= 1, [&](float v, int) { return order_key(v) >= mid && g.has(v); }, w, n);
    if (past(c, n0 + n, w0 + w)) lo = mid;
    else hi = mid - 1;
  }
  count_row<E>(cl, s, r, round ^= 1, [&](float v, int) { return order_key(v) > lo && g.has(v); }, w, n);
  w += w0;
  n += n0;
  const u64 own = r.weight(key_value(lo));
  // the ties it takes
  unsigned t = c.count > n ? c.count - n : 1;
  if (c.sum > w + t * own) t = (unsigned)((c.sum - w + own - 1) / own);
  unsigned a = 0, z = (unsigned)r.n - 1;                  // the t-th of them by index
  while (a < z) {
    const unsigned mid = a + (z - a) / 2;
    u64 dw;
    unsigned dn;
    count_row<E>(cl, s, r, round ^= 1, [&](float v, int i) { return order_key(v) == lo && (unsigned)i <= mid; }, dw, dn);
    if (dn >= t) z = mid;
    else a = mid + 1;
  }
  got = {n + t, w + t * own, own, (int)a};
  return got;
}

// One CTA an SM: two, of 64 registers a thread, spill (one row 21.7 us, 18.1; 64 x
// 131072 77.0, 71.3).
template <typename E>
__global__ void __launch_bounds__(kSmpThreads, 1) sample_rows_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  constexpr int P = 16 / sizeof(E);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Row r;
  r.rank = (int)cl.block_rank();
  r.ctas = (int)cl.num_blocks();
  const int row = blockIdx.x / r.ctas;
  r.x = reinterpret_cast<const E*>(a.x) + (long long)row * a.stride;
  r.n = a.n;
  r.vec = a.vec;
  r.shift = a.shift;
  r.inf = false;
  r.pow2 = s.pow2;
  SampleShared* lead = cl.map_shared_rank(&s, 0);
  clear(s.hist);
  if (tid < 32) s.pow2[tid] = exp2((double)tid / 32.0);
  if (tid < 4) s.listed[tid] = s.pushed[tid] = 0;
  if (tid == 0) s.first = 0xffffffffu;
  pdl_wait();
  pdl_trigger();

  // the largest; NaN if there is one
  auto top_nan = [](float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
  };
  float best = -INFINITY;
  sweep<E>(r, [&](const auto& v, int) {
    float m = top_nan(v[0], v[1]);
#pragma unroll
    for (int e = 2; e < P; e += 2) m = top_nan(m, top_nan(v[e], v[e + 1]));
    best = top_nan(best, m);
  });
  for (int o = 16; o > 0; o >>= 1) best = top_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.best[warp] = best;
  __syncthreads();
  if (warp == 0) {
    best = s.best[lane & (kSmpThreads / 32 - 1)];
    for (int o = kSmpThreads / 64; o > 0; o >>= 1) best = top_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) s.top = best;
  }
  cl.sync();
  best = lane < r.ctas ? cl.map_shared_rank(&s, lane)->top : -INFINITY;
  for (int o = 4; o > 0; o >>= 1) best = top_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
  r.top = __shfl_sync(0xffffffffu, best, 0);
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  const bool none = isnan(r.top) || r.top == -INFINITY;   // nothing to choose from
  if (none || !(T > 0.0f)) {
    if (!none) {                                          // the first of the largest
      unsigned at = 0xffffffffu;
      sweep<E>(r, [&](const auto& v, int i) {
#pragma unroll
        for (int e = 0; e < P; ++e)
          if (v[e] == r.top) at = min(at, (unsigned)(i + e));
      });
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == 0 && at != 0xffffffffu) atomicMin(&lead->first, at);
      cl.sync();
    }
    if (r.rank == 0 && tid == 0) {
      a.token[row] = none ? -1 : (int)s.first;
      if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
      if (a.kept) a.kept[row] = none ? 0 : 1;
    }
    cl.sync();                                            // nobody leaves while its memory is read
    return;
  }
  r.inf = isinf(r.top);
  if (r.inf) r.top = 0.0f;
  r.rate = r.inf ? 1.0 : 1.4426950408889634 / (double)T;
  r.scale = r.inf ? 1.0f : fminf(kBinsFold / T, 1e30f);

  const float pf = a.top_p ? a.top_p[row] : 1.0f, mf = a.min_p ? a.min_p[row] : 0.0f;
  const bool by_p = pf < 1.0f, by_m = mf > 0.0f;
  const double p = pf;
  const double log_m = by_m ? log2(fmin((double)mf, 1.0)) : 0.0;   // as logarithms: small weights are rounded too coarsely
  u64 wm = 0, wl = 0;                                     // of the tokens that min-p keeps, of the last bin's
  unsigned nm = 0, nl = 0;
  sweep<E>(r, [&](const auto& v, int) {
    // four at a time: their weights, then their atomics
#pragma unroll
    for (int e0 = 0; e0 < P; e0 += 4) {
      u64 w[4];
      int b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = r.weight(v[e0 + e]);
        b[e] = r.bin(v[e0 + e]);
      }
      unsigned old[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        old[e] = 0;
        if (v[e0 + e] == -INFINITY) {
          b[e] = kBins;
        } else if (b[e] == kBins - 1) {
          wl += w[e];
          ++nl;
        } else {
          atomicAdd(&s.hist.n[b[e]], 1u);
          old[e] = atomicAdd(&s.hist.lo[b[e]], (unsigned)w[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const unsigned h = (unsigned)(w[e] >> 32) + (old[e] + (unsigned)w[e] < old[e] ? 1u : 0u);
        if (b[e] < kBins - 1 && h) atomicAdd(&s.hist.hi[b[e]], h);
        if (by_m && b[e] < kBins && ((double)v[e0 + e] - (double)r.top) * r.rate >= log_m) {
          wm += w[e];
          ++nm;
        }
      }
    }
  });
  for (int o = 16; o > 0; o >>= 1) {
    wl += __shfl_xor_sync(0xffffffffu, wl, o);
    nl += __shfl_xor_sync(0xffffffffu, nl, o);
  }
  if (lane == 0 && nl) add_weight(s.hist, kBins - 1, wl, nl);
  if (by_m) {
    block_sum(s, wm, nm);
    if (tid == 0) {
      s.part_w[0][1] = wm;
      s.part_n[0][1] = nm;
    }
  }
  all_bins(cl, s, s.hist, 0, 0);
  if (by_m) {
    wm = 0;
    nm = 0;
    for (int c = 0; c < r.ctas; ++c) {
      const SampleShared* o = cl.map_shared_rank(&s, c);
      wm += o->part_w[0][1];
      nm += o->part_n[0][1];
    }
  }
  // every CTA has the same sums and finds the same bins
  const u64 total_w = s.hist.w[kBins - 1];
  const unsigned total_n = s.hist.n[kBins - 1];
  const int k = a.top_k ? a.top_k[row] : 0;
  const bool by_k = k > 0 && (unsigned)k < total_n;
  const Cut cut_k = by_count((unsigned)k);
  float uf = a.u[row];
  uf = uf >= 0.0f ? fminf(uf, 0.99999994f) : 0.0f;        // NaN: 0
  if (by_k) find_bin(s.cut[0], cut_k, s.hist, 0, 0);
  else if (by_p) find_bin(s.cut[0], reaches(p * (double)total_w), s.hist, 0, 0);
  if (by_m) find_bin(s.cut[1], by_count(nm), s.hist, 0, 0);
  __syncthreads();

  // the bins down to the last cut; a top-p of the top k needs all of those
  int last = kBins - 1;
  unsigned upto = total_n;
  auto down_to = [&](const CutBin& c) {
    if (c.bin < last) {
      last = c.bin;
      upto = c.n0 + c.count;
    }
  };
  const CutBin first_cut = s.cut[0];
  if (by_k || by_p) down_to(first_cut);
  if (by_m && !(by_k && by_p)) down_to(s.cut[1]);
  // Few tokens: all of them.  Else the bins that the cuts may fall in: k's is known,
  // p's and the draw's as closely as the weight down to the cut before is.
  Ranges<3> g(r, -1);
  bool few = upto <= kCap;
  g.set(0, 0, last);
  g.set(1, 0, last);
  g.set(2, 0, last);
  if (!few) {
    double lo = (double)total_w, hi = lo;
    int b0 = kBins - 1, b1 = b0;
    if (by_k) {
      lo = (double)first_cut.w0;
      hi = (double)first_cut.w;
      b0 = b1 = first_cut.bin;
    }
    unsigned count = 0;
    auto between = [&](const Cut& x, const Cut& y) {    // the bins of the cuts at x and at y
      __syncthreads();
      find_bin(s.cut[0], x, s.hist, 0, 0);
      find_bin(s.cut[2], y, s.hist, 0, 0);
      __syncthreads();
      count += s.cut[2].n0 + s.cut[2].count - s.cut[0].n0;
      b0 = s.cut[0].bin;
      b1 = s.cut[2].bin;
    };
    if (by_k) count += first_cut.count;
    g.set(0, by_k ? b0 : -1, by_k ? b1 : -1);
    g.set(1, -1, -1);
    if (by_p) {
      between(reaches(p * lo), reaches(p * hi));
      g.set(1, b0, b1);
      lo = (double)s.cut[0].w0;
      hi = (double)s.cut[2].w;
    }
    if (by_m) lo = fmin(lo, (double)wm);
    between(passes((double)uf * lo), passes((double)uf * hi));
    g.set(2, b0, b1);
    few = count <= kCap;
  }
  if (few) {
    collect<E>(s, lead, r, g, 0);
    cl.sync();
    if (r.rank != 0) {
      cl.sync();
      return;
    }
  }
  // One cut after the other; where the bins are listed, in the first CTA alone.
  // Of two that are bins apart only the nearer is looked for.
  int time = 0;
  auto cut_at = [&](const Cut& c, bool final) {
    __syncthreads();
    find_bin(s.cut[0], c, s.hist, 0, 0);
    __syncthreads();
    const CutBin at = s.cut[0];
    if (few) return find_listed(s, r, c, at, 0, false);
    return resolve<E>(cl, s, r, c, at, time++, final);
  };
  unsigned n = total_n;
  u64 wn = total_w;
  const bool m_nearer = by_m && !(by_k && by_p) && nm < n;
  if (by_k && !(m_nearer && nm <= (unsigned)k)) {
    n = (unsigned)k;
    wn = first_cut.w;
    // a bin that ends with the cut, or weighs nothing, need not be looked at
    if (first_cut.n0 + first_cut.count != n && first_cut.w != first_cut.w0)
      wn = few ? find_listed(s, r, cut_k, first_cut, 0, false).w : resolve<E>(cl, s, r, cut_k, first_cut, time++, false).w;
  }
  if (by_p && !(m_nearer && nm <= first_cut.n0)) {
    const Found f = cut_at(reaches(p * (double)wn), false);
    if (f.n < n) {
      n = f.n;
      wn = f.w;
    }
  }
  if (by_m && nm < n) {
    n = nm;
    wn = wm;
  }
  const Found f = cut_at(passes((double)uf * (double)wn), true);
  if (r.rank == 0 && tid == 0) {
    a.token[row] = f.index;
    if (a.prob) a.prob[row] = (float)((double)f.own / (double)wn);
    if (a.kept) a.kept[row] = (int)n;
  }
  cl.sync();
}

}  // namespace tos

using namespace tos;

extern "C" int tosk_sample_rows(const tosk_sample_t* t, cudaStream_t st) {
  SampleArgs a;
  a.x = t->x;
  a.stride = t->stride;
  a.n = t->n;
  const int es = t->type == TOSK_F32 ? 4 : 2;
  a.vec = ((uintptr_t)t->x & 15) == 0 && t->stride * es % 16 == 0;
  int lg = 0;
  while ((1ll << lg) < t->n) ++lg;
  a.shift = lg < 11 ? 51 : 62 - lg;              // weights below 2^52, their sum below 2^62
  a.temperature = t->temperature;
  a.top_k = t->top_k;
  a.top_p = t->top_p; a.min_p = t->min_p; a.u = t->u;
  a.token = t->token;
  a.prob = t->prob;
  a.kept = t->kept;
  // A cluster's SMs are neighbours, so that not every count of them fits at once:
  // 16 clusters of eight take two rounds (39.4 us; of four 25.9).
  int ctas = 8;
  while (ctas > 1 && (long long)t->n_rows * ctas > (ctas == 8 ? 104 : ctas == 4 ? 136 : 148)) ctas /= 2;
  while (ctas > 1 && t->n < 1024 * ctas) ctas /= 2;
  const long long grid = (long long)t->n_rows * ctas;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  const void* f = t->type == TOSK_F32 ? (const void*)sample_rows_kernel<float> : (const void*)sample_rows_kernel<__half>;
  const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SampleShared));
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kSmpThreads);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  void* args[] = {&a};
  return (int)cudaLaunchKernelExC(&cfg, f, args);
}
