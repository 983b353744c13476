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
//   2^-24: counts and weights  ->  prefix sums in the cluster's first CTA give the
//   bins of the cuts  ->  the bins down to the last cut, if they hold at most
//   kCap tokens, or else the bins of the cuts one after the other, go to the first
//   CTA's shared memory, are sorted there and resolved.
// A bin of more than kCap tokens is cut into 2048 finer ones; one of those that
// still holds too many (ties, all but always) is searched by bisection of the
// values, then of the indexes.
//
// Weights are whole numbers of 2^-S, S = 62 - ceil(log2 n), from 64-bit floats
// (2e-15): sums are exact whatever the order of the atomics, so results do not
// depend on it, and a token differs from an exact evaluation's only where u
// falls within ~1e-12 of a border.
//
// Bound: one read from HBM; the further passes find the row in L2.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "tos_dev.cuh"
#include "tos_kernels.h"

namespace cg = cooperative_groups;

namespace tos {

constexpr int kSmpThreads = 512;
constexpr int kBins = 2048;
constexpr int kCap = 2048;              // tokens that are sorted in shared memory
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

// What a cut is: the first token at which the count is `count`, or the sum of
// weights reaches (passes) `sum`.
enum { kByCount, kReach, kPass };
struct Cut {
  int mode;
  unsigned count;
  double sum;
};
__device__ __forceinline__ bool past(const Cut& c, unsigned n, u64 w) {
  return c.mode == kByCount ? n >= c.count : c.mode == kReach ? (double)w >= c.sum : (double)w > c.sum;
}
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
enum { kBinK, kBinP, kBinM, kBinCuts };

struct SampleShared {
  unsigned lo[kBins], hi[kBins], cnt[kBins];     // this CTA's histogram: weights in two words, counts
  u64 cum_w[kBins];                     // first CTA: all CTAs' histograms, then their inclusive sums
  unsigned cum_n[kBins];
  u64 list[kCap];                       // first CTA: tokens to sort, value over inverted index; or finer bins' weights
  unsigned fine_n[kBins];               // and their counts
  double pow2[32];
  u64 wsum[kSmpThreads / 32];
  unsigned wcnt[kSmpThreads / 32];
  u64 part_w[2][2];                     // this CTA's sums, two rounds apart
  unsigned part_n[2][2];
  float best[kSmpThreads / 32];
  float top;                            // this CTA's largest logit; NaN: it has one
  unsigned first;                       // its first place
  unsigned listed;
  CutBin cut[kBinCuts];                 // first CTA
  Found found;                          // first CTA
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
// that are less; cut finer, those have 41 bins an e-fold.
constexpr float kBinsFold = (kBins - 1) / (24 * 0.69314718f);
constexpr float kFineLast = 41.0f / kBinsFold;

struct Row {
  const void* x;
  int n, vec, shift;
  int rank, ctas;
  float top;                            // the largest logit
  double rate;                          // log2(e) / T
  float scale;                          // bins per unit of max - x
  const double* pow2;
  // how far below the top
  __device__ __forceinline__ float below(float v) const { return v == top ? 0.0f : top - v; }
  __device__ __forceinline__ float place(float v) const { return below(v) * scale; }
  __device__ __forceinline__ int bin(float v) const { return min(__float2int_rd(place(v)), kBins - 1); }
  __device__ __forceinline__ int fine(float v, int b) const {
    return min(__float2int_rd((place(v) - (float)b) * (b == kBins - 1 ? kFineLast : (float)kBins)), kBins - 1);
  }
  // 2^(shift - (top - v) rate) to the nearest whole number: 2^(m/32) from a table,
  // 2^r, |r| <= 1/64, by its Taylor sum (next term 2e-15).  Whole numbers come of
  // adding 1.5 2^52, 2^52.  In the last bin fp32 will do: each weight is below 2^-24
  // and off by 3e-6 of itself.
  __device__ __forceinline__ u64 weight(float v) const {
    if (v == top) return 1ull << shift;
    const float d = top - v;
    if (isinf(d)) return 0;                               // below an infinity, whatever T
    if (d * scale >= (float)(kBins - 1)) {
      float y;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(-d, (float)rate, (float)shift)));
      return __float2uint_rn(y);
    }
    const double y = fma((double)v - (double)top, rate, (double)shift);
    if (!(y > -1.0)) return 0;                            // T so small that the bins' scale has its limit
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
      f(v, (p0 + q * step + lane) * P);
    }
  }
}

__device__ __forceinline__ void add_weight(SampleShared& s, int b, u64 w, unsigned n = 1) {
  atomicAdd(&s.cnt[b], n);
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

__device__ __forceinline__ void clear_bins(SampleShared& s) {
  for (int b = threadIdx.x; b < kBins; b += kSmpThreads) s.lo[b] = s.hi[b] = s.cnt[b] = 0;
}

// Adds this CTA's bins to the first one's sums.  By atomics that return nothing, so
// that none is waited for.
__device__ __forceinline__ void push_bins(SampleShared& s, u64* w, unsigned* n) {
  for (int b = threadIdx.x; b < kBins; b += kSmpThreads)
    if (const unsigned c = s.cnt[b]) {
      atomicAdd(n + b, c);
      if (const u64 x = ((u64)s.hi[b] << 32) + s.lo[b]) atomicAdd(w + b, x);
    }
}
// First CTA: its sums, inclusive from (w0, n0) on.
__device__ __forceinline__ void scan_bins(SampleShared& s, u64* w, unsigned* n, u64 w0, unsigned n0) {
  const int b0 = threadIdx.x * kPerThread;
  u64 x[kPerThread], all;
  unsigned y[kPerThread], alln;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    x[i] = w[b0 + i] + (i ? x[i - 1] : 0);
    y[i] = n[b0 + i] + (i ? y[i - 1] : 0);
  }
  u64 sum = x[kPerThread - 1];
  unsigned sn = y[kPerThread - 1];
  block_scan(s, sum, sn, all, alln);
  sum += w0 - x[kPerThread - 1];
  sn += n0 - y[kPerThread - 1];
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    w[b0 + i] = sum + x[i];
    n[b0 + i] = sn + y[i];
  }
  __syncthreads();
}

// First CTA: the list sorted, falling.
__device__ __forceinline__ void sort_list(SampleShared& s, int count) {
  int m = 2;
  while (m < count) m <<= 1;
  for (int i = count + threadIdx.x; i < m; i += kSmpThreads) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= m; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < m / 2; i += kSmpThreads) {
        const int a = 2 * i - (i & (j - 1)), b = a + j;
        const u64 x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & k) == 0)) {
          s.list[a] = y;
          s.list[b] = x;
        }
      }
      __syncthreads();
    }
}

// First CTA: inclusive sums over the sorted list, from (w0, n0) on, this thread's
// entries threadIdx.x * 4 ..; own: their weights.
constexpr int kListed = kCap / kSmpThreads;
__device__ __forceinline__ void scan_list(SampleShared& s, const Row& r, int count, u64 w0, unsigned n0, u64 (&cum)[kListed],
                                          u64 (&own)[kListed]) {
  u64 sum = 0, all;
  unsigned n = 0, alln;
#pragma unroll
  for (int i = 0; i < kListed; ++i) {
    const int at = threadIdx.x * kListed + i;
    own[i] = at < count ? r.weight(key_value((unsigned)(s.list[at] >> 32))) : 0;
    sum += own[i];
    cum[i] = sum;
  }
  u64 incl = sum;
  block_scan(s, incl, n, all, alln);
#pragma unroll
  for (int i = 0; i < kListed; ++i) cum[i] += w0 + incl - sum;
}
// First CTA: the first entry of the list past the cut, or `other`.
__device__ __forceinline__ Found find_listed(SampleShared& s, const u64 (&cum)[kListed], const u64 (&own)[kListed], int count,
                                             unsigned n0, const Cut& c, const Found& other) {
  __syncthreads();
  if (threadIdx.x == 0) s.found = other;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kListed; ++i) {
    const int at = threadIdx.x * kListed + i;
    if (at < count && past(c, n0 + at + 1, cum[i]) && (at == 0 || !past(c, n0 + at, cum[i] - own[i])))
      s.found = {n0 + at + 1, cum[i], own[i], (int)~(unsigned)s.list[at]};
  }
  __syncthreads();
  return s.found;
}

// First CTA: the first bin past the cut, of inclusive sums from (w0, n0) on.
__device__ __forceinline__ void find_bin(CutBin& to, const Cut& c, const u64* w, const unsigned* n, u64 w0, unsigned n0) {
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int b = threadIdx.x * kPerThread + i;
    const u64 wb = b ? w[b - 1] : w0;
    const unsigned nb = b ? n[b - 1] : n0;
    if (n[b] > nb && past(c, n[b], w[b]) && (nb == 0 || !past(c, nb, wb))) to = {b, nb, n[b] - nb, wb, w[b]};
  }
}

// Tokens for which keep(value) go to the first CTA's list.
template <typename E, typename F>
__device__ __forceinline__ void collect(SampleShared* lead, const Row& r, F keep) {
  const int lane = threadIdx.x & 31;
  sweep<E>(r, [&](const auto& v, int i) {
    constexpr int P = 16 / sizeof(E);
    unsigned mine = 0;
#pragma unroll
    for (int e = 0; e < P; ++e) mine |= (v[e] > -INFINITY && keep(v[e]) ? 1u : 0u) << e;
    if (!__any_sync(0xffffffffu, mine != 0)) return;
    unsigned at = __popc(mine);                           // a place for each in the list
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned x = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += x;
    }
    unsigned base = 0;
    if (lane == 31) base = atomicAdd(&lead->listed, at);
    at += __shfl_sync(0xffffffffu, base, 31) - __popc(mine);
#pragma unroll
    for (int e = 0; e < P; ++e)
      if (mine >> e & 1) {
        if (at < kCap) lead->list[at] = (u64)order_key(v[e]) << 32 | ~(unsigned)(i + e);
        ++at;
      }
  });
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

// The token at which a cut falls, in the bin where it does; the same in every CTA.
template <typename E>
__device__ __noinline__ Found resolve(cg::cluster_group& cl, SampleShared& s, const Row& r, const Cut& c, CutBin at) {
  SampleShared* lead = cl.map_shared_rank(&s, 0);
  const int b = at.bin;
  int f = -1;                                             // the finer bin, if any
  if (at.count > kCap) {
    clear_bins(s);
    if (r.rank == 0)
      for (int i = threadIdx.x; i < kBins; i += kSmpThreads) {
        s.list[i] = 0;
        s.fine_n[i] = 0;
      }
    cl.sync();
    sweep<E>(r, [&](const auto& v, int) {
      constexpr int P = 16 / sizeof(E);
#pragma unroll 1
      for (int e = 0; e < P; ++e)
        if (v[e] > -INFINITY && r.bin(v[e]) == b) add_weight(s, r.fine(v[e], b), r.weight(v[e]));
    });
    __syncthreads();
    push_bins(s, lead->list, lead->fine_n);
    cl.sync();
    if (r.rank == 0) {
      scan_bins(s, s.list, s.fine_n, at.w0, at.n0);
      // nb == 0 in find_bin stands for the very first token: past is monotone, so
      // with tokens before the bin the test of what comes before holds
      find_bin(s.cut[kBinK], c, s.list, s.fine_n, at.w0, at.n0);
    }
    cl.sync();
    at = lead->cut[kBinK];
    f = at.bin;
  }
  const int cnt = (int)at.count;
  const u64 w0 = at.w0;
  const unsigned n0 = at.n0;
  auto mine = [&](float v) { return r.bin(v) == b && (f < 0 || r.fine(v, b) == f); };
  Found got;
  if (cnt <= kCap) {
    cl.sync();
    if (r.rank == 0 && threadIdx.x == 0) s.listed = 0;
    cl.sync();
    collect<E>(lead, r, mine);
    cl.sync();
    if (r.rank == 0) {
      sort_list(s, cnt);
      u64 cum[kListed], own[kListed];
      scan_list(s, r, cnt, w0, n0, cum, own);
      find_listed(s, cum, own, cnt, n0, c, Found{});
    }
    cl.sync();
    got = lead->found;
    return got;
  }
  // bisection: the largest key k such that what is not below it is past the cut
  unsigned lo = 0, hi = 0xffffffffu;
  int round = 0;
  u64 w;
  unsigned n;
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2 + 1;
    count_row<E>(cl, s, r, round ^= 1, [&](float v, int) { return order_key(v) >= mid && mine(v); }, w, n);
    if (past(c, n0 + n, w0 + w)) lo = mid;
    else hi = mid - 1;
  }
  count_row<E>(cl, s, r, round ^= 1, [&](float v, int) { return order_key(v) > lo && mine(v); }, w, n);
  w += w0;
  n += n0;
  const u64 own = r.weight(key_value(lo));
  // the ties it takes
  unsigned t;
  if (c.mode == kByCount) {
    t = c.count - n;
  } else {
    const double q = floor((c.sum - (double)w) / (double)own);
    t = q < 1.0 ? 1u : (unsigned)fmin(q, 1e9);
    while (t > 1 && past(c, 0, w + (t - 1) * own)) --t;
    while (!past(c, 0, w + t * own)) ++t;
  }
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

template <typename E>
__global__ void __launch_bounds__(kSmpThreads, 2) sample_rows_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint8_t raw[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Row r;
  r.rank = (int)cl.block_rank();
  r.ctas = (int)cl.num_blocks();
  const int row = blockIdx.x / r.ctas;
  r.x = reinterpret_cast<const E*>(a.x) + (long long)row * a.stride;
  r.n = a.n;
  r.vec = a.vec;
  r.shift = a.shift;
  r.pow2 = s.pow2;
  SampleShared* lead = cl.map_shared_rank(&s, 0);

  clear_bins(s);
  if (r.rank == 0)
    for (int i = tid; i < kBins; i += kSmpThreads) {
      s.cum_w[i] = 0;
      s.cum_n[i] = 0;
    }
  if (tid < 32) s.pow2[tid] = exp2((double)tid / 32.0);
  if (tid == 0) {
    s.listed = 0;
    s.first = 0xffffffffu;
  }
  // the largest; NaN if there is one
  auto top_nan = [](float x, float y) {
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
  };
  float best = -INFINITY;
  sweep<E>(r, [&](const auto& v, int) {
    constexpr int P = 16 / sizeof(E);
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
  best = -INFINITY;
  for (int c = 0; c < r.ctas; ++c) best = top_nan(best, cl.map_shared_rank(&s, c)->top);
  r.top = best;
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  const bool none = isnan(r.top) || r.top == -INFINITY;   // nothing to choose from
  if (none || !(T > 0.0f)) {
    if (!none) {                                          // the first of the largest
      unsigned at = 0xffffffffu;
      sweep<E>(r, [&](const auto& v, int i) {
        constexpr int P = 16 / sizeof(E);
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
  r.rate = 1.4426950408889634 / (double)T;
  r.scale = fminf(kBinsFold / T, 1e30f);

  const float pf = a.top_p ? a.top_p[row] : 1.0f, mf = a.min_p ? a.min_p[row] : 0.0f;
  const bool by_p = pf < 1.0f, by_m = mf > 0.0f;
  const double p = pf;
  const u64 m = (u64)ceil(fmin((double)mf, 1.0) * (double)(1ull << r.shift));
  u64 wm = 0, wl = 0;                                     // of the tokens that min-p keeps, of the last bin's
  unsigned nm = 0, nl = 0;
  sweep<E>(r, [&](const auto& v, int) {
    constexpr int P = 16 / sizeof(E);
#pragma unroll
    for (int e = 0; e < P; ++e) {
      if (v[e] == -INFINITY) continue;
      const u64 w = r.weight(v[e]);
      if (by_m && w >= m) {
        wm += w;
        ++nm;
      }
      const int b = r.bin(v[e]);
      if (b == kBins - 1) {
        wl += w;
        ++nl;
      } else {
        add_weight(s, b, w);
      }
    }
  });
  for (int o = 16; o > 0; o >>= 1) {
    wl += __shfl_xor_sync(0xffffffffu, wl, o);
    nl += __shfl_xor_sync(0xffffffffu, nl, o);
  }
  if (lane == 0 && nl) add_weight(s, kBins - 1, wl, nl);
  if (by_m) {
    block_sum(s, wm, nm);
    if (tid == 0) {
      s.part_w[0][1] = wm;
      s.part_n[0][1] = nm;
    }
  }
  __syncthreads();
  push_bins(s, lead->cum_w, lead->cum_n);
  cl.sync();
  if (by_m) {
    wm = 0;
    nm = 0;
    for (int c = 0; c < r.ctas; ++c) {
      const SampleShared* o = cl.map_shared_rank(&s, c);
      wm += o->part_w[0][1];
      nm += o->part_n[0][1];
    }
  }
  const int k = a.top_k ? a.top_k[row] : 0;
  if (r.rank == 0) {
    scan_bins(s, s.cum_w, s.cum_n, 0, 0);
    const u64 all = s.cum_w[kBins - 1];
    if (k > 0 && (unsigned)k < s.cum_n[kBins - 1]) find_bin(s.cut[kBinK], {kByCount, (unsigned)k, 0.0}, s.cum_w, s.cum_n, 0, 0);
    else if (by_p) find_bin(s.cut[kBinP], {kReach, 0, p * (double)all}, s.cum_w, s.cum_n, 0, 0);
    if (by_m) find_bin(s.cut[kBinM], {kByCount, nm, 0.0}, s.cum_w, s.cum_n, 0, 0);
  }
  cl.sync();
  const u64 total_w = lead->cum_w[kBins - 1];
  const unsigned total_n = lead->cum_n[kBins - 1];
  const bool by_k = k > 0 && (unsigned)k < total_n;
  const Cut cut_k = {kByCount, (unsigned)k, 0.0};
  float uf = a.u[row];
  uf = uf >= 0.0f ? fminf(uf, 0.99999994f) : 0.0f;        // NaN: 0

  // the bins down to the last cut; a top-p of the top k needs all of those
  int last = kBins - 1;
  unsigned upto = total_n;
  auto down_to = [&](const CutBin& c) {
    if (c.bin < last) {
      last = c.bin;
      upto = c.n0 + c.count;
    }
  };
  if (by_k) down_to(lead->cut[kBinK]);
  else if (by_p) down_to(lead->cut[kBinP]);
  if (by_m && !(by_k && by_p)) down_to(lead->cut[kBinM]);
  if (upto <= kCap) {
    collect<E>(lead, r, [&](float v) { return r.bin(v) <= last; });
    cl.sync();
    if (r.rank == 0) {
      sort_list(s, (int)upto);
      u64 cum[kListed], own[kListed];
      scan_list(s, r, (int)upto, 0, 0, cum, own);
      Found f = {total_n, total_w, 0, 0};                 // of a cut that lies behind the list: min-p's does not
      if (by_k) f = find_listed(s, cum, own, (int)upto, 0, cut_k, f);
      if (by_p) f = find_listed(s, cum, own, (int)upto, 0, {kReach, 0, p * (double)f.w}, f);
      if (by_m && nm < f.n) {
        f.n = nm;
        f.w = wm;
      }
      const unsigned n = f.n;
      const u64 wn = f.w;
      f = find_listed(s, cum, own, (int)upto, 0, {kPass, 0, (double)uf * (double)wn}, f);
      if (tid == 0) {
        a.token[row] = f.index;
        if (a.prob) a.prob[row] = (float)((double)f.own / (double)wn);
        if (a.kept) a.kept[row] = (int)n;
      }
    }
    cl.sync();
    return;
  }
  // one cut after the other
  auto cut_at = [&](const Cut& c) {
    if (r.rank == 0) find_bin(s.cut[kBinP], c, s.cum_w, s.cum_n, 0, 0);
    cl.sync();
    return resolve<E>(cl, s, r, c, lead->cut[kBinP]);
  };
  unsigned n = total_n;
  u64 wn = total_w;
  if (by_k) {
    const CutBin b = lead->cut[kBinK];
    n = (unsigned)k;
    wn = b.w;
    // a bin that ends with the cut, or weighs nothing, need not be looked at
    if (b.n0 + b.count != n && b.w != b.w0) wn = resolve<E>(cl, s, r, cut_k, b).w;
  }
  if (by_p) {
    const Found f = cut_at({kReach, 0, p * (double)wn});
    if (f.n < n) {
      n = f.n;
      wn = f.w;
    }
  }
  if (by_m && nm < n) {
    n = nm;
    wn = wm;
  }
  const Found f = cut_at({kPass, 0, (double)uf * (double)wn});
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
  int ctas = 8;
  while (ctas > 1 && (long long)t->n_rows * ctas > 2 * 148) ctas /= 2;
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
