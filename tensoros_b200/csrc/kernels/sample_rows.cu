// sample_rows.cu - a token for every row of logits, by temperature, top-k,
// top-p and min-p from given random numbers.
//
//   w_i = exp((x_i - max) / T), tokens in order of falling x, then rising index;
//   the first n stay: n <= top_k, n the least whose w's sum reaches top_p of the
//   top k's, w >= min_p; the token is the first whose sum passes u times theirs.
//
// All three filters and the draw cut one order, so nothing is sorted but what
// lies around a cut.  A cluster of up to eight CTAs takes a row:
//   max (and argmax)  ->  histogram of (max - x) / T, 64 bins an e-fold: counts
//   and weights  ->  prefix sums in the cluster's first CTA give the bins of the
//   cuts  ->  the bins down to the last cut, if they hold at most kCap tokens,
//   or else the bins of the cuts one after the other, go to the first CTA's
//   shared memory, are sorted there and resolved.
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
  unsigned lo[kBins], hi[kBins], cnt[kBins];     // a histogram: weights in two words, counts
  u64 list[kCap];                       // first CTA: tokens to sort, value over inverted index
  double pow2[32];
  u64 wsum[kSmpThreads / 32];
  unsigned wcnt[kSmpThreads / 32];
  u64 part_w[2][2];                     // this CTA's sums, two rounds apart
  unsigned part_n[2][2];
  u64 best[kSmpThreads / 32];
  u64 top;                              // this CTA's best token
  int nan;
  unsigned listed;
  u64 total_w;                          // first CTA
  unsigned total_n;
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
    return min(__float2int_rd((place(v) - (float)b) * kBins), kBins - 1);
  }
  // 2^(shift - (top - v) rate) to the nearest whole number: 2^(n/32) from a
  // table, 2^r, |r| <= 1/64, by its Taylor sum (next term 2e-15)
  __device__ __forceinline__ u64 weight(float v) const {
    if (v == top) return 1ull << shift;
    const double y = fma(-((double)top - (double)v), rate, (double)shift);
    if (!(y > -2.0)) return 0;
    const int m = __double2int_rn(y * 32.0);
    const double r = fma((double)m, -1.0 / 32, y) * 0.6931471805599453;
    double p = fma(r, 1.0 / 120, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0) * pow2[m & 31];
    return __double2ull_rn(__longlong_as_double(__double_as_longlong(p) + ((long long)(m >> 5) << 52)));
  }
};

// f(value, index, valid) of this CTA's elements; a warp's lanes go together.
template <typename E, typename F>
__device__ __forceinline__ void sweep(const Row& r, F f) {
  constexpr int P = 16 / sizeof(E), U = 2;
  const int pieces = (r.n + P - 1) / P, lane = threadIdx.x & 31;
  const E* x = reinterpret_cast<const E*>(r.x);
  for (int p0 = r.rank * kSmpThreads + (threadIdx.x & ~31); p0 < pieces; p0 += U * r.ctas * kSmpThreads) {
    float v[U][P];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = (p0 + q * r.ctas * kSmpThreads + lane) * P;
      if (r.vec && i + P <= r.n) {
        const uint4 w = *reinterpret_cast<const uint4*>(x + i);
        if constexpr (sizeof(E) == 4) {
          v[q][0] = __uint_as_float(w.x); v[q][1] = __uint_as_float(w.y);
          v[q][2] = __uint_as_float(w.z); v[q][3] = __uint_as_float(w.w);
        } else {
          const uint32_t h[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
            v[q][2 * e] = g.x;
            v[q][2 * e + 1] = g.y;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < P; ++e) v[q][e] = i >= 0 && i + e < r.n ? (float)x[i + e] : 0.0f;
      }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const int i = (p0 + q * r.ctas * kSmpThreads + lane) * P;
#pragma unroll
      for (int e = 0; e < P; ++e) f(v[q][e], i + e, i >= 0 && i + e < r.n);
    }
  }
}

__device__ __forceinline__ void add_weight(SampleShared& s, int b, u64 w) {
  atomicAdd(&s.cnt[b], 1u);
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

// First CTA: the sums of all CTAs' bins this thread has (kPerThread neighbours),
// inclusive within the thread.
__device__ __forceinline__ void merge_bins(cg::cluster_group& cl, SampleShared& s, u64 (&w)[kPerThread], unsigned (&n)[kPerThread]) {
  const int b0 = threadIdx.x * kPerThread;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) w[i] = n[i] = 0;
  for (unsigned c = 0; c < cl.num_blocks(); ++c) {
    const SampleShared* o = cl.map_shared_rank(&s, c);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      w[i] += (u64)o->hi[b0 + i] << 32;
      w[i] += o->lo[b0 + i];
      n[i] += o->cnt[b0 + i];
    }
  }
#pragma unroll
  for (int i = 1; i < kPerThread; ++i) {
    w[i] += w[i - 1];
    n[i] += n[i - 1];
  }
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

// First CTA: the first bin past the cut; w, n: the sums before this thread's bins
// and theirs, inclusive.
__device__ __forceinline__ void find_bin(CutBin& to, const Cut& c, u64 w0, unsigned n0, const u64 (&w)[kPerThread],
                                         const unsigned (&n)[kPerThread]) {
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const u64 wb = w0 + (i ? w[i - 1] : 0);
    const unsigned nb = n0 + (i ? n[i - 1] : 0);
    if (n0 + n[i] > nb && past(c, n0 + n[i], w0 + w[i]) && (nb == 0 || !past(c, nb, wb)))
      to = {(int)threadIdx.x * kPerThread + i, nb, n0 + n[i] - nb, wb, w0 + w[i]};
  }
}

// Tokens for which keep(value) go to the first CTA's list.
template <typename E, typename F>
__device__ __forceinline__ void collect(cg::cluster_group& cl, SampleShared& s, const Row& r, F keep) {
  SampleShared* lead = cl.map_shared_rank(&s, 0);
  const int lane = threadIdx.x & 31;
  sweep<E>(r, [&](float v, int i, bool valid) {
    const bool take = valid && v > -INFINITY && keep(v);
    const unsigned hit = __ballot_sync(0xffffffffu, take);
    if (hit == 0) return;
    unsigned at = 0;
    if (lane == 0) at = atomicAdd(&lead->listed, (unsigned)__popc(hit));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(hit & ((1u << lane) - 1));
    if (take && at < kCap) lead->list[at] = (u64)order_key(v) << 32 | ~(unsigned)i;
  });
}

// Count and weight over the row of the tokens for which keep(value, index), the
// same in every CTA.  round: 0, 1 in turn.
template <typename E, typename F>
__device__ __forceinline__ void count_row(cg::cluster_group& cl, SampleShared& s, const Row& r, int round, F keep, u64& w,
                                          unsigned& n) {
  w = 0;
  n = 0;
  sweep<E>(r, [&](float v, int i, bool valid) {
    if (valid && v > -INFINITY && keep(v, i)) {
      w += r.weight(v);
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
    __syncthreads();
    sweep<E>(r, [&](float v, int, bool valid) {
      if (valid && v > -INFINITY && r.bin(v) == b) add_weight(s, r.fine(v, b), r.weight(v));
    });
    cl.sync();
    if (r.rank == 0) {
      u64 w[kPerThread], all;
      unsigned n[kPerThread], alln;
      merge_bins(cl, s, w, n);
      u64 sum = w[kPerThread - 1];
      unsigned sn = n[kPerThread - 1];
      block_scan(s, sum, sn, all, alln);
      // nb == 0 in find_bin stands for the very first token: past is monotone, so
      // with tokens before the bin the test of what comes before holds
      find_bin(s.cut[kBinK], c, at.w0 + sum - w[kPerThread - 1], at.n0 + sn - n[kPerThread - 1], w, n);
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
    collect<E>(cl, s, r, mine);
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
__global__ void __launch_bounds__(kSmpThreads, 1) sample_rows_kernel(const __grid_constant__ SampleArgs a) {
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
  if (tid < 32) s.pow2[tid] = exp2((double)tid / 32.0);
  if (tid == 0) {
    s.listed = 0;
    s.nan = 0;
  }
  __syncthreads();
  // the largest, and the first of its kind
  float best = -INFINITY;
  int at = 0x7fffffff;
  bool nan = false;
  sweep<E>(r, [&](float v, int i, bool valid) {
    if (!valid) return;
    nan |= isnan(v);
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  });
  u64 top = (u64)order_key(best) << 32 | ~(unsigned)at;
  for (int o = 16; o > 0; o >>= 1) {
    const u64 b = __shfl_xor_sync(0xffffffffu, top, o);
    top = b > top ? b : top;
  }
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) {
    s.best[warp] = top;
    if (nan) s.nan = 1;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSmpThreads / 32; ++i) top = s.best[i] > top ? s.best[i] : top;
    s.top = top;
  }
  cl.sync();
  top = 0;
  nan = false;
  for (int c = 0; c < r.ctas; ++c) {
    const SampleShared* o = cl.map_shared_rank(&s, c);
    const u64 b = o->top;
    top = b > top ? b : top;
    nan |= o->nan != 0;
  }
  r.top = key_value((unsigned)(top >> 32));
  const float T = a.temperature ? a.temperature[row] : 1.0f;
  const bool none = nan || r.top == -INFINITY;            // nothing to choose from
  if (none || !(T > 0.0f)) {
    if (r.rank == 0 && tid == 0) {
      a.token[row] = none ? -1 : (int)~(unsigned)top;
      if (a.prob) a.prob[row] = none ? 0.0f : 1.0f;
      if (a.kept) a.kept[row] = none ? 0 : 1;
    }
    cl.sync();                                            // nobody leaves while its memory is read
    return;
  }
  r.rate = 1.4426950408889634 / (double)T;
  r.scale = fminf(64.0f / T, 1e30f);

  const float pf = a.top_p ? a.top_p[row] : 1.0f, mf = a.min_p ? a.min_p[row] : 0.0f;
  const bool by_p = pf < 1.0f, by_m = mf > 0.0f;
  const double p = pf, m = fmin((double)mf, 1.0) * (double)(1ull << r.shift);
  u64 wm = 0;
  unsigned nm = 0;
  sweep<E>(r, [&](float v, int, bool valid) {
    if (!valid || v == -INFINITY) return;
    const u64 w = r.weight(v);
    if (by_m && (double)w >= m) {
      wm += w;
      ++nm;
    }
    add_weight(s, r.bin(v), w);
  });
  if (by_m) {
    block_sum(s, wm, nm);
    if (tid == 0) {
      s.part_w[0][1] = wm;
      s.part_n[0][1] = nm;
    }
  }
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
  // what this thread of the first CTA has of the bins' sums
  u64 bw[kPerThread] = {}, bw0 = 0, total_w = 0;
  unsigned bn[kPerThread] = {}, bn0 = 0, total_n = 0;
  if (r.rank == 0) {
    merge_bins(cl, s, bw, bn);
    bw0 = bw[kPerThread - 1];
    bn0 = bn[kPerThread - 1];
    block_scan(s, bw0, bn0, total_w, total_n);
    bw0 -= bw[kPerThread - 1];
    bn0 -= bn[kPerThread - 1];
    if (tid == 0) {
      s.total_w = total_w;
      s.total_n = total_n;
    }
    if (k > 0 && (unsigned)k < total_n) find_bin(s.cut[kBinK], {kByCount, (unsigned)k, 0.0}, bw0, bn0, bw, bn);
    else if (by_p) find_bin(s.cut[kBinP], {kReach, 0, p * (double)total_w}, bw0, bn0, bw, bn);
    if (by_m) find_bin(s.cut[kBinM], {kByCount, nm, 0.0}, bw0, bn0, bw, bn);
  }
  cl.sync();
  total_w = lead->total_w;
  total_n = lead->total_n;
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
    collect<E>(cl, s, r, [&](float v) { return r.bin(v) <= last; });
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
    if (r.rank == 0) find_bin(s.cut[kBinP], c, bw0, bn0, bw, bn);
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
  a.shift = 62 - lg;
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
