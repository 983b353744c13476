// paged8_store.cu - rows into an 8-bit paged cache, and back.
//
// Append.  The new rows of a sequence touch blocks of 2^bshift rows; a group of
// W warps takes one block of one head, K or V: the largest magnitude of its new
// rows gives the scale that they need, 2^e (scale_for); a block that holds older
// rows keeps the larger of its own and that, and rounds the older rows anew only
// if it grew.  Elements are x / 2^e (exact) rounded to nearest.  Each source
// element is read once (eight passes of a warp stay in registers) and each byte
// written once, so HBM bounds it (8191 fp16 tokens, 8 heads x 128, K and V: 50 MB
// in 13.4 us, 3.8 TB/s, launch and last wave included; with fp32 arithmetic for
// fp16 rows 17.6); at one token a sequence the chain of loads (sequence, table, row,
// scale) does.
//
// Read.  Rows back as fp32 or fp16: 16 elements a thread, four of them in flight (the
// same tokens in 15 us, 3.4 TB/s; 256 tokens 6.8, where a warp a row took 17.5).
// Expand.  The keys and values of a prompt call's sequences as an fp16 pool in
// a workspace, pages of 128 rows, for the tensor-core kernels; exact, since
// every value is an fp16 number.  1 byte in, 2 out an element: 17 us for 8191 such
// tokens, where the attention that reads them takes 182.
#include <cuda_runtime.h>

#include "paged8.cuh"

namespace tos {

constexpr int kPutWarps = 8;
// Passes of a warp's rows that stay in registers: 32 (fp16: 24) warps an SM then.
template <typename E>
constexpr int kPutPasses = sizeof(E) == 4 ? 4 : 8;

struct PutArgs {
  Pool8 c;
  tosk_rows_t k, v;
  const int *cu, *kv_len;
  int n_tokens, units;                 // units: blocks at most
  int group;                           // warps a block: 1, 2, 4, 8
  int vec;                             // rows and heads on 16-byte pieces of the source, 8 of the cache
};

// N (8) elements of a source row.
template <typename E>
struct Piece8 {
  uint4 u[sizeof(E) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(E) / 2); ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void load(const E* p) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(E) / 2); ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (sizeof(E) == 4) {
      const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
      const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
};

__device__ __forceinline__ uint32_t magnitude(uint32_t m, float x) { return max(m, __float_as_uint(x) & 0x7fffffffu); }
// The largest magnitude of a piece: fp32 bits, or two fp16's.
template <typename E>
__device__ __forceinline__ uint32_t piece_max(uint32_t m, const Piece8<E>& y) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(E) / 2); ++i) {
    const uint32_t w[4] = {y.u[i].x, y.u[i].y, y.u[i].z, y.u[i].w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      m = sizeof(E) == 4 ? max(m, w[e] & 0x7fffffffu) : __vmaxu2(m, w[e] & 0x7fff7fffu);
  }
  return m;
}
// Its eight elements times inv, a power of two, as bytes.  fp16 in pairs, where inv
// is an fp16 number: products are exact, or so small that they become 0 either way;
// I8: 1536 + x rounds x to a whole number, its low byte.
template <int TYPE, typename E>
__device__ __forceinline__ uint2 piece_bytes(const Piece8<E>& y, float inv) {
  if constexpr (sizeof(E) == 2) {
    if (inv <= 32768.0f) {
      const __half2 f = __float2half2_rn(inv);
      const uint32_t w[4] = {y.u[0].x, y.u[0].y, y.u[0].z, y.u[0].w};
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&w[i]), f);
        if constexpr (TYPE == TOSK_I8) {
          x = __hmin2(__hmax2(x, __float2half2_rn(-127.0f)), __float2half2_rn(127.0f));
          x = __hadd2(x, __float2half2_rn(1536.0f));
          h[i] = *reinterpret_cast<const uint32_t*>(&x);
        } else {
          uint16_t b;
          asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(b) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
          h[i] = b;
        }
      }
      if constexpr (TYPE == TOSK_I8) return make_uint2(prmt(h[0], h[1], 0x6420u), prmt(h[2], h[3], 0x6420u));
      return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    }
  }
  float f[8];
  y.get(f);
  return make_uint2(pack_word<TYPE>(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv),
                    pack_word<TYPE>(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv));
}

template <int TYPE, typename E>
__global__ void __launch_bounds__(32 * kPutWarps, sizeof(E) == 4 ? 4 : 3) paged8_put_kernel(const __grid_constant__ PutArgs a) {
  const Pool8& c = a.c;
  __shared__ uint32_t smax[kPutWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp & (a.group - 1);
  pdl_wait();
  pdl_trigger();
  // this group's block, head and kind
  const long long id = ((long long)blockIdx.x * kPutWarps + warp) / a.group;
  const int head = (int)(id % c.n_kv), is_v = (int)(id / c.n_kv & 1), u = (int)(id / c.n_kv / 2);
  const int B = 1 << c.bshift;
  int r0 = 0, r1 = 0, fresh = 1, slot0 = 0, tok0 = 0;     // new rows of the block, its first slot; row r is token tok0 + r
  Row8 at = {-1, 0};
  if (u < a.units) {
    // sequence i's blocks begin at cu[i] / B + 2 i: no two sequences' overlap
    const int i = find_seq(c.n_seqs, u, [&](int x) { return (a.cu[x] >> c.bshift) + 2 * x; });
    const int c0 = a.cu[i], c1 = a.cu[i + 1], q0 = max(c0, 0), q1 = min(c1, a.n_tokens);
    const int base = a.kv_len[i] - (c1 - c0);             // slot of row c0
    const int first = max(base + (q0 - c0), 0);
    slot0 = ((first >> c.bshift) + (u - (c0 >> c.bshift) - 2 * i)) << c.bshift;
    const long long room = (long long)c.table_stride * c.page_size;
    if (c0 >= 0 && q1 > q0 && slot0 >= 0 && slot0 < room) {
      r0 = max(first - slot0, 0);
      r1 = min(base + (q1 - c0) - slot0, B);
      tok0 = c0 - base + slot0;
      fresh = r0 == 0;
      if (r0 < r1) at = row8(c, slot0, c.table[(long long)i * c.table_stride + page_index(c, slot0)]);
      if (at.at < 0) r1 = r0;
    }
  }
  const bool live = r0 < r1;
  const tosk_rows_t& rows = is_v ? a.v : a.k;
  const E* src = reinterpret_cast<const E*>(rows.src) + (long long)tok0 * rows.sstride + head * c.hd;
  uint8_t* dst = (is_v ? c.v : c.k) + at.at + head * c.hd;
  float* sp = (is_v ? c.vs : c.ks) + at.scale + head;
  const long long step = (long long)c.n_kv * c.hd;
  const float old = live && !fresh ? *sp : 0.0f;
  uint32_t m = 0;

  if (a.vec) {
    // LPR lanes a row, RPP rows a pass; the group's warps take passes in turn
    const int pieces = c.hd / 8;
    int lshift = 0;
    while ((1 << lshift) < pieces) ++lshift;
    const int rpp = 32 >> lshift, p = lane & ((1 << lshift) - 1), rr = lane >> lshift;
    const int stride = rpp * a.group, row0 = r0 + sub * rpp + rr;
    const bool has = live && p < pieces;
    constexpr int P = kPutPasses<E>;
    Piece8<E> x[P];
#pragma unroll
    for (int s = 0; s < P; ++s) {
      const int r = row0 + s * stride;
      x[s].zero();
      if (has && r < r1) x[s].load(src + r * rows.sstride + 8 * p);
    }
#pragma unroll
    for (int s = 0; s < P; ++s) m = piece_max(m, x[s]);
    for (int r = row0 + P * stride; has && r < r1; r += stride) {
      Piece8<E> y;
      y.load(src + r * rows.sstride + 8 * p);
      m = piece_max(m, y);
    }
    if constexpr (sizeof(E) == 2) m = __float_as_uint(__half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))));
    m = __reduce_max_sync(0xffffffffu, m);
    if (a.group > 1) {
      if (lane == 0) smax[warp] = m;
      __syncthreads();
      for (int w = warp - sub; w < warp - sub + a.group; ++w) m = max(m, smax[w]);
    }
    const float need = scale_for<TYPE>(m), now = isnan(need) || isnan(old) ? __uint_as_float(0x7fffffffu) : fmaxf(need, old);
    const float inv = 1.0f / now;                         // a power of two
    auto put = [&](const Piece8<E>& y, int r) {
      *reinterpret_cast<uint2*>(dst + r * step + 8 * p) = piece_bytes<TYPE>(y, inv);
    };
#pragma unroll
    for (int s = 0; s < P; ++s) {
      const int r = row0 + s * stride;
      if (has && r < r1) put(x[s], r);
    }
    for (int r = row0 + P * stride; has && r < r1; r += stride) {
      Piece8<E> y;
      y.load(src + r * rows.sstride + 8 * p);
      put(y, r);
    }
    if (live && !fresh && now > old) {                    // the older rows under the larger scale
      const float f = old * inv;
      for (int r = sub * rpp + rr; has && r < r0; r += stride) {
        uint2* w = reinterpret_cast<uint2*>(dst + r * step + 8 * p);
        uint2 q = *w;
        uint32_t h[4];
        cvt_word<TYPE>(q.x, h[0], h[1]);
        cvt_word<TYPE>(q.y, h[2], h[3]);
        float2 g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
        q.x = pack_word<TYPE>(g[0].x * f, g[0].y * f, g[1].x * f, g[1].y * f);
        q.y = pack_word<TYPE>(g[2].x * f, g[2].y * f, g[3].x * f, g[3].y * f);
        *w = q;
      }
    }
    if (live && sub == 0 && lane == 0 && !(now == old)) *sp = now;
    return;
  }

  // an element a lane
  const int n = live ? (r1 - r0) * c.hd : 0;
  for (int x = sub * 32 + lane; x < n; x += 32 * a.group)
    m = magnitude(m, (float)src[(r0 + x / c.hd) * rows.sstride + x % c.hd]);
  m = __reduce_max_sync(0xffffffffu, m);
  if (a.group > 1) {
    if (lane == 0) smax[warp] = m;
    __syncthreads();
    for (int w = warp - sub; w < warp - sub + a.group; ++w) m = max(m, smax[w]);
  }
  const float need = scale_for<TYPE>(m), now = isnan(need) || isnan(old) ? __uint_as_float(0x7fffffffu) : fmaxf(need, old);
  const float inv = 1.0f / now;
  for (int x = sub * 32 + lane; x < n; x += 32 * a.group) {
    const int r = r0 + x / c.hd, d = x % c.hd;
    dst[r * step + d] = (uint8_t)pack_word<TYPE>((float)src[r * rows.sstride + d] * inv, 0.0f, 0.0f, 0.0f);
  }
  if (live && !fresh && now > old)
    for (int x = sub * 32 + lane; x < r0 * c.hd; x += 32 * a.group) {
      uint8_t* w = dst + x / c.hd * step + x % c.hd;
      *w = (uint8_t)pack_word<TYPE>(elem8<TYPE>(*w) * (old * inv), 0.0f, 0.0f, 0.0f);
    }
  if (live && sub == 0 && lane == 0 && !(now == old)) *sp = now;
}

// --------------------------------------------------------------------- read
struct GetArgs {
  Pool8 c;
  tosk_rows_t k, v;
  const int *cu, *kv_len;
  int n_tokens, vec;
  int tokens;                          // a CTA
};

// 16 elements, scaled, to a row of E.  (Values are fp16 numbers: products of pairs
// are exact.)
template <int TYPE, typename E>
__device__ __forceinline__ void put16(E* dst, const uint4& w, float s) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  const __half2 f = __float2half2_rn(s);
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    cvt_word<TYPE>(u[i], h[2 * i], h[2 * i + 1]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&h[2 * i + e]), f);
      h[2 * i + e] = *reinterpret_cast<const uint32_t*>(&x);
    }
  }
  if constexpr (sizeof(E) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * i]));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * i + 1]));
      reinterpret_cast<float4*>(dst)[i] = make_float4(a.x, a.y, b.x, b.y);
    }
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(h[0], h[1], h[2], h[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(h[4], h[5], h[6], h[7]);
  }
}

// A token's row of all heads, by a warp, an element a lane: `row` its place, dst
// its output.
template <int TYPE, typename E>
__device__ __forceinline__ void read_row(const Pool8& c, const Row8& row, const uint8_t* pool, const float* scales, E* dst) {
  for (int x = threadIdx.x & 31; x < c.n_kv * c.hd; x += 32) {
    const float f = row.at < 0 ? 0.0f : elem8<TYPE>(pool[row.at + x]) * scales[row.scale + x / c.hd];
    if constexpr (sizeof(E) == 4) dst[x] = f;
    else dst[x] = __float2half_rn(f);
  }
}

// Rows r < n of K and V, rows[r] their places: 16 elements a thread, kWidePieces
// of them in flight; dst_k, dst_v NULL: not wanted.
constexpr int kWidePieces = 4;
constexpr int kMostPieces = 65535;     // of a CTA's rows: its divisions are products then
__device__ __forceinline__ uint32_t inverse_of(uint32_t d) { return 0xffffffffu / d + 1; }   // d > 1
__device__ __forceinline__ int divide(uint32_t x, uint32_t d, uint32_t inv) { return d == 1 ? x : __umulhi(x, inv); }   // x, d < 2^16
template <int TYPE, typename E>
__device__ __forceinline__ void read_rows(const Pool8& c, const Row8* rows, int n, E* dst_k, long long stride_k, E* dst_v,
                                          long long stride_v) {
  const int side = c.n_kv * c.hd / 16, both = dst_k && dst_v ? 2 * side : side, pieces = n * both, per_head = c.hd / 16;
  const uint32_t inv_both = inverse_of(both), inv_head = inverse_of(per_head);
  for (int p0 = threadIdx.x; p0 < pieces; p0 += 256 * kWidePieces) {
    uint4 w[kWidePieces];
    float s[kWidePieces];
    E* dst[kWidePieces];
#pragma unroll
    for (int x = 0; x < kWidePieces; ++x) {
      const int p = p0 + 256 * x;
      w[x] = make_uint4(0, 0, 0, 0);
      s[x] = 0.0f;
      dst[x] = nullptr;
      if (p < pieces) {
        const int r = divide(p, both, inv_both), q = p - r * both;
        const bool second = q >= side, is_v = !dst_k || second;
        const int e = second ? q - side : q;
        const Row8 row = rows[r];
        if (row.at < -1) continue;
        dst[x] = (is_v ? dst_v + r * stride_v : dst_k + r * stride_k) + e * 16;
        if (row.at >= 0) {
          w[x] = *reinterpret_cast<const uint4*>((is_v ? c.v : c.k) + row.at + e * 16);
          s[x] = (is_v ? c.vs : c.ks)[row.scale + divide(e, per_head, inv_head)];
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kWidePieces; ++x)
      if (dst[x]) put16<TYPE>(dst[x], w[x], s[x]);
  }
}

constexpr int kGetTokens = 128;        // at most, a CTA
template <int TYPE, typename E>
__global__ void __launch_bounds__(256) paged8_get_kernel(const __grid_constant__ GetArgs a) {
  const Pool8& c = a.c;
  __shared__ Row8 rows[kGetTokens];    // at -1: reads as zeros; -2: stays as it is
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * a.tokens, n = min(a.tokens, a.n_tokens - t0);
  for (int r = warp; r < n; r += 8) {
    const int t = t0 + r, i = find_seq(c.n_seqs, t, [&](int x) { return a.cu[x]; });
    const int c0 = a.cu[i], c1 = a.cu[i + 1], slot = a.kv_len[i] - c1 + t;
    Row8 row = {-2, 0};
    if (t >= c0 && t < c1 && slot >= 0 && slot < (long long)c.table_stride * c.page_size)
      row = row8(c, slot, c.table[(long long)i * c.table_stride + page_index(c, slot)]);
    if (lane == 0) rows[r] = row;
  }
  __syncthreads();
  E* k = a.k.dst ? reinterpret_cast<E*>(a.k.dst) + t0 * a.k.dstride : nullptr;
  E* v = a.v.dst ? reinterpret_cast<E*>(a.v.dst) + t0 * a.v.dstride : nullptr;
  if (a.vec) {
    read_rows<TYPE>(c, rows, n, k, a.k.dstride, v, a.v.dstride);
    return;
  }
  for (int r = warp; r < n; r += 8) {
    if (rows[r].at < -1) continue;
    if (k) read_row<TYPE>(c, rows[r], c.k, c.ks, k + r * a.k.dstride);
    if (v) read_row<TYPE>(c, rows[r], c.v, c.vs, v + r * a.v.dstride);
  }
}

// ------------------------------------------------------------------- expand
constexpr int kWideRows = 128;         // rows of a page of the fp16 pool

struct WideArgs {
  Pool8 c;
  const int* kv_len;
  __half *k, *v;
  int* table;                          // [n_seqs][stride]: the fp16 pool's pages
  int stride, max_kv, cap;             // cap: pages of the fp16 pool, and of the grid
  int keys;                            // a CTA, a power of two
  int vec;
};

template <int TYPE>
__global__ void __launch_bounds__(256) paged8_wide_kernel(const __grid_constant__ WideArgs a) {
  const Pool8& c = a.c;
  __shared__ int sseq, sfirst, swarp[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  const long long room = (long long)c.table_stride * c.page_size;
  auto keys = [&](int s) {
    const int n = min(a.kv_len[s], a.max_kv);
    return (int)max(0ll, min((long long)n, room));
  };
  // the sequence of page pg: sequences' pages lie one behind the other
  const int parts = kWideRows / a.keys, pg = blockIdx.x / parts, part = blockIdx.x % parts;
  // where the pool has no room for all of them, the last CTA makes the table say so:
  // an earlier call's page numbers may lie there
  const bool marks = blockIdx.x == gridDim.x - 1;
  if (tid == 0) sseq = -1;
  int before = 0;
  for (int s0 = 0; s0 < c.n_seqs; s0 += 256) {
    const int s = s0 + tid, n = s < c.n_seqs ? (keys(s) + kWideRows - 1) / kWideRows : 0;
    int sum = n;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += v;
    }
    __syncthreads();
    if (lane == 31) swarp[warp] = sum;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < 8; ++w) {
      if (w < warp) sum += swarp[w];
      all += swarp[w];
    }
    sum += before;
    if (n > 0 && pg >= sum - n && pg < sum) {
      sseq = s;
      sfirst = sum - n;
    }
    before += all;
    if (marks) {
      for (uint32_t over = __ballot_sync(0xffffffffu, n > 0 && sum > a.cap); over; over &= over - 1) {
        const int o = __ffs(over) - 1, no = __shfl_sync(0xffffffffu, n, o), first = __shfl_sync(0xffffffffu, sum, o) - no;
        int* row = a.table + (long long)(s0 + warp * 32 + o) * a.stride;
        for (int j = max(0, a.cap - first) + lane; j < no; j += 32) row[j] = -1;
      }
      before = min(before, a.cap);                        // 32 bits may not hold them all
    } else if (before > pg) {                             // the same for every thread
      break;
    }
  }
  __syncthreads();
  const int seq = sseq;
  if (seq < 0) return;
  const int j = pg - sfirst, n = keys(seq);
  if (part == 0 && tid == 0) a.table[(long long)seq * a.stride + j] = pg;
  const int* table = c.table + (long long)seq * c.table_stride;
  const long long width = (long long)c.n_kv * c.hd;
  const int r0 = part * a.keys, key0 = j * kWideRows + r0, have = min(a.keys, n - key0);
  const long long to = ((long long)pg * kWideRows + r0) * width;
  __shared__ Row8 rows[kWideRows];
  if (tid < have) rows[tid] = row8(c, key0 + tid, table[page_index(c, key0 + tid)]);
  __syncthreads();
  if (a.vec) {
    read_rows<TYPE>(c, rows, have, a.k + to, width, a.v + to, width);
    return;
  }
  for (int r = warp; r < have; r += 8) {
    read_row<TYPE>(c, rows[r], c.k, c.ks, a.k + to + r * width);
    read_row<TYPE>(c, rows[r], c.v, c.vs, a.v + to + r * width);
  }
}

}  // namespace tos

using namespace tos;

namespace {

int launch8(const void* f, long long grid, int threads, const void* arg, cudaStream_t st) {
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<void*>(arg)};
  return (int)cudaLaunchKernelExC(&cfg, f, args);
}

bool few_pieces(int rows, const tosk_paged8_t& kv) { return (long long)rows * kv.n_kv * kv.hd / 8 <= kMostPieces; }

// Rows that a CTA of 256 threads reads back, a power of two up to 128: as many as
// give four CTAs an SM, so that few rows go to many CTAs and of many rows a CTA's
// beginning is soon paid for; but no more than its 16-byte pieces may be (40,000
// rows of 32 heads x 128: 64 a CTA 188 us; 128, which goes an element a lane, 1546).
int rows_a_cta(long long rows, const tosk_paged8_t& kv) {
  int n = 1;
  while (n < 128 && n * 4 * 148 < rows && few_pieces(2 * n, kv)) n *= 2;
  return n;
}

bool rows_on(const void* p, long long stride, int type, int bytes) {
  return ((uintptr_t)p & (bytes - 1)) == 0 && stride * (type == TOSK_F32 ? 4 : 2) % bytes == 0;
}

}  // namespace

namespace tos {

Pool8 pool8_of(const tosk_paged8_t& kv) {
  Pool8 c;
  c.k = (uint8_t*)kv.k; c.v = (uint8_t*)kv.v;
  c.ks = kv.k_scale; c.vs = kv.v_scale;
  c.n_pages = kv.n_pages; c.page_size = kv.page_size;
  c.pshift = -1;
  c.bshift = 0;
  for (int i = 0; i < 31; ++i) {
    if (kv.page_size == 1 << i) c.pshift = i;
    if (kv.block == 1 << i) c.bshift = i;
  }
  c.bpp = kv.page_size / kv.block;
  c.n_kv = kv.n_kv; c.hd = kv.hd;
  c.table = kv.table; c.n_seqs = kv.n_seqs; c.table_stride = kv.table_stride;
  return c;
}

}  // namespace tos

extern "C" int tosk_paged8_put(const tosk_paged8_io_t* io, cudaStream_t st) {
  PutArgs a;
  a.c = pool8_of(io->kv);
  a.c.n_seqs = io->n_seqs;
  a.k = io->k; a.v = io->v;
  a.cu = io->cu; a.kv_len = io->kv_len;
  a.n_tokens = io->n_tokens;
  const long long units = (io->n_tokens >> a.c.bshift) + 2ll * io->n_seqs;
  if (units > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  a.units = (int)units;
  const int type = io->k.stype;
  a.vec = io->kv.hd % 8 == 0 && rows_on(io->k.src, io->k.sstride, type, 16) && rows_on(io->v.src, io->v.sstride, type, 16) &&
          (io->kv.hd * (type == TOSK_F32 ? 4 : 2)) % 16 == 0;
  // warps a block: as many as keep their rows in registers
  const long long elems = (long long)io->kv.block * io->kv.hd;
  a.group = 1;
  const int passes = type == TOSK_F32 ? kPutPasses<float> : kPutPasses<__half>;
  while (a.group < kPutWarps && elems > (long long)a.group * passes * 256) a.group *= 2;
  const long long groups = units * io->kv.n_kv * 2, grid = (groups * a.group + kPutWarps - 1) / kPutWarps;
  const void* f = io->kv.type == TOSK_I8
                      ? type == TOSK_F32 ? (const void*)paged8_put_kernel<TOSK_I8, float> : (const void*)paged8_put_kernel<TOSK_I8, __half>
                      : type == TOSK_F32 ? (const void*)paged8_put_kernel<TOSK_F8, float> : (const void*)paged8_put_kernel<TOSK_F8, __half>;
  return launch8(f, grid, 32 * kPutWarps, &a, st);
}

extern "C" int tosk_paged8_get(const tosk_paged8_io_t* io, cudaStream_t st) {
  GetArgs a;
  a.c = pool8_of(io->kv);
  a.c.n_seqs = io->n_seqs;
  a.k = io->k; a.v = io->v;
  a.cu = io->cu; a.kv_len = io->kv_len;
  a.n_tokens = io->n_tokens;
  const int type = io->k.dst ? io->k.dtype : io->v.dtype;
  a.tokens = rows_a_cta(io->n_tokens, io->kv);
  a.vec = io->kv.hd % 16 == 0 && few_pieces(a.tokens, io->kv) && rows_on(io->k.dst, io->k.dstride, type, 16) &&
          rows_on(io->v.dst, io->v.dstride, type, 16);
  const void* f = io->kv.type == TOSK_I8
                      ? type == TOSK_F32 ? (const void*)paged8_get_kernel<TOSK_I8, float> : (const void*)paged8_get_kernel<TOSK_I8, __half>
                      : type == TOSK_F32 ? (const void*)paged8_get_kernel<TOSK_F8, float> : (const void*)paged8_get_kernel<TOSK_F8, __half>;
  return launch8(f, ((long long)io->n_tokens + a.tokens - 1) / a.tokens, 256, &a, st);
}

namespace {
long long wide_pages(int n_seqs, long long total_kv) { return total_kv / kWideRows + n_seqs; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
size_t wide_pool_bytes(long long pages, int n_kv, int hd) { return up256((size_t)pages * kWideRows * n_kv * hd * 2); }
}  // namespace

extern "C" size_t tosk_paged8_wide_bytes(int n_seqs, long long total_kv, int max_kv, int n_kv, int hd) {
  return 2 * wide_pool_bytes(wide_pages(n_seqs, total_kv), n_kv, hd) +
         up256((size_t)n_seqs * ((size_t)max_kv / kWideRows + 1) * 4);
}

extern "C" int tosk_paged8_wide(const tosk_paged8_t* kv, const int* kv_len, int n_seqs, long long total_kv, int max_kv, void* ws,
                                tosk_paged_t* out, cudaStream_t st) {
  const long long pages = wide_pages(n_seqs, total_kv);
  const int keys = rows_a_cta(total_kv, *kv);
  if (pages > 0x7fffffffll / (kWideRows / keys)) return (int)cudaErrorInvalidValue;
  const size_t pool = wide_pool_bytes(pages, kv->n_kv, kv->hd);
  WideArgs a;
  a.c = pool8_of(*kv);
  a.c.n_seqs = n_seqs;
  a.kv_len = kv_len;
  a.k = reinterpret_cast<__half*>(ws);
  a.v = reinterpret_cast<__half*>(reinterpret_cast<uint8_t*>(ws) + pool);
  a.table = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(ws) + 2 * pool);
  a.stride = max_kv / kWideRows + 1;
  a.max_kv = max_kv;
  a.cap = (int)pages;
  a.keys = keys;
  a.vec = kv->hd % 16 == 0 && few_pieces(keys, *kv);
  memset(out, 0, sizeof(*out));
  out->k = a.k; out->v = a.v;
  out->type = TOSK_F16;
  out->n_pages = (int)pages;
  out->page_size = kWideRows;
  out->n_kv = kv->n_kv; out->hd = kv->hd;
  out->table = a.table;
  out->n_seqs = n_seqs;
  out->table_stride = a.stride;
  const void* f = kv->type == TOSK_I8 ? (const void*)paged8_wide_kernel<TOSK_I8> : (const void*)paged8_wide_kernel<TOSK_F8>;
  return launch8(f, pages * (kWideRows / keys), 256, &a, st);
}
