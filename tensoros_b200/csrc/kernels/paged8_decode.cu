// paged8_decode.cu - attention of one token a sequence over an 8-bit paged
// cache.
//
//   s_j = c 2^a(j) (q . k_j),  w_j = 2^(s_j - m),  o = sum_j w_j (2^b(j) v_j) / sum_j w_j
//
// with k_j, v_j as stored and 2^a, 2^b the scales of key j's block.  A CTA takes a
// piece of one sequence's keys for one key/value head and 8 or 16 query heads of
// its group; its four warps take every fourth step of 32 keys each and run alone
// until the end.  A step's K and V rows come by TMA (boxes of 16 rows of one head;
// where pages do not hold whole groups of 16, and where there is little to read,
// by cp.async) into the warp's own ring in shared memory, their scales by cp.async.
//
// Products are mma.sync, whose operands are made from the bytes in registers: a
// tile has 8 or 16 query rows, and tcgen05 would want 128 and its bytes as fp16 in
// shared memory.  All of it is exact but for the roundings of fp32:
//   I8 scores: 8-bit integer products of the bytes as they are with q as whole
//      numbers of 31 bits in four signed bytes, rows g and g + 8 of two tiles;
//   F8 scores: bytes to fp16, q as two-part fp16 numbers, rows g and g + 8;
//   sums: bytes to fp16 with their scale, which is a power of two (I8: one fma
//      takes off the conversion's offset and scales; F8: one product), weights as
//      two-part fp16 numbers.  Two products of 16 keys a chain, the sums over
//      the steps in fp32 registers.
// Operands are read in the order that suits bytes: a contraction may run over its
// dims or keys, and a product's columns over dims, in any order that both sides
// keep.  Lane (g, t) reads 16 dims of key g at once (two pieces: 2t, 2t + 1), q is
// laid out likewise; of V 8 dims of its four keys 2t, 2t + 1, 2t + 8, 2t + 9, and
// bytes of two keys are paired by prmt: column g of product j has dim 16 g + j.
//
// Bound: HBM.  Long sequences stream at 5.5 (I8) and 5.9 TB/s (F8) of the 6.05
// that the copies alone reach; a call costs 7.4 us beside (12 at first: the joining
// of the warps met one bank with all lanes, queries were split bit by bit).
// Sixteen sequences of 1 to 4096 keys, 32 / 32 heads x 128, I8: 57.4 us, 4.3 TB/s;
// four of 9,999 to 32,768, 32 / 8, F8: 49.4 us, 3.9 TB/s, 6.3 of them the joining.
#include <cuda_runtime.h>
#include <string.h>

#include <type_traits>

#include "paged8.cuh"
#include "paged_tc.cuh"

namespace tos {

constexpr int kD8Warps = 4;

struct Dec8Args {
  CUtensorMap mk, mv;             // [page][row][kv head][dim]: boxes of 16 rows x 128 (64) dims
  PagedProblem p;
  Pool8 c;
  int rtiles;                                                     // row tiles of a group
  int even, pieces;                                               // all keys shared evenly; or see share_out; or chunks
  int* counts;                                                    // with one of those: how many pieces every row has
  int q_vec;                                                      // four q elements are aligned
};

// A warp's step has 32 keys.  Its ring holds three tiles, K and V of the steps in
// turn, so that two of them are always on their way: after the scores of step s
// V of s + 1 is asked for in the place of K of s, after its sums K of s + 2 in
// that of V of s.  Steps of 16 keys took 89 us where steps of 32 took 71.
constexpr int kD8Step = 32;
template <int HD, int NQ>
struct Dec8Shape {
  static constexpr int kTile = kD8Step * HD;                      // bytes of a step's K or V
  static constexpr int kRing = kD8Warps * 3 * kTile;
  static constexpr int kQ = NQ * (HD / 16) * 512;                 // the queries' fragments: registers would spill
  static constexpr int kScales = kD8Warps * 3 * kD8Step * 4;      // of every tile's keys
  static constexpr int kSmem = kRing + kQ + kScales + kD8Warps * 3 * 8;
};

// Byte offset of piece c (16 bytes) of key r in a tile, as TMA swizzles it: rows of
// 128 bytes (256 dims: two such tiles), piece c at c ^ (r & 7); 64 dims: of 64,
// at c ^ (r / 2 & 3).  What is read together then lies in different banks: of
// K, by a quarter warp, pieces 2t + i of two keys; of V, by half a warp, 8 bytes
// of 4 pieces of the four keys 2t, of pieces 2, 3, 6, 7 the other half (64 dims:
// two and two share banks).
template <int HD>
__device__ __forceinline__ uint32_t piece_off(int r, int c) {
  return (uint32_t)(HD == 64 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4)
                             : (c >> 3) * (kD8Step * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
// The piece that a lane reads of K in round i.
template <int HD>
__device__ __forceinline__ int k_piece(int t4, int i) {
  return HD == 64 ? t4 : 8 * (i >> 1) + 2 * t4 + (i & 1);
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool have) {
  const int n = have ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* m, int dim, int head, int row, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(m), "r"(dim), "r"(head), "r"(row), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool have) {
  const int n = have ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void mma_h(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_h_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_i(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool first) {
  if (first)
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
  else
    asm(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// volatile: in the order written, or the compiler has all of a step's words in registers at once
template <int N>
__device__ __forceinline__ void lds(uint32_t at, uint32_t (&w)[N]) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
  else
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// Two half2 (x: key a's element, y: key b's) of the first or the second two of
// four dims, scaled by mul.  I8: add is -1152 times the scales, or with BIG,
// where a scale makes that no fp16 number, -1152.
template <int TYPE, bool BIG>
__device__ __forceinline__ void pair_keys(uint32_t a, uint32_t b, int half, __half2 mul, __half2 add, uint32_t (&h)[2]) {
  const uint32_t w = prmt(a, b, half ? 0x7362u : 0x5140u);        // {a0 b0 a1 b1}, or of 2 and 3
  if constexpr (TYPE == TOSK_I8) {
    const uint32_t x = w ^ 0x80808080u, m = 0x64646464u;
    h[0] = prmt(x, m, 0x4140u);
    h[1] = prmt(x, m, 0x4342u);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      h[i] = as_u32(BIG ? __hmul2(__hadd2(as_h2(h[i]), add), mul) : __hfma2(as_h2(h[i]), mul, add));
  } else {
    cvt_word<TYPE>(w, h[0], h[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) h[i] = as_u32(__hmul2(as_h2(h[i]), mul));
  }
}

// Keys that fill the GPU: every CTA takes an even share of all of them, whatever
// the sequences' lengths.  The keys of all sequences, in blocks of 128, lie in one
// line, for each kind of work over them (key/value head, row tile) once, a
// sequence's kinds one behind the other; CTA j has blocks [j W, (j + 1) W), as
// pieces of one or more (sequence, kind)s.  Before each one's blocks lie
// kPieceCost more that are none: what beginning and ending a piece takes (16
// sequences of 1 to 4096 keys, 32 heads, us: 2: 58.4; 4: 61; 8: 66).
constexpr int kShareSeqs = 1024;        // sequences up to which a CTA adds them up itself
constexpr int kPieceCost = 2;
struct Walk8 {
  int at, end, first, share;            // blocks: the next, the last + 1, where sequence `seq` begins; W
  int seq;
  int sums[kD8Warps];
};
struct Piece8Work {
  int seq, kind, k0, k1, index, count;  // seq < 0: no more; piece `index` of `count`
  int at, first;                        // the walk's next
};
// (an empty sequence has a block too, or nobody would write its zeros)
__device__ __forceinline__ int blocks_of(int keys) { return max(1, (keys + 127) >> 7) + kPieceCost; }

// Fewer and longer sequences (four pieces each or more): with B pieces for each
// kind, n sequences and N blocks in all, pieces of N / (B - n) blocks are never
// more than B, and a sequence's are made equal; a CTA has one.  (4 sequences of
// 9,999 to 32,768 keys, 32 / 8 heads, us: 48.7, in even shares, which cost many a
// CTA a second piece, 54.4; the sixteen above 68.4, 57.4.)
constexpr int kShareLeast = 4;          // blocks a piece
struct Share8 {
  int seq, kind, index, count, keys;    // seq < 0: no piece; piece `index` of `count` of its keys
  int sums[kD8Warps];
};
// (inclusive sum over the threads up to this one, sum over all)
__device__ __forceinline__ int2 block_sums(int v, int* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = v;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int i = 0; i < kD8Warps; ++i) {
    if (i < warp) v += sums[i];
    all += sums[i];
  }
  return make_int2(v, all);
}
template <typename F>
__device__ __forceinline__ bool begin_walk(Walk8& w, int n_seqs, int kinds, F keys_of) {
  constexpr int N = kShareSeqs / (32 * kD8Warps);
  int len[N], sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = threadIdx.x + i * 32 * kD8Warps;
    len[i] = s < n_seqs ? blocks_of(keys_of(s)) : 0;      // the order is the threads': any will do
    sum += len[i];
  }
  const int2 all = block_sums(sum, w.sums);
  const int total = all.y * kinds, share = (total + (int)gridDim.x - 1) / (int)gridDim.x, at = (int)blockIdx.x * share;
  if (at >= total) return false;
  int first = (all.x - sum) * kinds;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (at >= first && at < first + len[i] * kinds) {
      w.at = at;
      w.end = min(at + share, total);
      w.first = first;
      w.share = share;
      w.seq = threadIdx.x + i * 32 * kD8Warps;
    }
    first += len[i] * kinds;
  }
  __syncthreads();
  return true;
}
// The next sequence of a walk: thread by thread.
__device__ __forceinline__ int walk_next(int seq, int n_seqs) {
  constexpr int T = 32 * kD8Warps;
  if (seq + T < n_seqs) return seq + T;
  return seq % T + 1 < min(T, n_seqs) ? seq % T + 1 : -1;
}
// The same by every thread.
template <typename F>
__device__ __forceinline__ Piece8Work next_piece(const Walk8& w, int n_seqs, int kinds, F keys_of) {
  Piece8Work x;
  x.seq = w.seq;
  x.at = w.at;
  x.first = w.first;
  while (x.at < w.end) {
    int keys = keys_of(x.seq), len = blocks_of(keys);
    if (x.at >= x.first + len * kinds) {                  // the sequence is done
      x.first += len * kinds;
      x.seq = walk_next(x.seq, n_seqs);
      if (x.seq < 0) return x;
      keys = keys_of(x.seq);
      len = blocks_of(keys);
    }
    x.kind = (x.at - x.first) / len;
    const int begin = x.first + x.kind * len, stop = min(begin + len, w.end);
    const int b0 = max(0, x.at - begin - kPieceCost), b1 = stop - begin - kPieceCost;
    x.at = stop;
    if (b1 <= b0) continue;
    const int cta0 = (begin + kPieceCost) / w.share, cta1 = (begin + len - 1) / w.share;
    x.k0 = b0 * 128;
    x.k1 = min(keys, b1 * 128);
    x.index = (int)blockIdx.x - cta0;
    x.count = cta1 - cta0 + 1;
    return x;
  }
  x.seq = -1;
  return x;
}

template <typename F>
__device__ __forceinline__ void share_out(Share8& w, int n_seqs, int kinds, int pieces, F keys_of) {
  constexpr int N = kShareSeqs / (32 * kD8Warps);
  int keys[N], sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = threadIdx.x + i * 32 * kD8Warps;
    keys[i] = s < n_seqs ? keys_of(s) : -1;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) sum += keys[i] < 0 ? 0 : (keys[i] + 127) >> 7;
  const int all = block_sums(sum, w.sums).y, c = max(kShareLeast, (all + pieces - n_seqs - 1) / (pieces - n_seqs)) * 128;
  if (threadIdx.x == 0) w.seq = -1;
  int got[N];
  sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    got[i] = keys[i] < 0 ? 0 : max(1, (keys[i] + c - 1) / c);
    sum += got[i];
  }
  int at = (block_sums(sum, w.sums).x - sum) * kinds;     // the first CTA of this thread's sequences
  const int me = blockIdx.x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (me >= at && me < at + got[i] * kinds) {
      w.seq = threadIdx.x + i * 32 * kD8Warps;
      w.kind = (me - at) % kinds;                         // neighbours read the same pages' other heads
      w.index = (me - at) / kinds;
      w.count = got[i];
      w.keys = keys[i];
    }
    at += got[i] * kinds;
  }
  __syncthreads();
}

// Four CTAs an SM at 128 registers a thread: sixteen warps (twelve, with 168: 4.1
// TB/s over long sequences, sixteen 5.5; with the loop's operands spilled 3.8).  Some
// instances keep a little in local memory: of 128 dims by TMA 36 bytes a thread (I8) and
// 40 (F8).
template <int HD, int NQ, int TYPE, bool TMA>
__global__ void __launch_bounds__(32 * kD8Warps, HD == 256 || NQ == 2 ? 2 : TMA ? 4 : 3)
    paged8_decode_kernel(const __grid_constant__ Dec8Args a) {
  using T = Dec8Shape<HD, NQ>;
  constexpr int KS = kD8Step, NT = KS / 8, NG = KS / 16;          // keys a step; tiles of 8, groups of 16
  extern __shared__ __align__(1024) uint8_t sm[];
  const PagedProblem& p = a.p;
  const Pool8& c = a.c;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + T::kRing + T::kQ + T::kScales) + warp * 3;   // a tile of the warp's ring
  if (lane == 0) {
    for (int i = 0; i < 3; ++i) mbar_init(bars + i, 1);
    mbar_fence_init();
    if constexpr (TMA) asm volatile("prefetch.tensormap [%0];\n\tprefetch.tensormap [%1];" ::"l"(&a.mk), "l"(&a.mv) : "memory");
  }
  __syncwarp();
  pdl_wait();
  pdl_trigger();
  if ((smem_u32(sm) & 1023) != 0) {                               // the swizzle needs it; the launch gives it
    if (tid == 0) atomicCAS(p.err, 0, 61);
    return;
  }
  const int kinds = p.n_kv * a.rtiles;                            // of work that has the same keys
  __shared__ float2 sml[kD8Warps][8 * NQ];
  auto keys_of = [&](int s) {
    return (int)max(0ll, min((long long)min(p.kv_len[s], p.max_kv), (long long)c.table_stride * c.page_size));
  };
  __shared__ Walk8 walk;
  if (a.even && !begin_walk(walk, p.n_seqs, kinds, keys_of)) return;
  uint32_t phases = 0;                                            // of the three barriers
#pragma unroll 1
  do {
    int seq, kvh, r0, k0 = 0, k1, split, walk_at = 0, walk_first = 0;
    int part;                                                       // whether this is a part of the rows' keys
    if (a.even) {
      const Piece8Work x = next_piece(walk, p.n_seqs, kinds, keys_of);
      seq = x.seq;
      if (seq < 0) return;
      kvh = x.kind % p.n_kv;
      r0 = x.kind / p.n_kv * 8 * NQ;
      k0 = x.k0;
      k1 = x.k1;
      split = x.index;
      part = x.count > 1;
      if (split == 0 && tid < min(8 * NQ, p.group - r0)) a.counts[seq * p.heads + kvh * p.group + r0 + tid] = x.count;
      walk_at = x.at;
      walk_first = x.first;
    } else if (a.pieces) {
      __shared__ Share8 mine;
      share_out(mine, p.n_seqs, kinds, a.pieces, keys_of);
      seq = mine.seq;
      if (seq < 0) return;
      kvh = mine.kind % p.n_kv;
      r0 = mine.kind / p.n_kv * 8 * NQ;
      split = mine.index;
      part = mine.count > 1;
      k1 = mine.keys;
      if (part) {
        const int len = ((k1 + mine.count - 1) / mine.count + 31) & ~31;
        k0 = min(k1, split * len);
        k1 = min(k1, k0 + len);
      }
      if (split == 0 && tid < min(8 * NQ, p.group - r0)) a.counts[seq * p.heads + kvh * p.group + r0 + tid] = mine.count;
    } else {
      int b = blockIdx.x;
      kvh = b % p.n_kv;
      b /= p.n_kv;
      seq = b % p.n_seqs;
      b /= p.n_seqs;
      const int splits = p.splits ? p.splits : 1;
      split = b % splits;
      r0 = b / splits * 8 * NQ;
      k1 = keys_of(seq);
      part = p.splits;
      if (part) {
        k0 = split * p.chunk;
        k1 = min(k1, k0 + p.chunk);
        if (k0 >= k1) return;                                       // the joining kernel does not look there
      }
    }
    const int nr = min(8 * NQ, p.group - r0);                       // query heads of this tile
    const int* table = c.table + (long long)seq * c.table_stride;
    const uint32_t ring = smem_u32(sm) + warp * 3 * T::kTile;
    const uint32_t ring_s = smem_u32(sm) + T::kRing + T::kQ + warp * 3 * (KS * 4);
    // By TMA, a box a group of 16 keys (zeros where its page is none): lanes 0-15
    // have the page of a step's first group, 16-31 of its second.  Else by
    // cp.async, and lane i has the page of key i.  The entry is not looked at until
    // the step's copies are issued, so that its load is not waited for a step ahead.
    constexpr int SKIP = kD8Warps * KS;                             // from a warp's step to its next
    auto fetch_page = [&](int first) {                              // of the step of keys first ..
      const int key = first + (TMA ? lane & 16 : lane);
      return key < k1 ? table[page_index(c, key)] : -1;
    };
    // where the step lies whose K was asked for last: this lane's key's row and scale
    long long at = -1, at_s = 0;
    int the_page = -1;
    bool there = false;
    auto copy = [&](int first, int slot, const uint8_t* pool, const CUtensorMap* map, const float* scales) {
      if (first < k1) {
        cp_async4(ring_s + slot * (KS * 4) + lane * 4, scales + at_s, there);
        const uint32_t dst = ring + slot * T::kTile;
        if constexpr (TMA) {
          if (lane == 0) mbar_arrive_expect_tx(bars + slot, T::kTile);
          __syncwarp();
          if ((lane & 15) == 0) {
            const int key = first + lane, in_page = c.pshift >= 0 ? key & (c.page_size - 1) : key % c.page_size;
            const uint32_t to = dst + (lane >> 4) * (16 * (HD == 64 ? 64 : 128));
            tma_rows(to, map, 0, kvh, in_page, the_page, bars + slot);
            if constexpr (HD == 256) tma_rows(to + KS * 128, map, 128, kvh, in_page, the_page, bars + slot);
          }
        } else {
          constexpr int CH = HD / 16;                               // 16-byte pieces of a row
#pragma unroll
          for (int i = 0; i < KS * CH / 32; ++i) {
            const int idx = i * 32 + lane, key = idx / CH, pc = idx % CH;
            const long long o = __shfl_sync(0xffffffffu, at, key);
            const bool have = o >= 0 && pc < c.hd / 16;
            cp_async16(dst + piece_off<HD>(key, pc), have ? pool + o + pc * 16 : pool, have);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto ask_k = [&](int first, int page, int slot) {
      if (first < k1) {
        const int key = first + lane;
        const Row8 row = row8(c, key, page);
        there = row.at >= 0 && key < k1;
        at_s = there ? row.scale + kvh : 0;
        the_page = page;
        if constexpr (!TMA) at = there ? row.at + (long long)kvh * c.hd : -1;
      }
      copy(first, slot, c.k, &a.mk, c.ks);
    };
    auto ask_v = [&](int first, int slot) { copy(first, slot, c.v, &a.mv, c.vs); };
    auto arrived = [&](int slot) {
      asm volatile("cp.async.wait_group 2;" ::: "memory");          // all but the two tiles asked for last
      __syncwarp();                                                 // what the other lanes' copies brought is read too
      if constexpr (TMA) {
        const bool ok = mbar_wait(bars + slot, phases >> slot & 1, p.err, 62);
        phases ^= 1u << slot;
        return __all_sync(0xffffffffu, ok) != 0;
      }
      return true;
    };
    // this lane's share of its query's row, asked for ahead of the keys
    float x[NQ][HD / 16][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = n * 8 + g;
      const bool live = r < nr;
      const long long qo = (long long)seq * p.q_stride + (long long)(kvh * p.group + r0 + (live ? r : 0)) * c.hd;
#pragma unroll
      for (int s = 0; s < HD / 16; ++s) {
        const int d = 16 * k_piece<HD>(t4, s >> 2) + 4 * (s & 3);   // hd is a multiple of 16
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live && d < c.hd) {
          if (!a.q_vec)
            f = make_float4(load_elem(p.q, p.type, qo + d), load_elem(p.q, p.type, qo + d + 1), load_elem(p.q, p.type, qo + d + 2),
                            load_elem(p.q, p.type, qo + d + 3));
          else if (p.type == TOSK_F32) f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.q) + qo + d);
          else {
            const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const __half*>(p.q) + qo + d);
            const float2 y = __half22float2(as_h2(u.x)), z = __half22float2(as_h2(u.y));
            f = make_float4(y.x, y.y, z.x, z.y);
          }
        }
        x[n][s][0] = f.x; x[n][s][1] = f.y; x[n][s][2] = f.z; x[n][s][3] = f.w;
      }
    }
    int slot_k = 0, slot_v = 1, slot_n = 2;
    const int begin = k0 + warp * KS;
    int npage = fetch_page(begin);
    const int page1 = fetch_page(begin + SKIP);
    ask_k(begin, npage, slot_k);
    ask_v(begin, slot_v);
    npage = fetch_page(begin + 2 * SKIP);
    ask_k(begin + SKIP, page1, slot_n);

    // The queries while the keys fly: warp w makes the fragments of products w, w + 4 ..;
    // their scales, powers of two, are each lane's own row's.
    uint4* sq = reinterpret_cast<uint4*>(sm + T::kRing);            // [query tile][product][lane]
    float sc[NQ], m[NQ], l[NQ];
    float2 o[NQ][HD / 8];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx = 0.0f;
#pragma unroll
      for (int s = 0; s < HD / 16; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) mx = fmaxf(mx, fabsf(x[n][s][e]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float s2 = pow2_to_2p13(mx);                            // exact scaling of the row
      const float sg = p.scale_log2 < 0.0f ? -s2 : s2;
      sc[n] = fabsf(p.scale_log2) * pow2_inverse(s2);
      if constexpr (TYPE == TOSK_I8) {
        // whole numbers of 2^30 at most, in four signed bytes: rows g and g + 8 of two tiles
        bool odd = false;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
#pragma unroll
          for (int e = 0; e < 4; ++e) odd |= not_finite(x[n][s][e]);
        const uint32_t bad = __ballot_sync(0xffffffffu, odd);
        if (bad >> (lane & 28) & 15) sc[n] = __uint_as_float(0x7fffffffu);
        else sc[n] *= 1.0f / 65536.0f;                              // their bytes count from 2^-16 of the row's scale on
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
          if ((s >> 1 & (kD8Warps - 1)) == warp) {
            // a number plus 128 in every byte has its signed digits, each plus 128, as bytes
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = ((uint32_t)__float2int_rn(x[n][s][e] * sg * 65536.0f) + 0x80808080u) ^ 0x80808080u;
            const uint32_t a0 = prmt(v[0], v[1], 0x5140u), a1 = prmt(v[0], v[1], 0x7362u);
            const uint32_t b0 = prmt(v[2], v[3], 0x5140u), b1 = prmt(v[2], v[3], 0x7362u);
            const uint32_t limb[4] = {prmt(a0, b0, 0x5410u), prmt(a0, b0, 0x7632u), prmt(a1, b1, 0x5410u), prmt(a1, b1, 0x7632u)};
            // product s / 2 of a tile: words of rows g and g + 8 at its first 4 k's, then at its next
            uint2* to = reinterpret_cast<uint2*>(sq + (n * (HD / 16) + (s & ~1)) * 32 + lane) + (s & 1);
            to[0] = make_uint2(limb[3], limb[2]);
            to[64] = make_uint2(limb[1], limb[0]);
          }
      } else {
#pragma unroll
        for (int s = 0; s < HD / 16; ++s)
          if ((s & (kD8Warps - 1)) == warp) {
            uint4 u;
            split_pair(x[n][s][0] * sg, x[n][s][1] * sg, u.x, u.y);
            split_pair(x[n][s][2] * sg, x[n][s][3] * sg, u.z, u.w);
            sq[(n * (HD / 16) + s) * 32 + lane] = u;
          }
      }
      m[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) o[n][d] = make_float2(0.0f, 0.0f);
    }
    __syncthreads();
    if (a.even && tid == 0) {                                       // all have read the walk's last state
      walk.at = walk_at;
      walk.first = walk_first;
      walk.seq = seq;
    }
    const uint32_t sqa = smem_u32(sq) + lane * 16;

    bool dead = false;
    for (int first = begin; first < k1; first += SKIP) {
      if (!arrived(slot_k)) {
        dead = true;                                                // a wait ran out
        break;
      }
      const uint32_t kt = ring + slot_k * T::kTile, vt = ring + slot_v * T::kTile;
      const uint32_t ks = ring_s + slot_k * (KS * 4) + 8 * t4, vs = ring_s + slot_v * (KS * 4) + 8 * t4;
      float s[NQ][NT][2];                                           // scores of keys 8 x + 2t, 2t + 1
      if constexpr (TYPE == TOSK_I8) {
        // two tiles of keys at a time, for the registers
#pragma unroll
        for (int x0 = 0; x0 < NT; x0 += 2) {
          int c0[NQ][2][4], c1[NQ][2][4];
#pragma unroll
          for (int i = 0; i < HD / 64; ++i) {
            uint32_t w[2][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) lds<4>(kt + piece_off<HD>(8 * (x0 + x) + g, k_piece<HD>(t4, i)), w[x]);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                uint32_t qa[4], qb[4];
                lds<4>(sqa + (n * (HD / 16) + 4 * i + 2 * j) * 512, qa);
                lds<4>(sqa + (n * (HD / 16) + 4 * i + 2 * j + 1) * 512, qb);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                  mma_i(c0[n][x], qa, w[x][2 * j], w[x][2 * j + 1], i == 0 && j == 0);
                  mma_i(c1[n][x], qb, w[x][2 * j], w[x][2 * j + 1], i == 0 && j == 0);
                }
              }
          }
          // sums of bytes stay below 2^21 (256 dims: 2^22): two fit one int
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                s[n][x0 + x][e] =
                    fmaf((float)(c0[n][x][e] * 256 + c0[n][x][2 + e]), 65536.0f, (float)(c1[n][x][e] * 256 + c1[n][x][2 + e]));
        }
      } else {
        float c0[NQ][NT][4];
#pragma unroll
        for (int i = 0; i < HD / 64; ++i) {
          uint32_t w[NT][4];
#pragma unroll
          for (int x = 0; x < NT; ++x) lds<4>(kt + piece_off<HD>(8 * x + g, k_piece<HD>(t4, i)), w[x]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t qa[NQ][4];
#pragma unroll
            for (int n = 0; n < NQ; ++n) lds<4>(sqa + (n * (HD / 16) + 4 * i + j) * 512, qa[n]);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
              uint32_t b0, b1;
              cvt_word<TYPE>(w[x][j], b0, b1);
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                if (i == 0 && j == 0) mma_h_zero(c0[n][x], qa[n], b0, b1);
                else mma_h(c0[n][x], qa[n], b0, b1);
              }
            }
          }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int x = 0; x < NT; ++x)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[n][x][e] = c0[n][x][e] + c0[n][x][2 + e];
      }
      uint32_t pa[NQ][NG][4];
      const int left = k1 - first - 2 * t4;
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float w[2 * NT];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          uint32_t k2[2];
          lds<2>(ks + 32 * x, k2);
          w[2 * x] = s[n][x][0] * (__uint_as_float(k2[0]) * sc[n]);
          w[2 * x + 1] = s[n][x][1] * (__uint_as_float(k2[1]) * sc[n]);
        }
        if (left + 2 * t4 < KS) {                                   // the sequence's last step
#pragma unroll
          for (int e = 0; e < 2 * NT; ++e)
            if ((e >> 1) * 8 + (e & 1) >= left) w[e] = -INFINITY;
        }
        float top = fmaxf(w[0], w[1]);
#pragma unroll
        for (int e = 2; e < 2 * NT; e += 2) top = fmaxf(top, fmaxf(w[e], w[e + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m[n] + 8.0f)) {
          const float mn = top > m[n] + 8.0f ? top : m[n];
          const float f = mn == m[n] ? 1.0f : exp2f(m[n] - mn);     // 0 on the first keys
          m[n] = mn;
          l[n] *= f;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) o[n][d] = __fmul2_rn(o[n][d], make_float2(f, f));
        }
        const float bias = 7.0f - (m[n] == -INFINITY ? 0.0f : m[n]);
#pragma unroll
        for (int e = 0; e < 2 * NT; ++e) w[e] = ex2(w[e] + bias);
#pragma unroll
        for (int h = 0; h < NG; ++h) {
          l[n] += (w[4 * h] + w[4 * h + 1]) + (w[4 * h + 2] + w[4 * h + 3]);
          split_pair(w[4 * h], w[4 * h + 1], pa[n][h][0], pa[n][h][1]);
          split_pair(w[4 * h + 2], w[4 * h + 3], pa[n][h][2], pa[n][h][3]);
        }
      }
      __syncwarp();                                                 // K is read: its place takes the next V
      ask_v(first + SKIP, slot_k);
      if (!arrived(slot_v)) {
        dead = true;
        break;
      }
      __half2 mul[NG][2];
      float big = 0.0f;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        uint32_t v2[2];
        lds<2>(vs + 32 * x, v2);
        const float va = __uint_as_float(v2[0]), vb = __uint_as_float(v2[1]);
        mul[x >> 1][x & 1] = __floats2half2_rn(va, vb);
        big = fmaxf(big, fmaxf(va, vb));
      }
      constexpr int VP = HD == 256 ? 2 : 1, VH = HD == 64 ? 1 : 2;  // pieces a key, their halves
      const __half2 off = __float2half2_rn(-1152.0f);
      auto add_values = [&](auto large) {
#pragma unroll
        for (int x = 0; x < VP * VH; ++x) {
          uint32_t w[NG][4][2];
#pragma unroll
          for (int h = 0; h < NG; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = 16 * h + (e >> 1) * 8 + 2 * t4 + (e & 1);
              lds<2>(vt + (HD == 64 ? piece_off<HD>(key, g >> 1) + (g & 1) * 8
                                    : piece_off<HD>(key, g + 8 * (x >> 1)) + ((g >> 1 ^ x) & 1) * 8),
                     w[h][e]);
              // what lies behind the sequence may be e4m3's NaN, which a weight of 0 does not silence
              if (TYPE == TOSK_F8 && left + 2 * t4 < KS && key - 2 * t4 >= left) w[h][e][0] = w[h][e][1] = 0;
            }
#pragma unroll
          for (int j = 0; j < 4; ++j) {                             // two dims of every piece
            uint32_t b0[NG][2], b1[NG][2];
#pragma unroll
            for (int h = 0; h < NG; ++h) {
              constexpr bool L = decltype(large)::value;
              pair_keys<TYPE, L>(w[h][0][j >> 1], w[h][1][j >> 1], j & 1, mul[h][0], L ? off : __hmul2(off, mul[h][0]), b0[h]);
              pair_keys<TYPE, L>(w[h][2][j >> 1], w[h][3][j >> 1], j & 1, mul[h][1], L ? off : __hmul2(off, mul[h][1]), b1[h]);
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              float y[2][4];                                        // two products, then the fp32 sums
#pragma unroll
              for (int d = 0; d < 2; ++d) mma_h_zero(y[d], pa[n][0], b0[0][d], b1[0][d]);
#pragma unroll
              for (int d = 0; d < 2; ++d) mma_h(y[d], pa[n][1], b0[1][d], b1[1][d]);
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                float2& to = o[n][x * 8 + 2 * j + d];
                to = __fadd2_rn(to, __fadd2_rn(make_float2(y[d][0], y[d][1]), make_float2(y[d][2], y[d][3])));
              }
            }
          }
        }
      };
      // I8: -1152 times a scale beyond 2^5 is no fp16 number
      if (TYPE == TOSK_I8 && __any_sync(0xffffffffu, big > 32.0f)) add_values(std::true_type{});
      else add_values(std::false_type{});
      __syncwarp();                                                 // V is read: its place takes the K after the next
      ask_k(first + 2 * SKIP, npage, slot_v);
      npage = fetch_page(first + 3 * SKIP);
      const uint32_t s_ = slot_k;
      slot_k = slot_n;
      slot_n = slot_v;
      slot_v = s_;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                                // the rings are free: join the warps there
    // [warp][8 NQ queries][HD]; what a warp writes at once lies in different banks
    float* so = reinterpret_cast<float*>(sm);
    constexpr int SR = HD + HD / 4 + 1;
    auto place = [](int d) { return d + (d >> 5) * 8; };
    static_assert(T::kRing >= kD8Warps * 8 * NQ * SR * 4, "the sums of the warps");
    constexpr int DG = HD == 64 ? 8 : 16;                           // dims of a column
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
      if (t4 == 0) sml[warp][n * 8 + g] = make_float2(m[n] - 7.0f, l[n]);
      float* to = so + ((warp * NQ + n) * 8 + g) * SR;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        // of pieces 2, 3, 6, 7 the halves changed places
        const int at_d = (d / DG) * 128 + (HD == 64 ? d % DG : (d % DG) ^ (8 * (t4 & 1)));
        to[place(at_d + 2 * t4 * DG)] = o[n][d].x;                  // columns 2t and 2t + 1
        to[place(at_d + (2 * t4 + 1) * DG)] = o[n][d].y;
      }
    }
    dead = __syncthreads_or(dead);
    // a warp a query
    for (int r = warp; r < nr; r += kD8Warps) {
      float M = -INFINITY, L = 0.0f, f[kD8Warps];
#pragma unroll
      for (int w = 0; w < kD8Warps; ++w) M = fmaxf(M, sml[w][r].x);
#pragma unroll
      for (int w = 0; w < kD8Warps; ++w) {
        f[w] = M == -INFINITY ? 0.0f : exp2f(sml[w][r].x - M);
        L += f[w] * sml[w][r].y;
      }
      const int head = kvh * p.group + r0 + r;
      const long long row = (long long)seq * p.heads + head, to = (long long)split * p.total_q * p.heads + row;
      const float inv = L == 0.0f ? 0.0f : 1.0f / L;
      if (part && lane == 0) p.part_ml[to] = make_float2(M, L);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int d = lane + 32 * i;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kD8Warps; ++w) v = fmaf(f[w], so[(w * NQ * 8 + r) * SR + place(d)], v);
        if (d >= c.hd) continue;
        if (part) p.part_o[to * c.hd + d] = v;
        else store_elem(p.out, p.type, (long long)seq * p.out_stride + (long long)head * c.hd + d, L == 0.0f ? 0.0f : v * inv);
      }
    }
    if (!a.even || dead) return;
    // the sums lay where the next piece's copies go
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  } while (true);
}

}  // namespace tos

using namespace tos;

namespace {

int dec8_launch(const void* f, int smem, const Dec8Args& a, unsigned grid, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(32 * kD8Warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<Dec8Args*>(&a)};
  return (int)cudaLaunchKernelExC(&cfg, f, args);
}

// Boxes of 16 rows x 128 bytes (64 dims or fewer: 64) of one head.
bool dec8_map(CUtensorMap* m, const void* base, const tosk_paged8_t* kv) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  const bool narrow = kv->hd <= 64;
  const cuuint64_t dim[4] = {(cuuint64_t)kv->hd, (cuuint64_t)kv->n_kv, (cuuint64_t)kv->page_size, (cuuint64_t)kv->n_pages};
  const cuuint64_t row = (cuuint64_t)kv->n_kv * kv->hd;
  const cuuint64_t str[3] = {(cuuint64_t)kv->hd, row, row * kv->page_size};
  const cuuint32_t box[4] = {narrow ? 64u : 128u, 1, 16, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dim, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int TYPE>
int dec8(const Dec8Args& a, int nq, bool tma, unsigned n, cudaStream_t st) {
  if constexpr (HD <= 128)
    if (nq == 2) return dec8_launch((const void*)paged8_decode_kernel<HD, 2, TYPE, true>, Dec8Shape<HD, 2>::kSmem, a, n, st);
  const void* f = tma ? (const void*)paged8_decode_kernel<HD, 1, TYPE, true> : (const void*)paged8_decode_kernel<HD, 1, TYPE, false>;
  return dec8_launch(f, Dec8Shape<HD, 1>::kSmem, a, n, st);
}

// How the keys are cut.  Where a CTA for every 512 keys is more than the SMs
// hold at once: by the sequences' lengths, among as many CTAs as they do hold.
// Else, and where there are too many sequences or blocks for that: chunks of one
// length.
struct Plan8 {
  int ctas;                       // that share the keys; 0: chunks
  int pieces;                     // for each kind, see share_out; 0: even shares
  int splits, chunk;              // splits 0: none
  int slots;                      // most partial rows of a row
};
Plan8 plan8(int n_seqs, int max_kv, int heads, int n_kv, int hd) {
  const int group = heads / n_kv, tile = group > 8 && hd <= 128 ? 16 : 8, ctas = 148 * (hd <= 128 && group <= 8 ? 4 : 2);
  const long long kinds = (long long)n_kv * ((group + tile - 1) / tile), chunks = ((long long)max_kv + 511) / 512;
  const long long blocks = ((long long)max_kv + 127) / 128 + kPieceCost;
  if (chunks <= 1) return {0, 0, 0, max_kv, 0};
  // (by cp.async a group of more than 8 heads has twice the kinds)
  if (kinds * n_seqs * chunks > ctas && n_seqs <= kShareSeqs && 2 * kinds * n_seqs * blocks < (1ll << 31) - ctas) {
    // an even share is at least blocks x kinds / ctas
    const long long b = ctas / kinds, most = b + 2;
    const int slots = (int)(most < blocks ? most : blocks);
    if (b >= 4 * n_seqs) return {ctas, (int)b, 0, max_kv, slots};
    return {ctas, 0, 0, max_kv, slots};
  }
  const long long want = (ctas + kinds * n_seqs - 1) / (kinds * n_seqs), n = want < chunks ? want : chunks;
  if (n <= 1) return {0, 0, 0, max_kv, 0};
  const int chunk = (int)((max_kv + n - 1) / n + 127) / 128 * 128, s = (max_kv + chunk - 1) / chunk;
  return {0, 0, s > 1 ? s : 0, chunk, s > 1 ? s : 0};
}

// Rows that are no whole 16-byte pieces go the way over fp16 (below).
bool direct(int hd) { return hd % 16 == 0; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// A call over the cache's fp16 copy, which lies in front of its workspace.  The
// copy's pages have room for more keys than the cache's table row may hold: keys end
// there, while kv_len still says where the rows are.
int over_copy(tosk_paged_attn_t& x, const tosk_paged8_t* kv, long long total_kv, cudaStream_t st) {
  const size_t wide = tosk_paged8_wide_bytes(x.n_seqs, total_kv, x.max_kv, kv->n_kv, kv->hd);
  const int e = tosk_paged8_wide(kv, x.kv_len, x.n_seqs, total_kv, x.max_kv, x.ws, &x.kv, st);
  const long long room = (long long)kv->table_stride * kv->page_size;
  x.room = (int)(room < x.max_kv ? room : x.max_kv);
  x.ws = reinterpret_cast<uint8_t*>(x.ws) + wide;
  x.ws_bytes -= wide;
  return e;
}

}  // namespace

extern "C" size_t tosk_paged8_decode_ws_bytes(int n_seqs, int max_kv, int n_heads, int n_kv, int hd) {
  if (direct(hd)) {
    const Plan8 d = plan8(n_seqs, max_kv, n_heads, n_kv, hd);
    return up256(paged_slots_bytes(d.slots, n_seqs, n_heads, hd)) + (d.ctas ? (size_t)n_seqs * n_heads * 4 : 0);
  }
  return tosk_paged8_wide_bytes(n_seqs, (long long)n_seqs * max_kv, max_kv, n_kv, hd) +
         up256(tosk_paged_decode_ws_bytes(n_seqs, max_kv, 0, n_heads, n_kv, hd));
}

extern "C" int tosk_paged8_decode(const tosk_paged_attn_t* t, const tosk_paged8_t* kv, cudaStream_t st) {
  tosk_paged_attn_t x = *t;
  if (!direct(kv->hd)) {
    const int e = over_copy(x, kv, (long long)x.n_seqs * x.max_kv, st);
    return e ? e : tosk_paged_decode(&x, st);
  }
  Dec8Args a;
  a.c = pool8_of(*kv);
  memset(&x.kv, 0, sizeof(x.kv));
  x.kv.n_kv = kv->n_kv;
  x.kv.hd = kv->hd;
  x.kv.page_size = kv->page_size;
  x.kv.table = kv->table;
  x.kv.table_stride = kv->table_stride;
  a.p = paged_problem(&x);
  const Plan8 d = plan8(x.n_seqs, x.max_kv, x.n_heads, kv->n_kv, kv->hd);
  a.p.splits = d.splits;
  a.p.chunk = d.chunk;
  paged_part_views(a.p, x.ws, d.slots);
  uint8_t* behind = reinterpret_cast<uint8_t*>(x.ws) + up256(paged_slots_bytes(d.slots, x.n_seqs, x.n_heads, kv->hd));
  a.counts = d.ctas ? reinterpret_cast<int*>(behind) : nullptr;
  // Pages of whole groups of 16 keys: by TMA.  Its maps take the host 0.6 us, more than
  // TMA saves where there is little to read (1 sequence of 272 keys: 7.9 us, 8.6).
  const bool much = a.p.group > 8 || d.ctas > 0 || (long long)x.n_seqs * x.max_kv * kv->n_kv * kv->hd > (4 << 20);
  const bool tma = kv->page_size % 16 == 0 && much && dec8_map(&a.mk, kv->k, kv) && dec8_map(&a.mv, kv->v, kv);
  const int nq = a.p.group > 8 && kv->hd <= 128 && tma ? 2 : 1;
  a.rtiles = (a.p.group + 8 * nq - 1) / (8 * nq);
  a.q_vec = ((uintptr_t)x.q & (x.type == TOSK_F32 ? 15 : 7)) == 0 && x.q_stride % 4 == 0;
  const long long kinds = (long long)a.rtiles * kv->n_kv;
  a.even = d.ctas > 0 && !d.pieces;
  a.pieces = d.pieces;
  const int even = !tma && d.ctas > 148 * 3 ? 148 * 3 : d.ctas;   // by cp.async three CTAs an SM
  const long long grid = a.pieces ? kinds * a.pieces : a.even ? even : kinds * (d.splits ? d.splits : 1) * x.n_seqs;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  const unsigned n = (unsigned)grid;
  const bool i8 = kv->type == TOSK_I8;
  const int e = kv->hd <= 64    ? i8 ? dec8<64, TOSK_I8>(a, nq, tma, n, st) : dec8<64, TOSK_F8>(a, nq, tma, n, st)
                : kv->hd <= 128 ? i8 ? dec8<128, TOSK_I8>(a, nq, tma, n, st) : dec8<128, TOSK_F8>(a, nq, tma, n, st)
                                : i8 ? dec8<256, TOSK_I8>(a, nq, tma, n, st) : dec8<256, TOSK_F8>(a, nq, tma, n, st);
  return e || !d.slots ? e : paged_join(a.p, a.counts, st);
}

extern "C" size_t tosk_paged8_prompt_ws_bytes(int n_seqs, int total_q, long long total_kv, int max_kv, int n_heads, int n_kv, int hd) {
  return tosk_paged8_wide_bytes(n_seqs, total_kv, max_kv, n_kv, hd) +
         up256(tosk_paged_prompt_ws_bytes(n_seqs, total_q, max_kv, n_heads, n_kv, hd));
}

extern "C" int tosk_paged8_prompt(const tosk_paged_attn_t* t, const tosk_paged8_t* kv, long long total_kv, cudaStream_t st) {
  tosk_paged_attn_t x = *t;
  const int e = over_copy(x, kv, total_kv, st);
  return e ? e : tosk_paged_prompt(&x, st);
}
