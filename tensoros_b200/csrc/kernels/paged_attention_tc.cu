// paged_attention_tc.cu - attention of many query rows over an fp16 paged
// cache on the tensor cores (tcgen05): prompts, and a decode batch over its
// shared prefix.
//
//   S = Q K^T,  P = 2^(c S - m),  O += P V,  l += sum P     (128 x 128 tiles)
//
// Persistent CTAs, one an SM, take pieces of work in turn: 256 packed rows
// (token, query head of the group) of one sequence and one key/value head, as
// two row tiles of 128, over the keys in tiles of 128.  Twenty warps:
//   * one plans: which piece is this CTA's next (longest first, dealt there
//     and back), two ahead;
//   * one brings K and V tiles, page by page, into a ring of shared memory
//     slots (TMA boxes of a page's rows x 64 columns, swizzled 128 B; lane i
//     takes page i of the tile), into the next piece where the ring has room;
//   * one thread issues the MMAs in the order PV0(j) S0(j+1) PV1(j) S1(j+1),
//     so the tensor cores work on one row tile while the other's softmax runs;
//     accumulators in tensor memory: S0, S1 (128 columns each), O0, O1;
//   * sixteen, eight a row tile, hold a row and half of a tile's keys a thread:
//     weights under the maximum so far and the new maximum from one pass over
//     S, a vote of the row's two threads, P over S's columns as the A operand
//     of P V; at the end of a piece the output rows through shared memory.
// The maximum in use follows the true one only when that has grown by more
// than 2^8 (O is then scaled in tensor memory), so O is touched rarely.
// P carries a factor 2^7, at most 2^15, which keeps small weights out of
// fp16's subnormals; it cancels in O / l.
//
// What bounds it (B200; a piece a SM, 1024 to 8192 keys): a key tile of both
// row tiles takes 2.0 us for fp16 rows, where a library product's rate would
// take 1.5, and 4.0 for fp32 rows, whose two-part products are twice the work;
// a call costs 21 to 25 us beside its tiles.  The row tiles
// alternate between softmax and MMAs, two of them do not fill the tensor
// cores, and a third does not fit tensor memory.  Packed fp16 prompts of 6537
// tokens, 32 / 8 heads x 128: 190 us, 846 TFLOP/s.
// Steps on the way (the same prompts, us, each when it was made): one warpgroup a row tile 287; queries
// loaded in batches, registers moved to the softmax warps, halves of P handed
// on 235; one elected thread for all MMAs 208; four warpgroups 207; persistent
// 197; weights and maximum from one read of S 194; two pairs of eight
// exponentials on the FMA pipe 188 (none 197, four pairs 205).
//
// Precision.  fp16 rows: P is rounded to fp16 (half a step, 2^-11, of each
// weight, which is what the output's own rounding costs; sums and maxima are
// fp32).  fp32 rows: q, scaled by a power of two per row, and P go in as
// fp16 pairs hi + lo (22 bits), two MMAs each: 1.2e-6 against 64 bits (norm)
// over 7512 keys.  The accumulators, which cut off instead of rounding, are
// emptied into memory every few key tiles (fold_tiles).
//
// Keys behind a row's last one are masked in S; value rows behind the key
// range (a page's unused rows may hold anything) and, where only some rows see
// a key, values that are not finite are zeroed in shared memory, so that an
// unseen infinity never reaches a row.  Rows that do see one get it at the end of
// the CTA, when the pipeline is done and none of its bounded waits runs (patch_piece).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include "paged_common.cuh"
#include "paged_tc.cuh"

namespace tos {

constexpr int kTcCtas = 148;           // one a SM, each takes pieces of work in turn
constexpr int kTcThreads = 640;        // four softmax warpgroups; K/V copies, MMAs, plan, an idle warp
constexpr int kTcRegs = 96;            // a thread at launch, moved to the softmax warps afterwards
constexpr int kTcRegsSoftmax = 104, kTcRegsRest = 64;
static_assert(4 * kTcRegsSoftmax + kTcRegsRest <= 5 * kTcRegs, "registers of the launch");
constexpr int kCopyWarp = 16, kMmaWarp = 17, kPlanWarp = 18;
constexpr int kTileBar = 9;            // named barriers: 1..8 pair the two warps of 32 rows, 9 and 10 a row tile's eight,
constexpr int kEndBar = 11;            // 11 all twenty, when the pipeline is done
constexpr int kRows = 128;            // rows of a tile
constexpr int kKeys = 128;            // keys of a tile
constexpr float kBias = 7.0f;         // log2 of the factor that P carries
constexpr int kPoly = 3;              // of eight pairs of exponentials, those at 2 and 5 go to the FMA pipe
// Key tiles whose products one accumulator sums, of a row tile's nt.  It loses
// 1e-7 of itself a step of 16 keys.  fp32 rows: 3 (512 rows behind 7001 keys, us:
// 2: 174, 3: 157, 4: 152, 8: 144, never: 137; error in norm 1.2e-6, an fp32
// program's 1.6e-6), and 2 up to 2048 keys, where an fp32 program errs less (90
// rows behind 400 keys: 8e-7, with 3 1.1e-6, an fp32 program's 5.5e-7).  fp16
// rows: 32, a loss of 2.6e-5, a twentieth of their rounding (131,072 keys in one
// chain: 8e-4; 700 rows behind 20,000 keys, us: 8: 553, 16: 535, 32: 531, 64 and
// never: 520).
__host__ __device__ constexpr int fold_tiles(bool split, int nt) { return !split ? 32 : nt <= 16 ? 2 : 3; }
constexpr float kSlack = 8.0f;        // log2 by which the maximum may grow unfollowed

struct TcArgs {
  CUtensorMap mk, mv;                 // [page][row][kv head][dim]: boxes of box_rows rows x 64 dims
  PagedProblem p;
  int box_rows, q_vec, out_vec;
};

template <int HD, bool SPLIT>
struct TcShape {
  static constexpr int kHalves = HD / 64;
  static constexpr int kTile = kHalves * 16384;                 // bytes of a 128 x HD fp16 tile
  static constexpr int kQ = 2 * (SPLIT ? 2 : 1) * kTile;
  static constexpr int kSlots = HD == 128 ? (SPLIT ? 3 : 5) : 8;
  static constexpr int kBars = 2 * kSlots + 17;
  static constexpr int kStage = kQ >= 16 * 4096 ? 0 : 16 * 4096;     // output rows, where Q's place is too small for them
  static constexpr int kSmem = kQ + kSlots * kTile + kStage + kBars * 8 + 8 + 2 * 64 + 4 * kRows * 4 + 16;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
#define TOS_R8(r, i) \
  "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
// The registers of a tcgen05.ld hold their values only after the wait; tying
// them to it keeps every use behind it.
__device__ __forceinline__ void tc_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TOS_R8(r, 0), TOS_R8(r, 8), TOS_R8(r, 16), TOS_R8(r, 24)::"memory");
}
__device__ __forceinline__ void tc_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TOS_R8(r, 0), TOS_R8(r, 8)::"memory");
}
__device__ __forceinline__ void tc_wait_ld8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : TOS_R8(r, 0)::"memory");
}
#undef TOS_R8
// 2^x of two values on the FMA pipe, which has room beside the 16 exponentials
// a clock of the SFU.  x = n + f, |f| <= 1/2: n by adding 1.5 2^23, 2^f by a
// degree-4 polynomial fitted here for least relative error (2.6e-6, far below
// the weights' fp16 rounding), 2^n into the exponent.  Below 2^-126: 2^-126.
// A NaN gives kNanWeight, the largest float: a NaN's bits, 0x7fffffff, and the
// same shifted by 23 are added.
constexpr float kNanWeight = 3.402823466e38f;
__device__ __forceinline__ float max_nan(float x, float y) {
  float z;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
  return z;
}
__device__ __forceinline__ float2 exp2_fma(float2 x) {
  x.x = max_nan(x.x, -126.0f);
  x.y = max_nan(x.y, -126.0f);
  const float2 big = make_float2(12582912.0f, 12582912.0f), nbig = make_float2(-12582912.0f, -12582912.0f);
  const float2 n = __fadd2_rn(x, big);
  const float2 r = __fadd2_rn(n, nbig);
  const float2 f = __ffma2_rn(r, make_float2(-1.0f, -1.0f), x);
  float2 y = make_float2(0.00957010146f, 0.00957010146f);
  y = __ffma2_rn(y, f, make_float2(0.0559178603f, 0.0559178603f));
  y = __ffma2_rn(y, f, make_float2(0.240247488f, 0.240247488f));
  y = __ffma2_rn(y, f, make_float2(0.693121815f, 0.693121815f));
  y = __ffma2_rn(y, f, make_float2(0.999999261f, 0.999999261f));
  y.x = __uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23));
  y.y = __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23));
  return y;
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tc_ld8(uint32_t addr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr));
}
__device__ __forceinline__ void tc_st4(uint32_t addr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tma_page(void* dst, const CUtensorMap* m, int x, int head, int row, int page,
                                         uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(m), "r"(x), "r"(head), "r"(row), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

struct TileId {
  int seq, rt;                        // seq < 0: no such tile
};
struct PlanCursor {
  int s0, before;                     // sequences passed, and their tiles
};
// Sequences, one a lane, up to which tiles go by length.  One prompt of 2048 to
// 4096 tokens behind 15 to 30 short ones: 68 to 174 us sorted, 84 to 211 in the
// order given; with 120 short ones the search costs what it saves (246, 242),
// and 256 ragged prompts of up to 200 tokens take 268 us sorted, 244 not.
constexpr int kSortSeqs = 32;

__device__ __forceinline__ int row_tiles(const PagedProblem& p, const SeqTask& t) {
  return (t.qn * p.group + 2 * kRows - 1) / (2 * kRows);
}

// The lane whose running sum over the warp of `n` first passes f: its place,
// and f less what comes before it.  false: the warp's sum is subtracted.
__device__ __forceinline__ bool find_lane(int n, int& f, int& at) {
  const int lane = threadIdx.x & 31;
  int sum = n;
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += v;
  }
  const uint32_t hit = __ballot_sync(0xffffffffu, sum > f);
  if (hit) {
    at = __ffs(hit) - 1;
    f -= __shfl_sync(0xffffffffu, sum - n, at);
    return true;
  }
  f -= __shfl_sync(0xffffffffu, sum, 31);
  return false;
}

// The f-th row tile of the call (f grows from call to call of a CTA).
//
// Up to kSortSeqs sequences: in falling order of the tiles' key tiles, so that
// the long ones start first whatever the sequences' order.  In sequence s the
// tiles with at least w key tiles are the last count(w); the w of rank f is
// found by bisection over their sum, the sequence by a prefix sum.  More
// sequences: in their own order, a sequence's long tiles first; the cursor
// passes each once (4096 ragged prompts: 3.5 ms; a search a tile: 77 ms).
//
// Not inlined: the softmax warps' code is slower beside it (194 us for packed
// prompts against 189).
__device__ __noinline__ TileId pick_of_many(const PagedProblem& p, int f, PlanCursor& cur) {
  const int lane = threadIdx.x & 31;
  int at;
  if (p.n_seqs > kSortSeqs) {
    for (; cur.s0 < p.n_seqs; cur.s0 += 32) {
      const int s = cur.s0 + lane, n = s < p.n_seqs ? row_tiles(p, seq_task(p, s)) : 0;
      int g = f - cur.before;
      if (find_lane(n, g, at)) return {cur.s0 + at, __shfl_sync(0xffffffffu, n, at) - 1 - g};
      cur.before = f - g;
    }
    return {-1, 0};
  }
  const SeqTask t = lane < p.n_seqs ? seq_task(p, lane) : SeqTask{0, 0, 0, 0, nullptr};
  const int n = row_tiles(p, t);
  auto count = [&](int w) {
    if (w <= 0) return n;
    if (kKeys * (w - 1) >= t.kvn) return 0;
    const long long tok = (long long)kKeys * (w - 1) - t.off;    // first token that sees key kKeys (w - 1)
    const long long first = tok <= 0 ? 0 : tok * p.group / (2 * kRows);
    return first >= n ? 0 : n - (int)first;
  };
  auto total = [&](int w) { return __reduce_add_sync(0xffffffffu, count(w)); };
  if (f >= total(0)) return {-1, 0};
  int lo = 0, hi = (p.max_kv + kKeys - 1) / kKeys + 1;            // total(lo) > f >= total(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (total(mid) > f) lo = mid;
    else hi = mid;
  }
  const int above = count(lo + 1), c = count(lo) - above;         // this lane's tiles of lo key tiles
  f -= __reduce_add_sync(0xffffffffu, above);
  if (!find_lane(c, f, at)) return {-1, 0};
  return {at, __shfl_sync(0xffffffffu, n - above - c, at) + f};
}
__device__ __forceinline__ TileId pick_tile(const PagedProblem& p, int f, PlanCursor& cur) {
  if (p.n_seqs == 1) {
    const int n = row_tiles(p, seq_task(p, 0));
    return f < n ? TileId{0, n - 1 - f} : TileId{-1, 0};
  }
  return pick_of_many(p, f, cur);
}

// The k-th piece of this CTA: they go round the CTAs there and back.
__device__ __forceinline__ int piece_of(int k) {
  return k * (int)gridDim.x + (k & 1 ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
}

// Scores from the n-th on count for nothing.
template <int N>
__device__ __forceinline__ void mask_from(uint32_t (&s)[N], int n) {
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e >= n) s[e] = 0xff800000u;                                     // -inf
}
template <bool NANS, int N>
__device__ __forceinline__ float max_of(const uint32_t (&s)[N]) {
  auto top = [](float x, float y) { return NANS ? max_nan(x, y) : fmaxf(x, y); };
  float a = top(__uint_as_float(s[0]), __uint_as_float(s[1])), b = top(__uint_as_float(s[2]), __uint_as_float(s[3]));
#pragma unroll
  for (int e = 4; e < N; e += 4) {
    a = top(top(a, __uint_as_float(s[e])), __uint_as_float(s[e + 1]));
    b = top(top(b, __uint_as_float(s[e + 2])), __uint_as_float(s[e + 3]));
  }
  return top(a, b);
}
// Multiplies n columns of this warp's 32 rows in tensor memory.  Rarely
// called: out of line, so that its registers cost the loop around it none.
static __device__ __noinline__ void scale_cols(uint32_t addr, int n, float f) {
#pragma unroll 1
  for (int c = 0; c < n; c += 16) {
    uint32_t o[16];
    tc_ld16(addr + c, o);
    tc_wait_ld16(o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
    tmem_st16(addr + c, o);
  }
}
// The CTA's sums of chains that have ended: four columns of a warp's 32 rows
// lie side by side, `n` columns a warp.
__device__ __forceinline__ float* fold_at(const PagedProblem& p, int n) {
  return p.fold + (size_t)(blockIdx.x * kCopyWarp + (threadIdx.x >> 5)) * (32 * n) + (threadIdx.x & 31) * 4;
}
// Adds n columns of this warp's 32 rows in tensor memory to them (first: puts).
static __device__ __noinline__ void fold_cols(const PagedProblem& p, uint32_t addr, int n, bool first) {
  float* dst = fold_at(p, n);
#pragma unroll 1
  for (int c = 0; c < n; c += 16, dst += 512) {
    uint32_t o[16];
    tc_ld16(addr + c, o);
    float4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      x[e] = first ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(dst + 128 * e);
    tc_wait_ld16(o);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      *reinterpret_cast<float4*>(dst + 128 * e) =
          make_float4(x[e].x + __uint_as_float(o[4 * e]), x[e].y + __uint_as_float(o[4 * e + 1]),
                      x[e].z + __uint_as_float(o[4 * e + 2]), x[e].w + __uint_as_float(o[4 * e + 3]));
  }
}
// And them to the columns, at the end.
static __device__ __noinline__ void fold_back(const PagedProblem& p, uint32_t addr, int n) {
  const float* src = fold_at(p, n);
#pragma unroll 1
  for (int c = 0; c < n; c += 16, src += 512) {
    uint32_t o[16];
    tc_ld16(addr + c, o);
    float4 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = *reinterpret_cast<const float4*>(src + 128 * e);
    tc_wait_ld16(o);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[4 * e] = __float_as_uint(x[e].x + __uint_as_float(o[4 * e]));
      o[4 * e + 1] = __float_as_uint(x[e].y + __uint_as_float(o[4 * e + 1]));
      o[4 * e + 2] = __float_as_uint(x[e].z + __uint_as_float(o[4 * e + 2]));
      o[4 * e + 3] = __float_as_uint(x[e].w + __uint_as_float(o[4 * e + 3]));
    }
    tmem_st16(addr + c, o);
  }
  tmem_st_wait();
}
static __device__ __noinline__ void fold_scale(const PagedProblem& p, int n, float f) {
  float* dst = fold_at(p, n);
#pragma unroll 1
  for (int c = 0; c < n; c += 4, dst += 128) {
    float4* at = reinterpret_cast<float4*>(dst);
    *at = make_float4(at->x * f, at->y * f, at->z * f, at->w * f);
  }
}
// The two warps that share 32 rows.
__device__ __forceinline__ void pair_sync(int bar) { asm volatile("bar.sync %0, 64;" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool pair_any(int bar, bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 64, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"(bar), "r"((uint32_t)x)
      : "memory");
  return y != 0;
}

// In both register splits' code: what follows stays within the one or the other.
__device__ __forceinline__ void end_sync() { asm volatile("bar.sync %0, %1;" ::"n"(kEndBar), "n"(kTcThreads) : "memory"); }

__device__ __forceinline__ bool tile_any(int bar, bool x) {
  uint32_t y;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\tbar.red.or.pred q, %1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(y)
      : "r"(bar), "r"((uint32_t)x)
      : "memory");
  return y != 0;
}

// One piece of work: 256 packed rows of a sequence, one key/value head, keys
// [k0, k1).
struct __align__(16) Work {
  int seq, kvh, split, r0;            // seq < 0: no more
  int rows, q0, off, kvn;             // the sequence's packed rows and first token; its SeqTask's off, kvn
  int k0, k1, nt[2];                  // key tiles of the two row tiles
  int first;                          // keys that all rows see
  int pad[3];
};

// Rows r0 .. r1 - 1 of a tile of values in shared memory: elements that are not
// finite become zeros.  By a warp; whether any did.
template <int HALVES>
static __device__ __noinline__ bool clean_tile(uint8_t* vt, int r0, int r1) {
  const int lane = threadIdx.x & 31;
  const __half2 zero = __floats2half2_rn(0.0f, 0.0f);
  __half2 odd[4] = {zero, zero, zero, zero};             // NaN once one was met
#pragma unroll 1
  for (int h = 0; h < HALVES; ++h)
#pragma unroll 1
    for (int o = r0 * 128 + lane * 16; o < r1 * 128; o += 8 * 512) {
      uint4 u[8];
#pragma unroll
      for (int x = 0; x < 8; ++x)
        u[x] = o + x * 512 < r1 * 128 ? *reinterpret_cast<const uint4*>(vt + h * 16384 + o + x * 512) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const uint32_t w[4] = {u[x].x, u[x].y, u[x].z, u[x].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) odd[i] = __hfma2(*reinterpret_cast<const __half2*>(&w[i]), zero, odd[i]);
      }
    }
  const float2 f = __half22float2(__hadd2(__hadd2(odd[0], odd[1]), __hadd2(odd[2], odd[3])));
  if (!__any_sync(0xffffffffu, isnan(f.x) || isnan(f.y))) return false;
#pragma unroll 1
  for (int h = 0; h < HALVES; ++h)
#pragma unroll 1
    for (int o = r0 * 128 + lane * 16; o < r1 * 128; o += 512) {
      uint4* at = reinterpret_cast<uint4*>(vt + h * 16384 + o);
      uint4 u = *at;
      if (clean_piece<__half>(u)) *at = u;
    }
  return true;
}

constexpr uint32_t kNanRow = 0xffffffffu;    // in a row that is NaN by its weights: a NaN that no arithmetic gives

// A piece that may have met values that are not finite: an element of an output
// or partial row becomes the sum of those that its row sees, where there are
// such.  By a warp: a lane looks at eight dims of every KP-th key, 8 KP keys in
// flight, and adds up what the keys that all rows see have; of the others (at
// most 255), which were left out, it notes the ones with such a value, and adds
// them as the rows come to see them.
template <int HD>
static __device__ __noinline__ void patch_piece(const PagedProblem& p, const SeqTask& t, int kvh, int split, int r0) {
  constexpr int PC = HD / 8, KP = 32 / PC, U = 8;
  const int lane = threadIdx.x & 31, d0 = lane % PC * 8, sub = lane / PC;
  const bool has = d0 < p.hd;
  const int rows = min(t.qn * p.group, r0 + 2 * kRows), k0 = p.splits ? split * p.chunk : 0;
  int k1 = seen(p, t, row_token(p, rows - 1));
  if (p.splits) k1 = min(k1, k0 + p.chunk);
  const int first = max(k0, min(k1, seen(p, t, row_token(p, r0))));
  const __half* vb = reinterpret_cast<const __half*>(p.v) + d0;
  float s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s[e] = 0.0f;
  auto add = [&](const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      if (not_finite(f.x)) s[2 * i] += f.x;
      if (not_finite(f.y)) s[2 * i + 1] += f.y;
    }
  };
  uint32_t noted = 0;                                    // lane w: keys first + 32 w ..
#pragma unroll 1
  for (int j = k0; j < k1; j += U * KP) {
    uint4 u[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int key = j + x * KP + sub;
      const long long off = has && key < k1 ? kv_off(p, t.table, key, kvh) : -1;
      u[x] = off >= 0 ? *reinterpret_cast<const uint4*>(vb + off) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      uint4 c = u[x];
      const int key = j + x * KP + sub;
      const bool bad = clean_piece<__half>(c);
      if (bad && key < first) add(u[x]);
      const uint32_t late = __ballot_sync(0xffffffffu, bad && key >= first);
#pragma unroll
      for (int q = 0; q < KP; ++q) {
        const int at = j + x * KP + q - first;
        if (late >> (q * PC) & ((1u << PC) - 1) && lane == at >> 5) noted |= 1u << (at & 31);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    for (int o = PC; o < 32; o <<= 1) s[e] += __shfl_xor_sync(0xffffffffu, s[e], o);
  bool any = noted != 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) any |= !(s[e] == 0.0f);
  if (!__any_sync(0xffffffffu, any)) return;
  const int type = p.splits ? TOSK_F32 : p.type;
  void* out = p.splits ? p.part_o : p.out;
  int j = first;
#pragma unroll 1
  for (int rb = r0; rb < rows; rb += 32) {
    // a row a lane: the keys it sees, where it lies, whether it stays as it is
    const int r = min(rb + lane, rows - 1), tok = t.q0 + row_token(p, r), head = kvh * p.group + row_head(p, r);
    const long long at =
        p.splits ? ((long long)(p.slot0 + split) * p.total_q * p.heads + (long long)tok * p.heads + head) * p.hd
                 : (long long)tok * p.out_stride + (long long)head * p.hd;
    const int lim = min(k1, seen(p, t, row_token(p, r)));
    bool stays = lim <= k0;
    if (!stays)
      stays = type == TOSK_F32 ? reinterpret_cast<const uint32_t*>(out)[at] == kNanRow
                               : reinterpret_cast<const uint16_t*>(out)[at] == (uint16_t)kNanRow;
    const uint32_t skip = __ballot_sync(0xffffffffu, stays);
#pragma unroll 1
    for (int x = 0; x < min(32, rows - rb); ++x) {
      const int l = __shfl_sync(0xffffffffu, lim, x);
      for (; j < l; ++j)
        if (__shfl_sync(0xffffffffu, noted, (j - first) >> 5) >> ((j - first) & 31) & 1) {
          const long long off = has ? kv_off(p, t.table, j, kvh) : -1;
          if (off >= 0) add(*reinterpret_cast<const uint4*>(vb + off));
        }
      const long long to = __shfl_sync(0xffffffffu, at, x) + d0;
      if (skip >> x & 1 || !has || sub) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(s[e] == 0.0f)) store_elem(out, type, to + e, s[e]);
    }
  }
}

// Values that are not finite were left out or met: the CTA's pieces once more, by
// two warps, for whom nobody waits but the end of the CTA.
template <int HD>
static __device__ __noinline__ void patch_pieces(const PagedProblem& p, int which) {
  const int splits = p.splits ? p.splits : 1;
  PlanCursor cur = {0, 0};
  for (int k = 0;; ++k) {
    const int g = piece_of(k);
    const TileId id = pick_tile(p, g / p.n_kv / splits, cur);
    if (id.seq < 0) return;
    if ((k & 1) == which) patch_piece<HD>(p, seq_task(p, id.seq), g % p.n_kv, g / p.n_kv % splits, id.rt * 2 * kRows);
  }
}

// fp32 rows meet an infinite element of a key as infinity times the high part
// plus infinity times the low part of q, which is NaN where the low part is
// zero or of the other sign.  Of 64 keys' scores in tensor memory, those that
// are NaN by infinite elements alone become the sum of q's elements times them.
// A row a lane, of token tok and head `head`; left: keys from key0 on that it
// sees, 0: it has no scores to mend.
static __device__ __noinline__ void infinite_scores(const PagedProblem& p, uint32_t ts, int seq, int tok, int head, int key0,
                                                    int left) {
  const int lane = threadIdx.x & 31, kvh = head / p.group;
  const int* table = p.table + (long long)seq * p.table_stride;
  const float* q = reinterpret_cast<const float*>(p.q) + (long long)tok * p.q_stride + (long long)head * p.hd;
#pragma unroll 1
  for (int c = 0; c < 64; c += 8) {
    uint32_t s[8];
    tc_ld8(ts + c, s);
    tc_wait_ld8(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool mine = c + e < left && isnan(__uint_as_float(s[e]));
      if (!__any_sync(0xffffffffu, mine)) continue;
      const long long off = kv_off(p, table, key0 + c + e, kvh);
      float acc = 0.0f;
      bool nan = false;
#pragma unroll 1
      for (int i = 0; i < p.hd; i += 32) {
        const float k = off >= 0 && lane + i < p.hd ? load_elem(p.k, p.kv_type, off + lane + i) : 0.0f;
        nan |= __any_sync(0xffffffffu, isnan(k));
        uint32_t inf = __ballot_sync(0xffffffffu, isinf(k));
        while (inf) {
          const int b = __ffs(inf) - 1;
          inf &= inf - 1;
          const float kb = __shfl_sync(0xffffffffu, k, b);
          if (mine) acc += q[i + b] * kb;
        }
      }
      if (mine && !nan && !(acc == 0.0f)) s[e] = __float_as_uint(p.scale_log2 < 0.0f ? -acc : acc);
    }
    tc_st4(ts + c, {s[0], s[1], s[2], s[3]});
    tc_st4(ts + c + 4, {s[4], s[5], s[6], s[7]});
  }
  tmem_st_wait();
}

// Q rows of a row tile, 16 rows a warp, 8 or 16 lanes a row, eight elements
// each: asked into L2 early, then through registers into the swizzled K-major
// layout.  fp32 rows are scaled by a power of two and split into fp16 pairs.
template <int HD, bool SPLIT>
struct QRows {
  static constexpr int CH = HD / 8, RPS = 32 / CH, STEPS = 16 / RPS, PARTS = SPLIT ? 2 : 1;
  static constexpr int BATCH = STEPS;      // all in flight at once
  long long my_at;                    // lane i: element offset of row i (of the warp's 16), -1: none

  __device__ __forceinline__ void place(const PagedProblem& p, const Work& w, int row0) {
    const int pr = w.r0 + row0 + (threadIdx.x & 15);
    my_at = pr < w.rows ? (long long)(w.q0 + row_token(p, pr)) * p.q_stride +
                              (long long)(w.kvh * p.group + row_head(p, pr)) * p.hd
                        : -1;
  }
  // the rows' 128-byte lines into L2 (a row's first and second half of the warp each take every other one)
  __device__ __forceinline__ void ask(const PagedProblem& p) {
    const int es = SPLIT ? 4 : 2, first = (threadIdx.x >> 4) & 1;
    if (my_at >= 0)
      for (int o = first * 128; o < p.hd * es; o += 256)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const uint8_t*>(p.q) + my_at * es + o));
  }
  __device__ __forceinline__ void fetch(const PagedProblem& p, int s0, int vec, uint4 (&u)[BATCH][PARTS]) {
    const int lane = threadIdx.x & 31, c = lane % CH, rr0 = lane / CH;
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const long long row_at = __shfl_sync(0xffffffffu, my_at, (s0 + q) * RPS + rr0);
      const long long at = row_at + 8 * c;
#pragma unroll
      for (int w = 0; w < PARTS; ++w) u[q][w] = make_uint4(0, 0, 0, 0);
      if (row_at >= 0 && 8 * c < p.hd) {                       // hd is a multiple of 8
        if (vec) {
#pragma unroll
          for (int w = 0; w < PARTS; ++w)
            u[q][w] = SPLIT ? *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.q) + at + 4 * w)
                            : *reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(p.q) + at);
        } else if (SPLIT) {
          const uint32_t* x = reinterpret_cast<const uint32_t*>(p.q) + at;
          u[q][0] = make_uint4(x[0], x[1], x[2], x[3]);
          u[q][PARTS - 1] = make_uint4(x[4], x[5], x[6], x[7]);
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(p.q) + at;
          u[q][0] = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                               h[6] | (uint32_t)h[7] << 16);
        }
      }
    }
  }
  // dst: the row tile's high parts (low parts follow); what undoes a row's
  // scale goes to inv[row]
  __device__ __forceinline__ void store(const PagedProblem& p, int s0, int row0, uint8_t* dst, float* inv,
                                        const uint4 (&u)[BATCH][PARTS]) {
    const int lane = threadIdx.x & 31, c = lane % CH, rr0 = lane / CH;
    const float sgn = p.scale_log2 < 0.0f ? -1.0f : 1.0f;      // a negative scale goes into q
#pragma unroll
    for (int q = 0; q < BATCH; ++q) {
      const int row = row0 + (s0 + q) * RPS + rr0;
      uint8_t* d = dst + (c >> 3) * 16384 + sw128(row, c & 7);
      if (SPLIT) {
        const uint4 v0 = u[q][0], v1 = u[q][PARTS - 1];
        const float x[8] = {__uint_as_float(v0.x), __uint_as_float(v0.y), __uint_as_float(v0.z), __uint_as_float(v0.w),
                            __uint_as_float(v1.x), __uint_as_float(v1.y), __uint_as_float(v1.z), __uint_as_float(v1.w)};
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
#pragma unroll
        for (int o = CH / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float s2 = pow2_to_2p13(mx), f = sgn * s2;       // exact: powers of two
        if (c == 0) inv[row] = pow2_inverse(s2);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) split_pair(x[2 * e] * f, x[2 * e + 1] * f, hi[e], lo[e]);
        *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(d + TcShape<HD, SPLIT>::kTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      } else {
        const uint32_t flip = sgn < 0.0f ? 0x80008000u : 0u;
        *reinterpret_cast<uint4*>(d) =
            make_uint4(u[q][0].x ^ flip, u[q][0].y ^ flip, u[q][0].z ^ flip, u[q][0].w ^ flip);
      }
    }
  }
};

template <int HD, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1) paged_attn_tc_kernel(const __grid_constant__ TcArgs a) {
  using T = TcShape<HD, SPLIT>;
  extern __shared__ __align__(1024) uint8_t sm[];
  uint8_t* sq = sm;                                   // [tile][hi, lo][half][128 rows x 128 B]; then output rows
  uint8_t* ring = sm + T::kQ;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + T::kSlots * T::kTile + T::kStage);
  uint64_t* empty = full + T::kSlots;
  uint64_t* sfull = empty + T::kSlots;                // [2]: S of tile t is there
  uint64_t* pfull = sfull + 2;                        // [2][2]: half the keys of tile t's P are there
  uint64_t* odone = pfull + 4;                        // [2]: O of tile t has taken P in
  uint64_t* qfull = odone + 2;                        // [2][2]: Q of tile t of an even, an odd piece of work
  uint64_t* wfull = qfull + 4;                        // [2]: a piece of work is posted
  uint64_t* wempty = wfull + 2;                       // [2]: and read by all
  uint64_t* tailbar = wempty + 2;                     // the copy warp's own
  uint32_t& tmem_at = *reinterpret_cast<uint32_t*>(tailbar + 1);
  static_assert(T::kBars % 2 == 1, "work lies on 16 bytes");
  Work* work = reinterpret_cast<Work*>(tailbar + 2);  // [2]
  float* sx = reinterpret_cast<float*>(work + 2);     // [tile][half of the keys][row]: exchange of the two halves
  volatile int* odd_seen = reinterpret_cast<int*>(sx + 4 * kRows);   // values that are not finite were left out or met
  const PagedProblem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(sm) & 1023) {                          // the swizzled tiles need it; the launch gives it
    if (tid == 0) atomicCAS(p.err, 0, 41);
    return;
  }
  if (warp == kMmaWarp) tmem_alloc(&tmem_at, 512);
  if (tid == 0) {
    for (int i = 0; i < T::kSlots; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sfull + i, 1);
      mbar_init(pfull + 2 * i, kRows);
      mbar_init(pfull + 2 * i + 1, kRows);
      mbar_init(odone + i, 1);
      mbar_init(qfull + 2 * i, 2 * kRows);
      mbar_init(qfull + 2 * i + 1, 2 * kRows);
      mbar_init(wfull + i, 1);
      mbar_init(wempty + i, kCopyWarp + 2);           // the softmax warps, the copy warp, the MMA thread
    }
    mbar_init(tailbar, 1);
    mbar_fence_init();
    *odd_seen = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // The previous kernel is awaited by those who read or write memory; what
  // may follow starts after that (the copy warp's word for the CTA).

  if (warp >= kCopyWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcRegsRest));
    if (warp == kPlanWarp) {
      // ------------------------------------------------------------ the plan
      // The pieces, longest first, dealt so that the CTAs' sums are even.
      if (p.fixed_kv < 0) pdl_wait();                  // a prefix is planned from the arguments alone
      bool ok = true, more = true;
      int posted = 0;
      PlanCursor cur = {0, 0};
      const int splits = p.splits ? p.splits : 1;
      for (int k = 0; more && ok; ++k) {
        const int g = piece_of(k);
        Work w;
        w.seq = -1;
        w.kvh = g % p.n_kv;
        w.split = g / p.n_kv % splits;
        const TileId id = pick_tile(p, g / p.n_kv / splits, cur);
        more = id.seq >= 0;
        if (more) {
          const SeqTask t = seq_task(p, id.seq);
          w.seq = id.seq;
          w.r0 = id.rt * 2 * kRows;
          w.rows = t.qn * p.group;
          w.q0 = t.q0;
          w.off = t.off;
          w.kvn = t.kvn;
          w.k0 = 0;
          w.k1 = seen(p, t, row_token(p, min(w.rows, w.r0 + 2 * kRows) - 1));
          w.first = seen(p, t, row_token(p, w.r0));
          if (p.splits) {
            w.k0 = w.split * p.chunk;
            w.k1 = min(w.k1, w.k0 + p.chunk);
            if (w.k0 >= w.k1) continue;               // no row of the tile sees a key of this split
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int last = min(w.rows, w.r0 + (i + 1) * kRows) - 1;
            const int e = last >= w.r0 + i * kRows ? min(w.k1, seen(p, t, row_token(p, last))) : 0;
            w.nt[i] = e > w.k0 ? (e - w.k0 + kKeys - 1) / kKeys : 0;
          }
        }
        // for as long as a piece takes: twice the limit
        if (posted >= 2) {
          pdl_wait();
          const uint32_t ph = (posted / 2 - 1) & 1;
          ok = mbar_wait(wempty + (posted & 1), ph, nullptr, 0) || mbar_wait(wempty + (posted & 1), ph, p.err, 42);
        }
        ok = __all_sync(0xffffffffu, ok);
        if (ok && lane == 0) {
          work[posted & 1] = w;
          mbar_arrive(wfull + (posted & 1));
        }
        ++posted;
      }
    } else if (warp == kCopyWarp) {
      // ---------------------------------------------------------- K, V tiles
      pdl_wait();
      pdl_trigger();
      bool ok = true;
      int used = 0, tails = 0;                        // slots filled; tiles cut off by the key range
      for (int n = 0; ok; ++n) {
        ok = mbar_wait(wfull + (n & 1), (n >> 1) & 1, p.err, 43);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const Work& w = work[n & 1];
        const int seq = w.seq, kvh = w.kvh, k0 = w.k0, k1 = w.k1, first = w.first, nmax = max(w.nt[0], w.nt[1]);
        __syncwarp();
        if (lane == 0) mbar_arrive(wempty + (n & 1));
        if (seq < 0) break;
        const int* table = p.table + (long long)seq * p.table_stride;
        // lane i: the page of box i of the next tile, asked for a tile ahead
        auto page_of_box = [&](int j) {
          const int key = k0 + j * kKeys + lane * a.box_rows;
          return lane * a.box_rows < kKeys && key < k1 ? table[p.pshift >= 0 ? key >> p.pshift : key / p.page_size] : -1;
        };
        int ahead = page_of_box(0);
        for (int j = 0; j < nmax && ok; ++j) {
          const int kt = k0 + j * kKeys, have = min(kKeys, k1 - kt);
          const int need = (have + a.box_rows - 1) / a.box_rows;
          const int page = ahead, key = kt + lane * a.box_rows;
          const int row = p.pshift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
          ahead = page_of_box(j + 1);
          // K and V written out, each with its tensor map: chosen in a loop, the
          // copies of 16-token pages fall behind the MMAs (700 rows behind 20,000
          // keys 575 us, so 542)
          auto slot_free = [&]() {
            const int s = used % T::kSlots;
            if (used >= T::kSlots) ok = mbar_wait(empty + s, (used / T::kSlots - 1) & 1, p.err, 31);
            ok = __all_sync(0xffffffffu, ok);
            return s;
          };
          auto bring = [&](const CUtensorMap* map, int s, uint64_t* bar) {
            if (lane == 0) mbar_arrive_expect_tx(bar, need * a.box_rows * HD * 2);
            __syncwarp();
            if (lane < need) {
              uint8_t* dst = ring + s * T::kTile + lane * a.box_rows * 128;
#pragma unroll
              for (int h = 0; h < T::kHalves; ++h) tma_page(dst + h * 16384, map, 64 * h, kvh, row, page, bar);
            }
          };
          const int sk = slot_free();
          if (!ok) break;
          bring(&a.mk, sk, full + sk);
          ++used;
          const int sv = slot_free();
          if (!ok) break;
          // value rows behind the key range, and what is not finite where
          // only some rows see a key, meet weights of 0: zeros instead
          const bool some = kt + have > first, cut = some || have < kKeys;
          bring(&a.mv, sv, cut ? tailbar : full + sv);
          if (cut) {
            ok = mbar_wait(tailbar, tails & 1, p.err, 32);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            ++tails;
            uint8_t* tile = ring + sv * T::kTile;
            for (int h = 0; h < T::kHalves; ++h)
              for (int o = have * 128 + lane * 16; o < kKeys * 128; o += 512)
                *reinterpret_cast<uint4*>(tile + h * 16384 + o) = make_uint4(0, 0, 0, 0);
            if (some && clean_tile<T::kHalves>(tile, max(first - kt, 0), have)) *odd_seen = 1;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + sv);
          }
          ++used;
        }
      }
      // every copy lands before the CTA may end
      for (int i = max(0, used - T::kSlots); i < used; ++i)
        mbar_wait(full + i % T::kSlots, (i / T::kSlots) & 1, p.err, 33);
    } else if (warp == kMmaWarp) {
      // ----------------------------------------------------- MMAs, one thread
      if (elect_one()) {
        constexpr uint32_t kIdS = (1u << 4) | (8u << 24) | ((uint32_t)(kKeys >> 3) << 17);
        constexpr uint32_t kIdO = (1u << 4) | (8u << 24) | ((uint32_t)(HD >> 3) << 17) | (1u << 16);   // V is N-major
        const uint32_t tmem = tmem_at;
        pdl_wait();                                   // its own waits are not to count what came before
        bool ok = true;
        int base = 0, c0 = 0, c1 = 0;                 // ring uses and key tiles of the two row tiles before this piece
        for (int n = 0; ok; ++n) {
          ok = mbar_wait(wfull + (n & 1), (n >> 1) & 1, p.err, 44);
          if (!ok) break;
          const Work& w = work[n & 1];
          if (w.seq < 0) break;
          const int n0 = w.nt[0], n1 = w.nt[1], nmax = max(n0, n1);
          // S of row tile i on key tile j (the first of the two row tiles waits for K)
          auto issue_s = [&](int i, int j) {
            const int u = base + 2 * j, slot = u % T::kSlots;
            if (i == 0 || j >= n0) ok = ok && mbar_wait(full + slot, (u / T::kSlots) & 1, p.err, 34);
            if (!ok) return;
            const uint32_t kd = desc_k(smem_u32(ring + slot * T::kTile));
            const uint32_t qd = desc_k(smem_u32(sq + i * (T::kQ / 2)));
            const uint32_t d = tmem + i * kKeys;
#pragma unroll
            for (int part = 0; part < (SPLIT ? 2 : 1); ++part)          // low parts first: less is cut off small sums
#pragma unroll
              for (int k = 0; k < HD / 16; ++k) {
                const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                mma_f16_ss(d, qd + (SPLIT && part == 0 ? T::kTile >> 4 : 0) + off, kd + off, kIdS, part + k > 0);
              }
            mma_commit(sfull + i);
            if (i == 1 || j >= n1) mma_commit(empty + slot);
          };
          for (int i = 0; i < 2 && ok; ++i) {
            ok = mbar_wait(qfull + 2 * i + (n & 1), (n >> 1) & 1, p.err, 35);
            tc_fence_after();
            if (ok && (i ? n1 : n0) > 0) issue_s(i, 0);
          }
          if (!ok) break;
          mbar_arrive(wempty + (n & 1));
          for (int j = 0; j < nmax && ok; ++j)
            for (int i = 0; i < 2 && ok; ++i) {
              if (j >= (i ? n1 : n0)) continue;
              const int u = base + 2 * j + 1, slot = u % T::kSlots;
              if (i == 0 || j >= n0) ok = mbar_wait(full + slot, (u / T::kSlots) & 1, p.err, 36);
              const uint32_t vd0 = desc_mn(smem_u32(ring + slot * T::kTile), 16384);
              const uint32_t d = tmem + 256 + i * HD;
              const uint32_t ph = ((i ? c1 : c0) + j) & 1;
              for (int half = 0; half < 2 && ok; ++half) {
                ok = mbar_wait(pfull + 2 * i + half, ph, p.err, 37);
                if (!ok) break;
                tc_fence_after();
                const uint32_t vd = vd0 + half * (kKeys / 2 * 128 >> 4), pa = tmem + i * kKeys + half * 64;
#pragma unroll
                for (int part = 0; part < (SPLIT ? 2 : 1); ++part)
#pragma unroll
                  for (int k = 0; k < kKeys / 32; ++k)
                    mma_f16_ts(d, pa + (k >> 1) * 32 + part * 16 + (k & 1) * 8, vd + (k * 2048 >> 4), kIdO,
                               part + k + half > 0 ? true : j % fold_tiles(SPLIT, i ? n1 : n0) != 0);
              }
              if (!ok) break;
              mma_commit(odone + i);
              if (i == 1 || j >= n1) mma_commit(empty + slot);
              if (j + 1 < (i ? n1 : n0)) issue_s(i, j + 1);
            }
          base += 2 * nmax;
          c0 += n0;
          c1 += n1;
        }
      }
      __syncwarp();
    }
    end_sync();
    if (warp == kMmaWarp) {
      tc_fence_after();
      tmem_dealloc(tmem_at, 512);
    }
    if (warp > kMmaWarp && *odd_seen) patch_pieces<HD>(p, warp & 1);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTcRegsSoftmax));
    // --------------------------------------------------------------- softmax
    // row tile, half of a tile's keys (and of the output's dims), 32 rows
    const int i = warp >> 3, hf = (warp >> 2) & 1, wq = warp & 3, r = wq * 32 + lane;
    const int bar = 1 + i * 4 + wq;                                      // this warp and the other half's
    const int row0 = i * kRows + (warp & 7) * 16;                        // Q rows this warp brings (of 256)
    uint8_t* q_tile = sq + i * (T::kQ / 2);
    float* mine = sx + (i * 2 + hf) * kRows + r;
    float* other = sx + (i * 2 + (hf ^ 1)) * kRows + r;
    const uint32_t lanes = (uint32_t)wq << 21;                          // TMEM lane of the warp's first row, << 16
    const uint32_t ts = tmem_at + lanes + i * kKeys, to = tmem_at + lanes + 256 + i * HD + hf * (HD / 2);
    uint8_t* stage = (T::kStage ? ring + T::kSlots * T::kTile + i * 32768 : q_tile) + (hf * 4 + wq) * 4096;
    bool ok = true;     // a wait that ran out: no more waiting, and all warps of the row tile leave together
    int cnt = 0;                                                        // key tiles so far
    pdl_wait();
    QRows<HD, SPLIT> qr;
    Work w;
    // the n-th piece of work, and its Q rows on their way to L2
    auto take = [&](int n) {
      if (ok) ok = mbar_wait(wfull + (n & 1), (n >> 1) & 1, p.err, 38);
      w = work[n & 1];
      if (!__all_sync(0xffffffffu, ok)) w.seq = -1;
      __syncwarp();
      if (w.seq >= 0) {
        if (lane == 0) mbar_arrive(wempty + (n & 1));
        qr.place(p, w, row0);
        if (n) qr.ask(p);                                                // the first is fetched at once
      }
    };
    take(0);
    for (int n = 0;; ++n) {
      // also: every warp of the row tile has written its last output rows
      if (tile_any(kTileBar + i, !ok) || w.seq < 0) break;
#pragma unroll 1
      for (int s0 = 0; s0 < QRows<HD, SPLIT>::STEPS; s0 += QRows<HD, SPLIT>::BATCH) {
        uint4 u[QRows<HD, SPLIT>::BATCH][QRows<HD, SPLIT>::PARTS];
        qr.fetch(p, s0, a.q_vec, u);
        qr.store(p, s0, (warp & 7) * 16, q_tile, sx + i * 2 * kRows, u);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(qfull + 2 * i + (n & 1));
      float inv_q = 1.0f;                                                // undoes the row's scale
      if (SPLIT) {
        tile_any(kTileBar + i, false);
        inv_q = sx[i * 2 * kRows + r];
        tile_any(kTileBar + i, false);                                   // read by all: sx is free
      }
      // without a key tile no MMA stands between the warps' Q rows and the
      // output rows that go to the same place
      if (w.nt[i] == 0) tile_any(kTileBar + i, false);
      const int pr = w.r0 + i * kRows + r, nt = w.nt[i], k0 = w.k0;
      const bool live = pr < w.rows;
      const int tok = w.q0 + row_token(p, pr), head = w.kvh * p.group + row_head(p, pr), seq = w.seq;
      const SeqTask st = {w.q0, 0, w.kvn, w.off, nullptr};
      const int all = live ? seen(p, st, row_token(p, pr)) : 0, lim = min(all, w.k1);   // keys this row sees, here
      const long long slot = (long long)(p.slot0 + (p.splits ? w.split : 0)) * p.total_q * p.heads + (long long)tok * p.heads + head;
      const float sc = fmaxf(fabsf(p.scale_log2) * inv_q, 1.2e-38f);   // not 0: a masked score is -inf * sc
      float m = -INFINITY, l = 0.0f;
      const int chain = fold_tiles(SPLIT, nt);
      for (int j = 0; j < nt; ++j) {
        if (j > 0 && j % chain == 0) {
          // The tensor cores cut off what their accumulator has no room for,
          // so a long chain of sums shrinks.  Every few tiles the sums are
          // added up in memory, rounded to nearest, and the chain begins anew.
          if (ok) ok = mbar_wait(odone + i, (cnt + j - 1) & 1, p.err, 46);
          __syncwarp();
          tc_fence_after();
          fold_cols(p, to, HD / 2, j == chain);
          tc_fence_before();
          pair_sync(bar);                                               // the MMAs overwrite all dims
        }
        if (ok) ok = mbar_wait(sfull + i, (cnt + j) & 1, p.err, 39);
        __syncwarp();
        tc_fence_after();
        const int left = lim - (k0 + j * kKeys) - 64 * hf;              // keys of this half tile that the row sees
        const bool cut = __any_sync(0xffffffffu, left < 64);
        const float2 sc2 = make_float2(sc, sc);
        // the row's maximum over this half's keys
        auto half_top = [&]() {
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t s[32];
            tc_ld32(ts + 64 * hf + 32 * c, s);
            tc_wait_ld(s);
            if (cut) mask_from(s, left - 32 * c);
            top = SPLIT ? max_nan(top, max_of<true>(s)) : fmaxf(top, max_of<false>(s));
          }
          return top * sc;
        };
        // a first or a much larger maximum: agree on the row's over both
        // halves, scale O (each half its dims) and l to it
        auto agree = [&](float top) {
          *mine = top;
          pair_sync(bar);
          top = fmaxf(top, *other);
          const float mn = j == 0 || top > m + kSlack ? top : m;
          if (j > 0) {
            const float f = mn == m ? 1.0f : exp2f(m - mn);
            if (ok) ok = mbar_wait(odone + i, (cnt + j - 1) & 1, p.err, 40);
            __syncwarp();
            tc_fence_after();
            scale_cols(to, HD / 2, f);
            l *= f;
            if (j >= chain) fold_scale(p, HD / 2, f);
            // either half's P lets MMAs add to all dims: both halves' O first
            tmem_st_wait();
            tc_fence_before();
            pair_sync(bar);
          }
          m = mn;
        };
        float2 sum[2];
        if (SPLIT) {
          // S is read twice, for the maximum and for the weights: the parts of
          // P take too many registers to be kept until the maximum is known
          float top = half_top();
          if (pair_any(bar, j == 0 || !(top <= m + kSlack || isnan(l)))) {
            if (__any_sync(0xffffffffu, isnan(top) && !isnan(l))) {
              infinite_scores(p, ts + 64 * hf, seq, tok, head, k0 + j * kKeys + 64 * hf, isnan(l) ? 0 : left);
              top = half_top();
            }
            agree(top);
          }
          const float bias = kBias - (m == -INFINITY ? 0.0f : m);
          const float2 bias2 = make_float2(bias, bias);
          sum[0] = sum[1] = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t s[32], hi[16], lo[16];
            tc_ld32(ts + 64 * hf + 32 * c, s);
            tc_wait_ld(s);
            if (cut) mask_from(s, left - 32 * c);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sc2, bias2);
              const float2 v = make_float2(ex2(x.x), ex2(x.y));
              sum[e & 1] = __fadd2_rn(sum[e & 1], v);
              split_pair(v.x, v.y, hi[e], lo[e]);
            }
            // over these 32 keys' own S: high parts, then low parts
            tmem_st16(ts + 64 * hf + 32 * c, hi);
            tmem_st16(ts + 64 * hf + 32 * c + 16, lo);
          }
        } else {
          // the weights under the maximum so far, and the maximum with them;
          // P goes over S only once no row of the two halves has outgrown it
          float top;
          bool again = j == 0;
          if (!again) {
            uint32_t hi[2][16];
            const float bias = kBias - (m == -INFINITY ? 0.0f : m);
            const float2 bias2 = make_float2(bias, bias);
            sum[0] = sum[1] = make_float2(0.0f, 0.0f);
            top = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t s[16];
              tc_ld16(ts + 64 * hf + 16 * c, s);
              tc_wait_ld16(s);
              if (cut) mask_from(s, left - 16 * c);
              top = fmaxf(top, max_of<false>(s));
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float2 x =
                    __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sc2, bias2);
                const float2 v = e % kPoly == kPoly - 1 ? exp2_fma(x) : make_float2(ex2(x.x), ex2(x.y));
                sum[e & 1] = __fadd2_rn(sum[e & 1], v);
                const __half2 H = __floats2half2_rn(v.x, v.y);
                hi[c >> 1][8 * (c & 1) + e] = *reinterpret_cast<const uint32_t*>(&H);
              }
            }
            top *= sc;
            again = pair_any(bar, top > m + kSlack);
            if (!again) {
              tmem_st16(ts + 64 * hf, hi[0]);
              tmem_st16(ts + 64 * hf + 32, hi[1]);
            }
          } else {
            top = half_top();
          }
          if (again) {
            agree(top);
            const float bias = kBias - (m == -INFINITY ? 0.0f : m);
            const float2 bias2 = make_float2(bias, bias);
            sum[0] = sum[1] = make_float2(0.0f, 0.0f);
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {                               // 8 keys' P over S that has been read
              uint32_t s[8], hi[4];
              tc_ld8(ts + 64 * hf + 8 * c, s);
              tc_wait_ld8(s);
              if (cut) mask_from(s, left - 8 * c);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 x =
                    __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sc2, bias2);
                const float2 v = make_float2(ex2(x.x), ex2(x.y));
                sum[0] = __fadd2_rn(sum[0], v);
                const __half2 H = __floats2half2_rn(v.x, v.y);
                hi[e] = *reinterpret_cast<const uint32_t*>(&H);
              }
              tc_st4(ts + 64 * hf + 32 * (c >> 2) + 4 * (c & 3), hi);
            }
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(pfull + 2 * i + hf);
        const float part = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        // a NaN score that exp2_fma met makes the row NaN as any other does
        // (a maximum that keeps NaN costs packed prompts 1%)
        l += !SPLIT && part >= kNanWeight ? __int_as_float(0x7fffffff) : part;
      }
      cnt += nt;
      take(n + 1);
      if (ok && nt > 0) ok = mbar_wait(odone + i, (cnt - 1) & 1, p.err, 45);
      __syncwarp();
      tc_fence_after();
      pair_sync(bar);
      *mine = l;
      pair_sync(bar);
      l += *other;
      // ----------------------------------------------------------- output
      // A row a thread in tensor memory; 32 dims (fp32) or the half's dims
      // (fp16) go through shared memory (Q's, which no MMA reads any more),
      // 128 bytes a row, so that eight lanes write a row's pieces side by side.
      if (lim <= k0) l = 0.0f;                                          // sees nothing here, whatever exp2 made of -inf
      const bool f32 = p.splits || p.type == TOSK_F32;
      const int es = f32 ? 4 : 2;
      const float inv = l == 0.0f || nt == 0 ? 0.0f : p.splits && !isnan(l) ? 1.0f : 1.0f / l;
      if (p.splits && live && hf == 0) p.part_ml[slot] = make_float2(m - kBias, l);
      const long long row_at =
          !live ? -1 : p.splits ? slot * p.hd : (long long)tok * p.out_stride + (long long)head * p.hd;
      float2 odd = make_float2(0.0f, 0.0f);                             // NaN once an infinity or NaN was seen
      const bool none = __any_sync(0xffffffffu, !(inv > 0.0f));        // or NaN, by the weights
      // the staged rows' `bytes` to dims from dim0 on
      auto flush = [&](int dim0, int bytes) {
        __syncwarp();
        const int c = lane & 7, dim = dim0 + c * (16 / es);
#pragma unroll 4
        for (int q = 0; q < 8; ++q) {
          const int row = q * 4 + (lane >> 3);
          const long long at = __shfl_sync(0xffffffffu, row_at, row);
          if (at < 0 || c * 16 >= bytes || dim >= p.hd) continue;
          const uint4 v = *reinterpret_cast<const uint4*>(stage + sw128(row, c));
          if (p.splits) {
            *reinterpret_cast<uint4*>(p.part_o + at + dim) = v;
          } else if (a.out_vec) {
            *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p.out) + (at + dim) * es) = v;
          } else {
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (f32) {
                reinterpret_cast<uint32_t*>(p.out)[at + dim + e] = x[e];
              } else {
                reinterpret_cast<uint16_t*>(p.out)[at + dim + 2 * e] = (uint16_t)x[e];
                reinterpret_cast<uint16_t*>(p.out)[at + dim + 2 * e + 1] = (uint16_t)(x[e] >> 16);
              }
            }
          }
        }
        __syncwarp();
      };
      if (nt > chain) fold_back(p, to, HD / 2);
#pragma unroll 1
      for (int c32 = 0; c32 < HD / 64; ++c32) {
        uint32_t o[32];
        tc_ld32(to + 32 * c32, o);
        tc_wait_ld(o);
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 v = __fmul2_rn(make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), make_float2(inv, inv));
          odd = __ffma2_rn(v, make_float2(0.0f, 0.0f), odd);
          o[e] = __float_as_uint(v.x);
          o[e + 1] = __float_as_uint(v.y);
        }
        if (none) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = inv == 0.0f ? 0u : isnan(inv) ? kNanRow : o[e];
        }
        if (f32) {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<uint4*>(stage + sw128(lane, c)) = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
          flush(hf * (HD / 2) + 32 * c32, 128);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t h[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const __half2 H = __floats2half2_rn(__uint_as_float(o[8 * c + 2 * q]), __uint_as_float(o[8 * c + 2 * q + 1]));
              h[q] = none && isnan(inv) ? kNanRow : *reinterpret_cast<const uint32_t*>(&H);
            }
            *reinterpret_cast<uint4*>(stage + sw128(lane, 4 * c32 + c)) = make_uint4(h[0], h[1], h[2], h[3]);
          }
        }
      }
      if (!f32) flush(hf * (HD / 2), HD);
      tc_fence_before();                                                // O and S are read: the next piece's MMAs may come
      if (live && !isnan(l) && isnan(odd.x + odd.y)) *odd_seen = 1;      // not by its weights
    }
    end_sync();
  }
}

}  // namespace tos

using namespace tos;

namespace {
// K or V pool as [page][row][kv head][dim], boxes of box_rows rows of one
// head x 64 dims (dims past hd read as zeros).
bool pool_map(CUtensorMap* m, const void* base, const PagedProblem& p, int box_rows) {
  const PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dim[4] = {(cuuint64_t)p.hd, (cuuint64_t)p.n_kv, (cuuint64_t)p.page_size, (cuuint64_t)p.n_pages};
  const cuuint64_t row = (cuuint64_t)p.n_kv * p.hd * 2;
  const cuuint64_t str[3] = {(cuuint64_t)p.hd * 2, row, row * p.page_size};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)box_rows, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dim, str, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool SPLIT>
int tc_launch(const TcArgs& a, unsigned grid, cudaStream_t st) {
  const void* f = (const void*)paged_attn_tc_kernel<HD, SPLIT>;
  // the softmax warps wait for registers that the launch must have brought
  static const int regs = [f] {
    cudaFuncAttributes fa;
    return cudaFuncGetAttributes(&fa, f) == cudaSuccess ? fa.numRegs : 0;
  }();
  if (regs < kTcRegs) return (int)cudaErrorNotSupported;
  const cudaError_t e =
      cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<HD, SPLIT>::kSmem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = TcShape<HD, SPLIT>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<TcArgs*>(&a)};
  return (int)cudaLaunchKernelExC(&cfg, f, args);
}
}  // namespace

namespace tos {

// What the tensor-core kernel takes: an fp16 cache in 16-byte rows of at most
// 128 elements, pages that tile 128 keys or are tiled by them.
bool paged_tc_ok(const PagedProblem& p) {
  const int ps = p.page_size;
  return p.kv_type == TOSK_F16 && p.hd % 8 == 0 && p.hd <= 128 && ps >= 8 &&
         (ps < kKeys ? kKeys % ps == 0 : ps % kKeys == 0) && ((uintptr_t)p.k & 15) == 0 && ((uintptr_t)p.v & 15) == 0 &&
         (long long)ps * p.n_kv * p.hd * 2 < (1ll << 39);
}

// Bytes of PagedProblem::fold that rows over so many keys may need: fp32 rows
// (fp16 rows, beyond more keys; a call's workspace goes by its sizes alone).
size_t paged_tc_fold_bytes(int keys) { return keys > fold_tiles(true, 0) * kKeys ? (size_t)kTcCtas * 2 * kRows * 128 * 4 : 0; }

// Row tiles of one key/value head that a call can have at most.
long long paged_tc_tiles(int n_seqs, int total_q, int max_q, int group) {
  const long long each = ((long long)max_q * group + 2 * kRows - 1) / (2 * kRows) * n_seqs;
  const long long all = (long long)total_q * group / (2 * kRows) + n_seqs;
  return each < all ? each : all;
}

int paged_tc_run(const PagedProblem& p, cudaStream_t st) {
  TcArgs a;
  a.p = p;
  a.box_rows = p.page_size < kKeys ? p.page_size : kKeys;
  long long grid = paged_tc_tiles(p.n_seqs, p.total_q, p.max_q, p.group) * (p.splits ? p.splits : 1) * p.n_kv;
  if (grid > 0x3fffffffll) return (int)cudaErrorInvalidValue;    // the plan counts pieces in 32 bits
  if (grid > kTcCtas) grid = kTcCtas;
  a.q_vec = ((uintptr_t)p.q & 15) == 0 && p.q_stride % (p.type == TOSK_F32 ? 4 : 8) == 0;
  a.out_vec = ((uintptr_t)p.out & 15) == 0 && p.out_stride % (p.type == TOSK_F32 ? 4 : 8) == 0;
  if (!pool_map(&a.mk, p.k, p, a.box_rows) || !pool_map(&a.mv, p.v, p, a.box_rows)) return (int)cudaErrorNotSupported;
  const bool split = p.type == TOSK_F32;
  const int keys = p.splits ? p.chunk : p.fixed_kv >= 0 ? p.fixed_kv : p.max_kv;
  if (!p.fold && keys > fold_tiles(split, 0) * kKeys) return (int)cudaErrorInvalidValue;
  if (p.hd <= 64) return split ? tc_launch<64, true>(a, (unsigned)grid, st) : tc_launch<64, false>(a, (unsigned)grid, st);
  return split ? tc_launch<128, true>(a, (unsigned)grid, st) : tc_launch<128, false>(a, (unsigned)grid, st);
}

}  // namespace tos
