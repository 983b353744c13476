// paged_decode.cu - attention of few rows a sequence over a paged cache:
// single tokens, and prompts too short for the tiled kernels.
//
// fp16 cache.  A CTA takes a chunk of one sequence's keys for one key/value
// head and 8 or 16 packed rows (token, query head of the group); its four
// warps take every fourth 16-key step each and run alone, without any exchange
// until the end:
//   * the step's K and V rows stream through the warp's own ring in shared
//     memory (cp.async, 16-byte pieces, 8 KB a step at 128 dims; the page's
//     table entry fetched one step ahead).  Rows past the end and pages that
//     are none come as zeros;
//   * S = Q K^T and P V by mma.sync m16n8k16: eight rows' fp16 high parts are
//     rows 0-7 of A and their low parts rows 8-15, so fp32 queries and weights
//     cost no extra instruction and the two row halves are added afterwards.
//     tcgen05 wants 128 rows; here there are 8 or 16;
//   * O += P V in fp32 registers, rounded to nearest: an accumulator that the
//     tensor cores keep is cut off at every step (32,768 keys of one sign
//     in one chunk came out 5e-5 small);
//   * running maximum and sum per row as in the prompt kernel (followed
//     only beyond a factor 2^8, weights biased by 2^7).
// The four warps' results are joined in shared memory; with a split key axis
// the joining kernel adds the chunks, without one this kernel adds a prefix's.
//
// Bound: HBM.  A 16-key step is 8 KB and 32 MMAs (HD 128), ~1/16 of what the
// tensor pipe does in the time the bytes take.  Sixteen sequences of 1..4096
// keys, 32 x 128: 91 to 95 us, 5.1 to 5.3 TB/s.  Short sequences leave the bus
// idle while CTAs start and end (32 / 8 heads: 64 of 256 keys 30 us, 2.3 TB/s).
#include <cuda_runtime.h>

#include "paged_common.cuh"
#include "paged_tc.cuh"

namespace tos {

constexpr int kDecWarps = 4;
constexpr int kStep = 16;             // keys a warp step

// DEEP: three stages a warp (of 128 dims) and two CTAs an SM, for many keys a
// CTA; else two stages and three CTAs, which start and end beside one another.
// (64 sequences of ~256 keys: 47.0 us deep, 41.6 not; 16 of ~2000: 92.8, 96.7.)
template <int HD, bool DEEP>
struct DecShape {
  static constexpr int kRow = HD * 2;                            // bytes of a key row in shared memory
  static constexpr int kStage = 2 * kStep * kRow;                // K and V
  static constexpr int kDepth = (HD == 64 ? 2 : 1) * (DEEP || HD == 256 ? 3 : 2);
  static constexpr int kSmem = kDecWarps * kDepth * kStage;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool have) {
  const int n = have ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ int page_of(const PagedProblem& p, int key) {
  return p.pshift >= 0 ? key >> p.pshift : key / p.page_size;
}
// Element offset of a key's row, -1 where its page is none.
__device__ __forceinline__ long long row_at(const PagedProblem& p, int key, int page, int kvh) {
  if (page < 0 || page >= p.n_pages) return -1;
  const int r = p.pshift >= 0 ? key & (p.page_size - 1) : key % p.page_size;
  return (((long long)page * p.page_size + r) * p.n_kv + kvh) * p.hd;
}

// K and V rows of the KEYS keys from `first` on into a stage: rows of `rowb`
// bytes (CH 16-byte pieces, `chs` of them in use, `es` elements each), piece c
// of row k at c ^ (k & 7); V `voff` bytes behind K.  whole: the keys lie in one
// page (`page`), else lane k holds key k's.
template <int KEYS, int CH, typename E>
__device__ __forceinline__ void copy_step(const PagedProblem& p, int whole, int first, int end, int page, int kvh, int chs,
                                          int es, uint32_t dst, uint32_t voff, uint32_t rowb, const E* kb, const E* vb) {
  constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;                 // rows an instruction (CH 64: half a row)
  const int lane = threadIdx.x & 31;
  if (whole) {
    const long long row = row_at(p, first, page, kvh);
    const long long step = (long long)p.n_kv * p.hd;
    const int key0 = lane / CH;
    long long off = row + key0 * step + (lane % CH) * es;
#pragma unroll
    for (int i = 0; i < KEYS * CH / 32; ++i) {
      const int idx = i * 32 + lane, key = idx / CH, c = idx % CH;
      const bool have = row >= 0 && c < chs && first + key < end;
      const long long o = have ? (CH <= 32 ? off + i * RPI * step : row + key * step + c * es) : 0;
      const uint32_t d = dst + key * rowb + ((c ^ (key & 7)) << 4);
      cp16(d, kb + o, have);
      cp16(d + voff, vb + o, have);
    }
  } else {
    const long long row = row_at(p, first + lane, page, kvh);    // lanes < KEYS; -1 behind the end
#pragma unroll
    for (int i = 0; i < KEYS * CH / 32; ++i) {
      const int idx = i * 32 + lane, key = idx / CH, c = idx % CH;
      const long long off = __shfl_sync(0xffffffffu, row, key);
      const bool have = off >= 0 && c < chs;
      const long long o = have ? off + c * es : 0;
      const uint32_t d = dst + key * rowb + ((c ^ (key & 7)) << 4);
      cp16(d, kb + o, have);
      cp16(d + voff, vb + o, have);
    }
  }
}

struct DecArgs {
  PagedProblem p;
  int rtiles;              // row tiles of the longest sequence
  int q_vec;               // pairs of q elements are aligned
  int whole;               // a page holds whole steps
  int late_wait;           // 1: runs beside the prefix kernel, whose end it awaits at its own end
  int pre;                 // without splits: slots of the prefix to add to each row, 0: none
};

// The values of a step from row r0 on, in shared memory at vs: those that are
// not finite become zeros.  By a warp; whether any did.
template <int KEYS, int CH, typename E>
static __device__ __noinline__ bool clean_step(uint8_t* vs, int r0, int rowb) {
  bool any = false;
  for (int i = max(r0, 0) * CH + (int)(threadIdx.x & 31); i < KEYS * CH; i += 32) {
    uint4* at = reinterpret_cast<uint4*>(vs + i / CH * rowb + i % CH * 16);
    uint4 u = *at;
    if (clean_piece<E>(u)) {
      *at = u;
      any = true;
    }
  }
  __syncwarp();
  return __any_sync(0xffffffffu, any);
}

// One row at the end of a CTA, by a warp: M, L its maximum (base 2) and sum,
// v[i] its sum at dim lane + 32 i.  A split's partial row, or the output row
// with the prefix's partial rows added to it.  [k0, k1): the CTA's keys; first:
// those before are seen by all its rows; dirty: of the others, values that are
// not finite were left out.  What the row sees of them goes into it here; and
// where a value met a weight of zero (rounded, or the low part of one), the
// NaN in v becomes the sum of such values.
__device__ __forceinline__ void finish_row(const DecArgs& a, const SeqTask& t, int kvh, int split, int r, float M, float L,
                                           float (&v)[8], int k0, int k1, int first, bool dirty) {
  const PagedProblem& p = a.p;
  const int lane = threadIdx.x & 31;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) nan |= lane + 32 * i < p.hd && isnan(v[i]);
  nan = __any_sync(0xffffffffu, nan && !isnan(L));
  if (nan || dirty) {
    float s[8];
    bad_values(p, t.table, kvh, nan ? k0 : max(k0, first), min(k1, seen(p, t, row_token(p, r))), s);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = nan && !(s[i] == 0.0f) ? s[i] : v[i] + s[i];
  }
  const int tok = t.q0 + row_token(p, r), head = kvh * p.group + row_head(p, r);
  const long long row = (long long)tok * p.heads + head, step = (long long)p.total_q * p.heads;
  if (p.splits) {
    const long long part = (p.slot0 + split) * step + row;
    if (lane == 0) p.part_ml[part] = make_float2(M, L);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.hd) p.part_o[part * p.hd + lane + 32 * i] = v[i];
    return;
  }
  for (int s0 = 0; s0 < a.pre; s0 += 32) {               // lane i: slot s0 + i
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (s0 + lane < a.pre) ml = p.part_ml[(s0 + lane) * step + row];
    float mx = ml.x;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(M, mx), base = mn == -INFINITY ? 0.0f : mn;
    const float f = exp2f(M - base), c = exp2f(ml.x - base);
    float l = ml.y * c;
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    M = mn;
    L = fmaf(L, f, l);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= f;
    const int m = min(32, a.pre - s0);
    for (int s = 0; s < m; s += 4) {
      float x[4][8];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[u][i] = s + u < m && lane + 32 * i < p.hd ? p.part_o[((s0 + s + u) * step + row) * p.hd + lane + 32 * i] : 0.0f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float cu = __shfl_sync(0xffffffffu, c, (s + u) & 31);
        if (s + u < m) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(x[u][i], cu, v[i]);
        }
      }
    }
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  const long long oo = (long long)tok * p.out_stride + (long long)head * p.hd;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (lane + 32 * i < p.hd) store_elem(p.out, p.type, oo + lane + 32 * i, L == 0.0f ? 0.0f : v[i] * inv);
}

// High and low part's sum.  Beside an infinite high part the low one counts
// for nothing: it may be zero, or of the other sign, times infinity.
__device__ __forceinline__ float parts_sum(float hi, float lo) { return isinf(hi) ? hi : hi + lo; }

// Whether this CTA's rows wait for the prefix kernel's: by all threads, once.
__device__ __forceinline__ void await_prefix(const DecArgs& a) {
  if (a.late_wait) {
    pdl_trigger();
    pdl_wait();
  }
}

template <int HD, int NQ, bool DEEP>
__global__ void __launch_bounds__(32 * kDecWarps) paged_decode_kernel(const __grid_constant__ DecArgs a) {
  using T = DecShape<HD, DEEP>;
  extern __shared__ __align__(128) uint8_t sm[];
  const PagedProblem& p = a.p;
  if (!a.late_wait) {
    pdl_wait();
    pdl_trigger();
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  int b = blockIdx.x;
  const int kvh = b % p.n_kv;
  b /= p.n_kv;
  const int splits = p.splits ? p.splits : 1, split = b % splits;
  b /= splits;
  const int seq = b % p.n_seqs, r0 = (a.rtiles - 1 - b / p.n_seqs) * 8 * NQ;   // long rows first
  const SeqTask t = seq_task(p, seq);
  const int nr = min(8 * NQ, t.qn * p.group - r0);                 // rows of this tile
  int k0 = 0, k1 = nr > 0 ? seen(p, t, row_token(p, r0 + nr - 1)) : 0;
  if (p.splits) {
    k0 = split * p.chunk;
    k1 = min(k1, k0 + p.chunk);
  }
  const int all = nr > 0 ? seen(p, t, row_token(p, r0)) : 0;       // keys that all rows see
  const int some = all < k1 ? all : 0x7fffffff;                    // the first that only some see, if any
  if (nr > 0 && (k0 < k1 || !p.splits)) {
    const int steps = (k1 - k0 + kStep - 1) / kStep;
    const uint32_t ring = smem_u32(sm) + warp * T::kDepth * T::kStage;
    const __half* kb = reinterpret_cast<const __half*>(p.k);
    const __half* vb = reinterpret_cast<const __half*>(p.v);
    constexpr int CH = HD / 8;                                   // 16-byte pieces of a row
    const int chs = p.hd / 8;
    // The page of a step (or, where pages are no multiple of a step, of key
    // `lane` of it).  The entry is not looked at until the step's copies are
    // issued, so that its load is not waited for a step ahead.
    auto fetch_page = [&](int st) {
      const int key = k0 + st * kStep + (a.whole ? 0 : lane & 15);
      return st < steps && key < k1 ? t.table[page_of(p, key)] : -1;
    };
    auto issue = [&](int st, int page) {
      if (st < steps) {
        const uint32_t dst = ring + (st / kDecWarps % T::kDepth) * T::kStage;
        const int first = k0 + st * kStep;
        copy_step<kStep, CH>(p, a.whole, first, k1, page, kvh, chs, 8, dst, kStep * T::kRow, T::kRow, kb, vb);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the ring's first stages, then the queries while they fly
    int pages[T::kDepth];
#pragma unroll
    for (int d = 0; d < T::kDepth; ++d) pages[d] = fetch_page(warp + d * kDecWarps);
#pragma unroll
    for (int d = 0; d < T::kDepth - 1; ++d) issue(warp + d * kDecWarps, pages[d]);
    int npage = pages[T::kDepth - 1];

    uint32_t qa[NQ][HD / 16][4];
    float sc[NQ], m[NQ], l[NQ];
    float2 o[NQ][HD / 8];
    int lim[NQ];                                                  // keys that this lane's row sees
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int r = n * 8 + g, row = r0 + (r < nr ? r : 0);       // this lane's row
      const bool live = r < nr;
      lim[n] = live ? min(k1, seen(p, t, row_token(p, row))) : 0;
      const long long qo = (long long)(t.q0 + row_token(p, row)) * p.q_stride +
                           (long long)(kvh * p.group + row_head(p, row)) * p.hd;
      float x[HD / 16][4];
      float mx = 0.0f;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const int d = 16 * k + 2 * t4 + 8 * (e >> 1);           // hd is a multiple of 8
          float2 f = make_float2(0.0f, 0.0f);
          if (live && d < p.hd) {
            if (!a.q_vec) f = make_float2(load_elem(p.q, p.type, qo + d), load_elem(p.q, p.type, qo + d + 1));
            else if (p.type == TOSK_F32) f = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p.q) + qo + d);
            else f = __half22float2(*reinterpret_cast<const __half2*>(reinterpret_cast<const __half*>(p.q) + qo + d));
          }
          x[k][e] = f.x;
          x[k][e + 1] = f.y;
          mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float s2 = pow2_to_2p13(mx);                          // exact scaling of the row
      const float sg = p.scale_log2 < 0.0f ? -s2 : s2;
      sc[n] = fmaxf(fabsf(p.scale_log2) * pow2_inverse(s2), 1.2e-38f);  // not 0: a masked score is -inf * sc
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        split_pair(x[k][0] * sg, x[k][1] * sg, qa[n][k][0], qa[n][k][1]);
        split_pair(x[k][2] * sg, x[k][3] * sg, qa[n][k][2], qa[n][k][3]);
      }
      m[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) o[n][d] = make_float2(0.0f, 0.0f);
    }
    // ldmatrix row addresses: K: lanes 0-7 / 8-15 keys 0-7 at the two halves
    // of 16 dims, 16-31 keys 8-15; V (transposed): 0-15 keys, 16-31 the next 8 dims
    const int krow = (lane & 7) + ((lane >> 4) << 3), kch = (lane >> 3) & 1;
    const int vrow = lane & 15, vch = lane >> 4;
    bool dirty = false;

    for (int st = warp; st < steps; st += kDecWarps) {
      issue(st + (T::kDepth - 1) * kDecWarps, npage);
      npage = fetch_page(st + T::kDepth * kDecWarps);
      asm volatile("cp.async.wait_group %0;" ::"n"(T::kDepth - 1) : "memory");
      __syncwarp();
      const uint32_t kbase = ring + (st / kDecWarps % T::kDepth) * T::kStage, vbase = kbase + kStep * T::kRow;
      if (k0 + (st + 1) * kStep > some)                           // a prompt's last steps
        dirty |= clean_step<kStep, CH, __half>(sm + (vbase - smem_u32(sm)), some - k0 - st * kStep, T::kRow);
      float s[NQ][2][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][c][e] = 0.0f;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        uint32_t bk[4];
        ldsm4(bk, kbase + krow * T::kRow + (((2 * k + kch) ^ (krow & 7)) << 4));
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          mma16816(s[n][0], qa[n][k], bk[0], bk[1]);
          mma16816(s[n][1], qa[n][k], bk[2], bk[3]);
        }
      }
      uint32_t pa[NQ][4];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const int left = lim[n] - (k0 + st * kStep);              // keys of the step that the row sees
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = (e >> 1) * 8 + 2 * t4 + (e & 1);
          w[e] = key < left ? parts_sum(s[n][e >> 1][e & 1], s[n][e >> 1][2 + (e & 1)]) * sc[n] : -INFINITY;
        }
        float top = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m[n] + 8.0f)) {
          const float mn = top > m[n] + 8.0f ? top : m[n];
          const float f = mn == m[n] ? 1.0f : exp2f(m[n] - mn);   // 0 on the first keys
          m[n] = mn;
          l[n] *= f;
#pragma unroll
          for (int d = 0; d < HD / 8; ++d) o[n][d] = __fmul2_rn(o[n][d], make_float2(f, f));
        }
        const float bias = 7.0f - (m[n] == -INFINITY ? 0.0f : m[n]);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = ex2(w[e] + bias);
        l[n] += (w[0] + w[1]) + (w[2] + w[3]);
        split_pair(w[0], w[1], pa[n][0], pa[n][1]);
        split_pair(w[2], w[3], pa[n][2], pa[n][3]);
      }
      // How many products are under way before the first is added.  One CTA an
      // SM (256 dims) has no other warps to hide them: 8 x 3000 keys 68.6 us,
      // 87.0 one by one; 16 rows, 8 tokens behind 300 keys, 22.5, 23.6.  At 8 rows
      // of 128 dims they cost: 16 sequences of 1 to 4096 keys 106.8, 93.8 one by one.
      constexpr int B = HD == 256 ? 4 : NQ;
#pragma unroll
      for (int d0 = 0; d0 < HD / 16; d0 += B) {
        float c[B][NQ][2][4];
#pragma unroll
        for (int x = 0; x < B; ++x) {
          uint32_t bv[4];
          ldsm4t(bv, vbase + vrow * T::kRow + (((2 * (d0 + x) + vch) ^ (vrow & 7)) << 4));
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma16816_zero(c[x][n][0], pa[n], bv[0], bv[1]);
            mma16816_zero(c[x][n][1], pa[n], bv[2], bv[3]);
          }
        }
#pragma unroll
        for (int x = 0; x < B; ++x)
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float(&t)[4] = c[x][n][e];
              float2& to = o[n][2 * (d0 + x) + e];
              to = __fadd2_rn(to, make_float2(parts_sum(t[0], t[2]), parts_sum(t[1], t[3])));
            }
      }
      __syncwarp();                                               // the stage may be filled again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                              // the rings are free: join the warps there
    float* so = reinterpret_cast<float*>(sm);                     // [warp][8 NQ queries][HD]
    __shared__ float2 sml[kDecWarps][8 * NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
      if (t4 == 0) sml[warp][n * 8 + g] = make_float2(m[n] - 7.0f, l[n]);
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
        *reinterpret_cast<float2*>(so + ((warp * NQ + n) * 8 + g) * HD + 8 * d + 2 * t4) = o[n][d];
    }
    dirty = __syncthreads_or(dirty);
    // a warp a query
    await_prefix(a);
    for (int r = warp; r < nr; r += kDecWarps) {
      float M = -INFINITY, L = 0.0f, f[kDecWarps], v[8];
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sml[w][r].x);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        f[w] = M == -INFINITY ? 0.0f : exp2f(sml[w][r].x - M);
        L += f[w] * sml[w][r].y;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        v[i] = 0.0f;
        if (d < HD) {
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) v[i] = fmaf(f[w], so[(w * NQ * 8 + r) * HD + d], v[i]);
        }
      }
      finish_row(a, t, kvh, split, r0 + r, M, L, v, k0, k1, all, dirty);
    }
  } else {
    await_prefix(a);
  }
}

// ---------------------------------------------------------------------------
// The same over an fp32 cache, in fp32 throughout (packed FMAs: the tensor
// cores have no fp32 product, and the bytes leave the FMA pipe room for 8
// query heads a K/V row: 4 FMAs a byte read against the ~5 that HBM lets by).
// A warp's step is 8 keys.  Scores: lane (key, quarter of the dims), the four
// quarters added by two shuffles; the weights go through shared memory; sums:
// a lane has the dims 4 lane .. (64 dims: half the keys too).
// ---------------------------------------------------------------------------
template <int HD, int Q>
struct Dec32Shape {
  static constexpr int kKeysStep = 8;
  static constexpr int kRow = HD * 4;
  static constexpr int kStage = 2 * kKeysStep * kRow;
  static constexpr int kDepth = HD == 64 ? 6 : 3;
  static constexpr int kRing = kDecWarps * kDepth * kStage;
  static constexpr int kSmem = kRing + Q * HD * 4 + kDecWarps * kKeysStep * Q * 4;
};

template <int HD, int Q>
__global__ void __launch_bounds__(32 * kDecWarps) paged_decode_f32_kernel(const __grid_constant__ DecArgs a) {
  using T = Dec32Shape<HD, Q>;
  constexpr int KS = T::kKeysStep, CH = HD / 4;                  // keys a step, 16-byte pieces of a row
  constexpr int KG = CH < 32 ? 2 : 1, NC = CH > 32 ? CH / 32 : 1; // key groups of the sums, pieces a lane
  extern __shared__ __align__(128) uint8_t sm[];
  const PagedProblem& p = a.p;
  if (!a.late_wait) {
    pdl_wait();
    pdl_trigger();
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int b = blockIdx.x;
  const int kvh = b % p.n_kv;
  b /= p.n_kv;
  const int splits = p.splits ? p.splits : 1, split = b % splits;
  b /= splits;
  const int seq = b % p.n_seqs, r0 = (a.rtiles - 1 - b / p.n_seqs) * Q;   // long rows first
  const SeqTask t = seq_task(p, seq);
  const int nr = min(Q, t.qn * p.group - r0);                 // rows of this tile
  int k0 = 0, k1 = nr > 0 ? seen(p, t, row_token(p, r0 + nr - 1)) : 0;
  if (p.splits) {
    k0 = split * p.chunk;
    k1 = min(k1, k0 + p.chunk);
  }
  const int all = nr > 0 ? seen(p, t, row_token(p, r0)) : 0;       // keys that all rows see
  const int some = all < k1 ? all : 0x7fffffff;                    // the first that only some see, if any
  if (nr > 0 && (k0 < k1 || !p.splits)) {
    const int steps = (k1 - k0 + KS - 1) / KS;
    const uint8_t* ringp = sm + warp * T::kDepth * T::kStage;
    const uint32_t ring = smem_u32(ringp);
    float* sq = reinterpret_cast<float*>(sm + T::kRing);                  // [Q][HD]
    float* sp = sq + Q * HD + warp * KS * Q;                              // [key][query]
    const float* kb = reinterpret_cast<const float*>(p.k);
    const float* vb = reinterpret_cast<const float*>(p.v);
    const int chs = p.hd / 4;
    auto fetch_page = [&](int st) {
      const int key = k0 + st * KS + (a.whole ? 0 : lane & 7);
      return st < steps && key < k1 ? t.table[page_of(p, key)] : -1;
    };
    auto issue = [&](int st, int page) {
      if (st < steps) {
        const uint32_t dst = ring + (st / kDecWarps % T::kDepth) * T::kStage;
        copy_step<KS, CH>(p, a.whole, k0 + st * KS, k1, page, kvh, chs, 4, dst, KS * T::kRow, T::kRow, kb, vb);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int pages[T::kDepth];
#pragma unroll
    for (int d = 0; d < T::kDepth; ++d) pages[d] = fetch_page(warp + d * kDecWarps);
#pragma unroll
    for (int d = 0; d < T::kDepth - 1; ++d) issue(warp + d * kDecWarps, pages[d]);
    int npage = pages[T::kDepth - 1];
    for (int i = tid; i < Q * HD; i += 32 * kDecWarps) {
      const int r = i / HD, d = i % HD;
      sq[i] = r < nr && d < p.hd ? load_elem(p.q, p.type, (long long)(t.q0 + row_token(p, r0 + r)) * p.q_stride +
                                                              (long long)(kvh * p.group + row_head(p, r0 + r)) * p.hd + d)
                                 : 0.0f;
    }
    __syncthreads();
    float m[Q], l[Q];
    int lim[Q];                                                   // keys that the rows see
    float2 o[Q][NC][2];
#pragma unroll
    for (int n = 0; n < Q; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.0f;
      lim[n] = n < nr ? min(k1, seen(p, t, row_token(p, r0 + n))) : 0;
#pragma unroll
      for (int c = 0; c < NC; ++c) o[n][c][0] = o[n][c][1] = make_float2(0.0f, 0.0f);
    }
    const int key = lane & 7, quarter = lane >> 3;
    bool dirty = false;
    for (int st = warp; st < steps; st += kDecWarps) {
      issue(st + (T::kDepth - 1) * kDecWarps, npage);
      npage = fetch_page(st + T::kDepth * kDecWarps);
      asm volatile("cp.async.wait_group %0;" ::"n"(T::kDepth - 1) : "memory");
      __syncwarp();
      const uint8_t* ks = ringp + (st / kDecWarps % T::kDepth) * T::kStage;
      const uint8_t* vs = ks + KS * T::kRow;
      if (k0 + (st + 1) * KS > some)                              // a prompt's last steps
        dirty |= clean_step<KS, CH, float>(sm + (vs - sm), some - k0 - st * KS, T::kRow);
      float2 s[Q];
#pragma unroll
      for (int n = 0; n < Q; ++n) s[n] = make_float2(0.0f, 0.0f);
#pragma unroll 4
      for (int i = 0; i < CH / 4; ++i) {
        const int c = quarter + 4 * i;
        const float4 kx = *reinterpret_cast<const float4*>(ks + key * T::kRow + ((c ^ key) << 4));
#pragma unroll
        for (int n = 0; n < Q; ++n) {
          const float4 qx = *reinterpret_cast<const float4*>(sq + n * HD + 4 * c);
          s[n] = __ffma2_rn(make_float2(qx.x, qx.y), make_float2(kx.x, kx.y), s[n]);
          s[n] = __ffma2_rn(make_float2(qx.z, qx.w), make_float2(kx.z, kx.w), s[n]);
        }
      }
      float x[Q];
      bool grown = false;
#pragma unroll
      for (int n = 0; n < Q; ++n) x[n] = s[n].x + s[n].y;
#pragma unroll
      for (int n = 0; n < Q; ++n) x[n] += __shfl_xor_sync(0xffffffffu, x[n], 8);
#pragma unroll
      for (int n = 0; n < Q; ++n) {
        x[n] += __shfl_xor_sync(0xffffffffu, x[n], 16);
        x[n] = k0 + st * KS + key < lim[n] ? x[n] * p.scale_log2 : -INFINITY;
        grown |= x[n] > m[n] + 8.0f;
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int n = 0; n < Q; ++n) {
          float top = x[n];
#pragma unroll
          for (int w = 4; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          const float mn = fmaxf(m[n], top), f = mn == m[n] ? 1.0f : exp2f(m[n] - mn);   // 0 on the first keys
          m[n] = mn;
          l[n] *= f;
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[n][c][e] = __fmul2_rn(o[n][c][e], make_float2(f, f));
        }
      }
#pragma unroll
      for (int n = 0; n < Q; ++n) {
        const float w = ex2(x[n] - (m[n] == -INFINITY ? 0.0f : m[n]));
        l[n] += w;
        if (quarter == (n & 3)) sp[key * Q + n] = w;
      }
      __syncwarp();
      // weights of keys behind the end are 0, their values zeros
#pragma unroll
      for (int kk = 0; kk < KS / KG; ++kk) {
        const int ky = kk * KG + (KG == 2 ? lane >> 4 : 0);
        float w[Q];
#pragma unroll
        for (int n = 0; n < Q; ++n) w[n] = sp[ky * Q + n];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int pc = (KG == 2 ? lane & 15 : lane) + 32 * c;
          const float4 vx = *reinterpret_cast<const float4*>(vs + ky * T::kRow + ((pc ^ (ky & 7)) << 4));
#pragma unroll
          for (int n = 0; n < Q; ++n) {
            o[n][c][0] = __ffma2_rn(make_float2(w[n], w[n]), make_float2(vx.x, vx.y), o[n][c][0]);
            o[n][c][1] = __ffma2_rn(make_float2(w[n], w[n]), make_float2(vx.z, vx.w), o[n][c][1]);
          }
        }
      }
      __syncwarp();                                               // the stage and the weights may be written again
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                              // the rings are free: join the warps there
    float* so = reinterpret_cast<float*>(sm);                     // [warp][query][HD]
    __shared__ float2 sml[kDecWarps][Q];
#pragma unroll
    for (int n = 0; n < Q; ++n) {
#pragma unroll
      for (int w = 4; w > 0; w >>= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], w);
      if (lane == 0) sml[warp][n] = make_float2(m[n], l[n]);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float2 x = o[n][c][0], y = o[n][c][1];
        if (KG == 2) {
          x.x += __shfl_xor_sync(0xffffffffu, x.x, 16); x.y += __shfl_xor_sync(0xffffffffu, x.y, 16);
          y.x += __shfl_xor_sync(0xffffffffu, y.x, 16); y.y += __shfl_xor_sync(0xffffffffu, y.y, 16);
        }
        const int pc = (KG == 2 ? lane & 15 : lane) + 32 * c;
        if (KG == 1 || lane < 16)
          *reinterpret_cast<float4*>(so + (warp * Q + n) * HD + 4 * pc) = make_float4(x.x, x.y, y.x, y.y);
      }
    }
    dirty = __syncthreads_or(dirty);
    await_prefix(a);
    for (int r = warp; r < nr; r += kDecWarps) {
      float M = -INFINITY, L = 0.0f, f[kDecWarps], v[8];
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, sml[w][r].x);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        f[w] = M == -INFINITY ? 0.0f : exp2f(sml[w][r].x - M);
        L += f[w] * sml[w][r].y;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        v[i] = 0.0f;
        if (d < HD) {
#pragma unroll
          for (int w = 0; w < kDecWarps; ++w) v[i] = fmaf(f[w], so[(w * Q + r) * HD + d], v[i]);
        }
      }
      finish_row(a, t, kvh, split, r0 + r, M, L, v, k0, k1, all, dirty);
    }
  } else {
    await_prefix(a);
  }
}

}  // namespace tos

using namespace tos;

namespace {
int dec_launch(const void* f, int smem, const DecArgs& a, unsigned grid, cudaStream_t st) {
  const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(32 * kDecWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<DecArgs*>(&a)};
  return (int)cudaLaunchKernelExC(&cfg, f, args);
}

template <int HD, bool DEEP>
int dec16(const DecArgs& a, int nq, unsigned n, cudaStream_t st) {
  if constexpr (HD <= 128)
    if (nq == 2) return dec_launch((const void*)paged_decode_kernel<HD, 2, DEEP>, DecShape<HD, DEEP>::kSmem, a, n, st);
  return dec_launch((const void*)paged_decode_kernel<HD, 1, DEEP>, DecShape<HD, DEEP>::kSmem, a, n, st);
}

template <int HD>
int dec32(const DecArgs& a, int q, unsigned n, cudaStream_t st) {
  if (q == 1) return dec_launch((const void*)paged_decode_f32_kernel<HD, 1>, Dec32Shape<HD, 1>::kSmem, a, n, st);
  if (q == 4) return dec_launch((const void*)paged_decode_f32_kernel<HD, 4>, Dec32Shape<HD, 4>::kSmem, a, n, st);
  return dec_launch((const void*)paged_decode_f32_kernel<HD, 8>, Dec32Shape<HD, 8>::kSmem, a, n, st);
}
}  // namespace

namespace tos {

// What these kernels take: a cache whose rows are whole 16-byte pieces.
bool paged_decode_ok(const PagedProblem& p) {
  return p.hd % (p.kv_type == TOSK_F16 ? 8 : 4) == 0 && ((uintptr_t)p.k & 15) == 0 && ((uintptr_t)p.v & 15) == 0;
}

// Few rows a sequence (single tokens, short prompts).  fp16: row tiles of 16
// where a sequence has more than 8 rows (256 dims: of 8, for the registers),
// else of 8.  fp32: of 1, 4 or 8, the smallest that holds the rows.
int paged_decode_run(const PagedProblem& p, int pre_slots, cudaStream_t st) {
  DecArgs a;
  a.p = p;
  a.late_wait = pre_slots > 0;
  a.pre = p.splits ? 0 : pre_slots;
  const bool f16 = p.kv_type == TOSK_F16;
  const long long rows = (long long)p.max_q * p.group;
  const int nq = rows > 8 && p.hd <= 128 ? 2 : 1;
  const int block = f16 ? 8 * nq : rows == 1 ? 1 : rows <= 4 ? 4 : 8;
  const long long rt = (rows + block - 1) / block;
  const long long grid = rt * p.n_kv * (p.splits ? p.splits : 1) * p.n_seqs;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  a.rtiles = (int)rt;
  a.whole = p.page_size % (f16 ? kStep : 8) == 0;
  a.q_vec = ((uintptr_t)p.q & (p.type == TOSK_F32 ? 7 : 3)) == 0 && p.q_stride % 2 == 0;
  const unsigned n = (unsigned)grid;
  const bool deep = (p.splits ? p.chunk : p.max_kv) > 1024;
  if (f16 && p.hd <= 64) return deep ? dec16<64, true>(a, nq, n, st) : dec16<64, false>(a, nq, n, st);
  if (f16 && p.hd <= 128) return deep ? dec16<128, true>(a, nq, n, st) : dec16<128, false>(a, nq, n, st);
  if (f16) return dec16<256, true>(a, nq, n, st);
  return p.hd <= 64 ? dec32<64>(a, block, n, st) : p.hd <= 128 ? dec32<128>(a, block, n, st) : dec32<256>(a, block, n, st);
}

}  // namespace tos
