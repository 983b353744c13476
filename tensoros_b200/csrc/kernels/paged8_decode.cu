// paged8_decode.cu - attention of one token a sequence over an 8-bit paged
// cache.
//
//   s_j = c 2^a(j) (q . k_j),  w_j = 2^(s_j - m),  o = sum_j w_j (2^b(j) v_j) / sum_j w_j
//
// with k_j, v_j as stored and 2^a, 2^b the scales of key j's block.  A CTA takes
// a chunk of one sequence's keys for one key/value head and 8 or 16 query heads
// of its group; its four warps take every fourth 16-key step each and run alone
// until the end.  A step's K and V rows and their 32 scales stream through the
// warp's own ring in shared memory (cp.async, 16-byte pieces).
//
// The stored bytes become fp16 in registers, exactly, on the way to mma.sync
// m16n8k16 (two-part queries and weights as rows 0-7 and 8-15: fp32 accuracy at
// no further instruction).  The fragments are loaded in an order that suits
// bytes, not ldmatrix: the contraction may run over the dims, and the columns
// over them, in any order that both sides keep.
//   S: a lane (g, t) reads 16 dims of key g at once; four neighbouring bytes are
//      its two half2 of one product, so dims 64 i + 16 t + 4 w + (0..3) are
//      "rows" 2t, 2t+1, 2t+8, 2t+9 of product 4 i + w, and q is loaded likewise.
//   P V: lane (g, t) reads 16 dims (16 g ..) of its four keys 2t, 2t+1, 2t+8,
//      2t+9; bytes of two keys are paired by prmt.  Product j has dims 16 g + j
//      as its columns.
// K's scale multiplies the score in fp32; V's, a power of two, goes into the
// conversion (I8: one fma takes off the offset and scales; F8: one product), so
// V stays exact in fp16.  Sums over the steps are fp32 registers.
//
// Bound: HBM, with the conversions close behind.
#include <cuda_runtime.h>
#include <string.h>

#include <type_traits>

#include "paged8.cuh"
#include "paged_tc.cuh"

namespace tos {

constexpr int kD8Warps = 4;
constexpr int kD8Step = 16;                                      // keys a warp step

struct Dec8Args {
  PagedProblem p;
  Pool8 c;
  int rtiles;                                                     // row tiles of a group
  int q_vec;                                                      // four q elements are aligned
  int whole;                                                      // a page holds whole steps
};

template <int HD>
struct Dec8Shape {
  static constexpr int kTile = kD8Step * HD;                      // bytes of a step's K, of its V
  static constexpr int kScales = 2 * kTile;                       // then 16 scales of K, 16 of V
  static constexpr int kStage = 2 * kTile + 128;
  static constexpr int kDepth = HD == 64 ? 6 : HD == 128 ? 4 : 3;
  static constexpr int kSmem = kD8Warps * kDepth * kStage;
};

// Byte offset of piece c (16 bytes) of key r in a step's K and V, so that a
// quarter warp's reads lie in different banks: of K, 4 pieces of two keys; of V,
// 2 pieces of four keys 2t (64 dims: two keys a 128-byte line).
template <int HD>
__device__ __forceinline__ uint32_t k_off(int r, int c) {
  return (uint32_t)(HD == 64 ? r * 64 + c * 16 : r * HD + ((c ^ ((r & 1) << 2)) << 4));
}
template <int HD>
__device__ __forceinline__ uint32_t v_off(int r, int c) {
  const int x = ((r >> 1) & 3) << 1;
  return (uint32_t)(HD == 64 ? (r >> 1) * 128 + (((((r & 1) << 2) | c) ^ x) << 4) : r * HD + ((c ^ x) << 4));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool have) {
  const int n = have ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool have) {
  const int n = have ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void mma_h(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_h_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <int N>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  }
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// The four half2 (x: key a's element, y: key b's) of four dims, scaled by mul.
// I8: add is -1152 times the scales, or with BIG, where a scale makes that no
// fp16 number, -1152.
template <int TYPE, bool BIG>
__device__ __forceinline__ void pair_keys(uint32_t a, uint32_t b, __half2 mul, __half2 add, uint32_t (&h)[4]) {
  if constexpr (TYPE == TOSK_I8) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    const uint32_t lo = prmt(a, b, 0x5140u), hi = prmt(a, b, 0x7362u);   // {a0 b0 a1 b1}, {a2 b2 a3 b3}
    const uint32_t m = 0x64646464u;
    h[0] = prmt(lo, m, 0x4140u);
    h[1] = prmt(lo, m, 0x4342u);
    h[2] = prmt(hi, m, 0x4140u);
    h[3] = prmt(hi, m, 0x4342u);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = as_u32(BIG ? __hmul2(__hadd2(as_h2(h[i]), add), mul) : __hfma2(as_h2(h[i]), mul, add));
  } else {
    cvt_word<TYPE>(prmt(a, b, 0x5140u), h[0], h[1]);
    cvt_word<TYPE>(prmt(a, b, 0x7362u), h[2], h[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = as_u32(__hmul2(as_h2(h[i]), mul));
  }
}

template <int HD, int NQ, int TYPE>
__global__ void __launch_bounds__(32 * kD8Warps) paged8_decode_kernel(const __grid_constant__ Dec8Args a) {
  using T = Dec8Shape<HD>;
  extern __shared__ __align__(128) uint8_t sm[];
  const PagedProblem& p = a.p;
  const Pool8& c = a.c;
  pdl_wait();
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  int b = blockIdx.x;
  const int kvh = b % p.n_kv;
  b /= p.n_kv;
  const int splits = p.splits ? p.splits : 1, split = b % splits;
  b /= splits;
  const int seq = b % p.n_seqs, r0 = b / p.n_seqs * 8 * NQ;
  const int nr = min(8 * NQ, p.group - r0);                       // query heads of this tile
  int k0 = 0, k1 = (int)max(0ll, min((long long)min(p.kv_len[seq], p.max_kv), (long long)c.table_stride * c.page_size));
  if (p.splits) {
    k0 = split * p.chunk;
    k1 = min(k1, k0 + p.chunk);
    if (k0 >= k1) return;                                         // the joining kernel does not look there
  }
  const int steps = (k1 - k0 + kD8Step - 1) / kD8Step;
  const int* table = c.table + (long long)seq * c.table_stride;
  uint8_t* ringp = sm + warp * T::kDepth * T::kStage;
  const uint32_t ring = smem_u32(ringp);
  constexpr int CH = HD / 16;                                     // 16-byte pieces of a row
  const int chs = c.hd / 16;
  auto fetch_page = [&](int st) {
    const int key = k0 + st * kD8Step + (a.whole ? 0 : lane & 15);
    return st < steps && key < k1 ? table[page_index(c, key)] : -1;
  };
  // lane i, i + 16: key i's row; the scales go first, lane i of K, 16 + i of V
  auto issue = [&](int st, int page) {
    if (st < steps) {
      const uint32_t dst = ring + (st / kD8Warps % T::kDepth) * T::kStage;
      const int first = k0 + st * kD8Step, mine = first + (lane & 15);
      const Row8 row = row8(c, mine, page);
      const bool there = row.at >= 0 && mine < k1;
      const float* sc = lane < 16 ? c.ks : c.vs;
      cp_async4(dst + T::kScales + lane * 4, there ? sc + row.scale + kvh : sc, there);
      const long long off = there ? row.at + (long long)kvh * c.hd : -1;
#pragma unroll
      for (int i = 0; i < kD8Step * CH / 32; ++i) {
        const int idx = i * 32 + lane, key = idx / CH, pc = idx % CH;
        const long long o = __shfl_sync(0xffffffffu, off, key);
        const bool have = o >= 0 && pc < chs;
        cp_async16(dst + k_off<HD>(key, pc), have ? c.k + o + pc * 16 : c.k, have);
        cp_async16(dst + T::kTile + v_off<HD>(key, pc), have ? c.v + o + pc * 16 : c.v, have);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int pages[T::kDepth];
#pragma unroll
  for (int d = 0; d < T::kDepth; ++d) pages[d] = fetch_page(warp + d * kD8Warps);
#pragma unroll
  for (int d = 0; d < T::kDepth - 1; ++d) issue(warp + d * kD8Warps, pages[d]);
  int npage = pages[T::kDepth - 1];

  // the queries while they fly
  uint32_t qa[NQ][HD / 16][4];
  float sc[NQ], m[NQ], l[NQ];
  float2 o[NQ][HD / 8];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = n * 8 + g;
    const bool liv = r < nr;
    const long long qo = (long long)seq * p.q_stride + (long long)(kvh * p.group + r0 + (liv ? r : 0)) * c.hd;
    float x[HD / 16][4];
    float mx = 0.0f;
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
      const int d = 64 * (s >> 2) + 16 * t4 + 4 * (s & 3);        // hd is a multiple of 16
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (liv && d < c.hd) {
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
      x[s][0] = f.x; x[s][1] = f.y; x[s][2] = f.z; x[s][3] = f.w;
      mx = fmaxf(mx, fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w))));
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float s2 = pow2_to_2p13(mx);                            // exact scaling of the row
    const float sg = p.scale_log2 < 0.0f ? -s2 : s2;
    sc[n] = fabsf(p.scale_log2) * pow2_inverse(s2);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s) {
      split_pair(x[s][0] * sg, x[s][1] * sg, qa[n][s][0], qa[n][s][1]);
      split_pair(x[s][2] * sg, x[s][3] * sg, qa[n][s][2], qa[n][s][3]);
    }
    m[n] = -INFINITY;
    l[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) o[n][d] = make_float2(0.0f, 0.0f);
  }

  for (int st = warp; st < steps; st += kD8Warps) {
    issue(st + (T::kDepth - 1) * kD8Warps, npage);
    npage = fetch_page(st + T::kDepth * kD8Warps);
    asm volatile("cp.async.wait_group %0;" ::"n"(T::kDepth - 1) : "memory");
    __syncwarp();
    const uint8_t* kt = ringp + (st / kD8Warps % T::kDepth) * T::kStage;
    const uint8_t* vt = kt + T::kTile;
    const float* scales = reinterpret_cast<const float*>(kt + T::kScales);
    float s[NQ][2][4];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][x][e] = 0.0f;
#pragma unroll
    for (int i = 0; i < HD / 64; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t w[4];
        lds<4>(kt + k_off<HD>(8 * x + g, 4 * i + t4), w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t b0, b1;
          cvt_word<TYPE>(w[j], b0, b1);
#pragma unroll
          for (int n = 0; n < NQ; ++n) mma_h(s[n][x], qa[n][4 * i + j], b0, b1);
        }
      }
    const float2 ka = *reinterpret_cast<const float2*>(scales + 2 * t4), kb = *reinterpret_cast<const float2*>(scales + 8 + 2 * t4);
    const float ks[4] = {ka.x, ka.y, kb.x, kb.y};
    uint32_t pa[NQ][4];
    const int left = k1 - (k0 + st * kD8Step);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = (e >> 1) * 8 + 2 * t4 + (e & 1);
        w[e] = key < left ? (s[n][e >> 1][e & 1] + s[n][e >> 1][2 + (e & 1)]) * (ks[e] * sc[n]) : -INFINITY;
      }
      float top = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
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
      for (int e = 0; e < 4; ++e) w[e] = ex2(w[e] + bias);
      l[n] += (w[0] + w[1]) + (w[2] + w[3]);
      split_pair(w[0], w[1], pa[n][0], pa[n][1]);
      split_pair(w[2], w[3], pa[n][2], pa[n][3]);
    }
    const float2 va = *reinterpret_cast<const float2*>(scales + 16 + 2 * t4), vb = *reinterpret_cast<const float2*>(scales + 24 + 2 * t4);
    const __half2 mula = __floats2half2_rn(va.x, va.y), mulb = __floats2half2_rn(vb.x, vb.y);
    constexpr int VW = HD == 64 ? 2 : 4, VP = HD == 256 ? 2 : 1;  // words a key, pieces of them
    auto add_values = [&](auto big, __half2 adda, __half2 addb) {
#pragma unroll
      for (int x = 0; x < VP; ++x) {
        uint32_t w[4][VW];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = (e >> 1) * 8 + 2 * t4 + (e & 1);
          lds<VW>(HD == 64 ? vt + v_off<HD>(key, g >> 1) + (g & 1) * 8 : vt + v_off<HD>(key, g + 8 * x), w[e]);
        }
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          uint32_t b0[4], b1[4];
          pair_keys<TYPE, decltype(big)::value>(w[0][j], w[1][j], mula, adda, b0);
          pair_keys<TYPE, decltype(big)::value>(w[2][j], w[3][j], mulb, addb, b1);
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              float y[4];
              mma_h_zero(y, pa[n], b0[d], b1[d]);
              float2& to = o[n][x * 16 + 4 * j + d];
              to = __fadd2_rn(to, make_float2(y[0], y[1]));
              to = __fadd2_rn(to, make_float2(y[2], y[3]));
            }
        }
      }
    };
    // I8: -1152 times a scale beyond 2^5 is no fp16 number
    const __half2 off = __float2half2_rn(-1152.0f);
    if (TYPE == TOSK_I8 && __any_sync(0xffffffffu, fmaxf(fmaxf(va.x, va.y), fmaxf(vb.x, vb.y)) > 32.0f))
      add_values(std::true_type{}, off, off);
    else
      add_values(std::false_type{}, __hmul2(off, mula), __hmul2(off, mulb));
    __syncwarp();                                                 // the stage may be filled again
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();                                                // the rings are free: join the warps there
  float* so = reinterpret_cast<float*>(sm);                       // [warp][8 NQ queries][HD]
  static_assert(T::kSmem >= kD8Warps * 8 * NQ * HD * 4, "the sums of the warps");
  __shared__ float2 sml[kD8Warps][8 * NQ];
  constexpr int DG = HD == 64 ? 8 : 16;                           // dims of a column
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
    if (t4 == 0) sml[warp][n * 8 + g] = make_float2(m[n] - 7.0f, l[n]);
    float* to = so + ((warp * NQ + n) * 8 + g) * HD;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      to[(d / DG) * 128 + 2 * t4 * DG + d % DG] = o[n][d].x;      // columns 2t and 2t + 1
      to[(d / DG) * 128 + (2 * t4 + 1) * DG + d % DG] = o[n][d].y;
    }
  }
  __syncthreads();
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
    const long long row = (long long)seq * p.heads + head, part = (long long)split * p.total_q * p.heads + row;
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (p.splits && lane == 0) p.part_ml[part] = make_float2(M, L);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int d = lane + 32 * i;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kD8Warps; ++w) v = fmaf(f[w], so[(w * NQ * 8 + r) * HD + d], v);
      if (d >= c.hd) continue;
      if (p.splits) p.part_o[part * c.hd + d] = v;
      else store_elem(p.out, p.type, (long long)seq * p.out_stride + (long long)head * c.hd + d, L == 0.0f ? 0.0f : v * inv);
    }
  }
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

template <int HD, int TYPE>
int dec8(const Dec8Args& a, int nq, unsigned n, cudaStream_t st) {
  if constexpr (HD <= 128)
    if (nq == 2) return dec8_launch((const void*)paged8_decode_kernel<HD, 2, TYPE>, Dec8Shape<HD>::kSmem, a, n, st);
  return dec8_launch((const void*)paged8_decode_kernel<HD, 1, TYPE>, Dec8Shape<HD>::kSmem, a, n, st);
}

// Splits of the keys (0: none) and their length: four CTAs an SM, at least 512
// keys each.
struct Plan8 {
  int splits, chunk;
};
Plan8 plan8(int n_seqs, int max_kv, int n_kv) {
  const long long tiles = (long long)n_seqs * n_kv, want = (4 * 148 + tiles - 1) / tiles, most = ((long long)max_kv + 511) / 512;
  const long long s = want < most ? want : most;
  if (s <= 1) return {0, max_kv};
  const int chunk = (int)((max_kv + s - 1) / s + 127) / 128 * 128, n = (max_kv + chunk - 1) / chunk;
  return n > 1 ? Plan8{n, chunk} : Plan8{0, max_kv};
}

// Rows that are no whole 16-byte pieces go the way over fp16 (below).
bool direct(int hd) { return hd % 16 == 0; }
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

extern "C" size_t tosk_paged8_decode_ws_bytes(int n_seqs, int max_kv, int n_heads, int n_kv, int hd) {
  if (direct(hd)) return paged_slots_bytes(plan8(n_seqs, max_kv, n_kv).splits, n_seqs, n_heads, hd);
  return tosk_paged8_wide_bytes(n_seqs, (long long)n_seqs * max_kv, max_kv, n_kv, hd) +
         up256(tosk_paged_decode_ws_bytes(n_seqs, max_kv, 0, n_heads, n_kv, hd));
}

extern "C" int tosk_paged8_decode(const tosk_paged_attn_t* t, const tosk_paged8_t* kv, cudaStream_t st) {
  tosk_paged_attn_t x = *t;
  if (!direct(kv->hd)) {
    const long long total = (long long)x.n_seqs * x.max_kv;
    const size_t wide = tosk_paged8_wide_bytes(x.n_seqs, total, x.max_kv, kv->n_kv, kv->hd);
    const int e = tosk_paged8_wide(kv, x.kv_len, x.n_seqs, total, x.max_kv, x.ws, &x.kv, &x.kv_len, st);
    if (e) return e;
    x.ws = reinterpret_cast<uint8_t*>(x.ws) + wide;
    x.ws_bytes -= wide;
    return tosk_paged_decode(&x, st);
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
  const Plan8 d = plan8(x.n_seqs, x.max_kv, kv->n_kv);
  a.p.splits = d.splits;
  a.p.chunk = d.chunk;
  paged_part_views(a.p, x.ws, d.splits);
  const int nq = a.p.group > 8 && kv->hd <= 128 ? 2 : 1;
  a.rtiles = (a.p.group + 8 * nq - 1) / (8 * nq);
  a.whole = kv->page_size % kD8Step == 0;
  a.q_vec = ((uintptr_t)x.q & (x.type == TOSK_F32 ? 15 : 7)) == 0 && x.q_stride % 4 == 0;
  const long long grid = (long long)a.rtiles * kv->n_kv * (d.splits ? d.splits : 1) * x.n_seqs;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  const unsigned n = (unsigned)grid;
  const bool i8 = kv->type == TOSK_I8;
  const int e = kv->hd <= 64    ? i8 ? dec8<64, TOSK_I8>(a, nq, n, st) : dec8<64, TOSK_F8>(a, nq, n, st)
                : kv->hd <= 128 ? i8 ? dec8<128, TOSK_I8>(a, nq, n, st) : dec8<128, TOSK_F8>(a, nq, n, st)
                                : i8 ? dec8<256, TOSK_I8>(a, nq, n, st) : dec8<256, TOSK_F8>(a, nq, n, st);
  return e || !d.splits ? e : paged_join(a.p, st);
}

extern "C" size_t tosk_paged8_prompt_ws_bytes(int n_seqs, int total_q, long long total_kv, int max_kv, int n_heads, int n_kv, int hd) {
  return tosk_paged8_wide_bytes(n_seqs, total_kv, max_kv, n_kv, hd) +
         up256(tosk_paged_prompt_ws_bytes(n_seqs, total_q, max_kv, n_heads, n_kv, hd));
}

extern "C" int tosk_paged8_prompt(const tosk_paged_attn_t* t, const tosk_paged8_t* kv, long long total_kv, cudaStream_t st) {
  tosk_paged_attn_t x = *t;
  const size_t wide = tosk_paged8_wide_bytes(x.n_seqs, total_kv, x.max_kv, kv->n_kv, kv->hd);
  const int e = tosk_paged8_wide(kv, x.kv_len, x.n_seqs, total_kv, x.max_kv, x.ws, &x.kv, &x.kv_len, st);
  if (e) return e;
  x.ws = reinterpret_cast<uint8_t*>(x.ws) + wide;
  x.ws_bytes -= wide;
  return tosk_paged_prompt(&x, st);
}
