// paged_rotary.cu - per-head RMS norm and rotary positions of packed tokens
// in one pass, and the same on the way into a paged K/V cache.
//
// For every token t and head:  x <- x / sqrt(mean x^2 + eps) * w   (optional)
// and for every pair i < rot/2, (a, b) <- (a cos - b sin, b cos + a sin) at the
// angle pos[t] * theta_i.  The pass reads and writes each element once and
// computes ~8 flops on it, so HBM bounds it (launch latency at a few tokens).
//
// Angles.  theta_i comes as turns per position in units of 2^-64; the product
// with pos wraps modulo 2^64, i.e. whole turns drop out exactly, and its top
// 32 bits as a signed fraction of a turn go through sincospi.  The angle's
// error is the 24-bit rounding of a number in [-1, 1): below 2e-7 rad at any
// position (a product in fp32 would be off by pos * 6e-8).
//
// Layout.  A lane holds V neighbouring pairs of a head (V = 8 for fp16 and 4
// for fp32: 16-byte pieces), a group of lanes one head, a warp 32 / group heads
// at a time (a round) and one token at all times.  The warp computes the
// token's sines and cosines once, a pair a lane, into shared memory; they serve
// all its heads.  A lane's pieces come by cp.async into its own places in
// shared memory, kAhead rounds ahead, and only that lane reads them: the
// rounds in flight cost no registers, so 28 warps an SM keep ~100 KB coming
// (four rounds in registers left room for 16 warps: 23.8 us for the long
// prompt, 49 for the packed append).  Few tokens: a token's heads are dealt to
// several warps.  4099 tokens, 32 / 8 heads x 128, fp16, norm: 18.7 us, 4.5 TB/s
// (the long prompt); append of 8191 such tokens 40 us, 5.0 TB/s.  Where size, alignment or rot does not allow 16-byte pieces,
// a plain element-wise kernel.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tos_dev.cuh"
#include "tos_kernels.h"

namespace tos {

constexpr int kRotWarps = 4;   // warps per CTA
constexpr int kMaxPairs = 128; // of a head (head_dim <= 256)
constexpr int kAhead = 4;      // rounds in flight (3: 19.9 us for the long prompt, 6: 19.3, 4: 18.8)
constexpr int kRotDeep = 16;   // warps an SM before a token's heads are dealt to several (28: 20.5 us, 56: 21.2)

// N consecutive elements (8 or 16 bytes) from shared memory
template <int N>
__device__ __forceinline__ void take_n(const float* p, float (&v)[N]) {
  static_assert(N == 4, "16 bytes");
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
template <int N>
__device__ __forceinline__ void take_n(const __half* p, float (&v)[N]) {
  uint32_t w[N / 2];
  if constexpr (N == 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// products and sums of two elements at a time
template <int N>
__device__ __forceinline__ void mul_to(float (&a)[N], const float (&b)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 r = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
    a[i] = r.x;
    a[i + 1] = r.y;
  }
}
// (a, b) <- (a c - b s, b c + a s); ns = -s
template <int N>
__device__ __forceinline__ void turn(float (&a)[N], float (&b)[N], const float (&c)[N], const float (&ns)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 x = make_float2(a[i], a[i + 1]), y = make_float2(b[i], b[i + 1]);
    const float2 k = make_float2(c[i], c[i + 1]), z = make_float2(ns[i], ns[i + 1]);
    const float2 u = __ffma2_rn(x, k, __fmul2_rn(y, z));
    const float2 v = __fmul2_rn(x, z);
    const float2 m = __ffma2_rn(y, k, make_float2(-v.x, -v.y));
    a[i] = u.x; a[i + 1] = u.y;
    b[i] = m.x; b[i + 1] = m.y;
  }
}

template <int N>
__device__ __forceinline__ void store_n(void* base, int type, long long off, const float (&v)[N]) {
  if (type == TOSK_F32) {
    float* p = reinterpret_cast<float*>(base) + off;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = v[i];
    }
  } else {
    __half* p = reinterpret_cast<__half*>(base) + off;
    if constexpr (N % 4 == 0) {
      uint32_t u[N / 2];
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
      else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) p[i] = __float2half_rn(v[i]);
    }
  }
}

struct RotParams {
  tosk_rotary_args_t a;
  int group;       // lanes per head (a power of two)
  int parts;       // warps that share a token's heads (grid y)
};

// Angle of pair i at position pos: magnitude * (cos, sin).
__device__ __forceinline__ float2 pair_turn(const tosk_rotary_t& rot, int i, long long pos) {
  const unsigned long long f = rot.turn[i] * (unsigned long long)pos;
  float s, c;
  sincospif((float)(int)(f >> 32) * 4.656612873077393e-10f, &s, &c);   // 2^-31: half turns
  return make_float2(c * rot.mag, s * rot.mag);
}

// Element offset / head_dim of the row of the cache that token t goes to, -1: none.
__device__ __forceinline__ long long cache_row(const tosk_rotary_args_t& a, int s, int r) {
  if (s < 0 || s >= a.kv.n_seqs || r < 0 || r / a.kv.page_size >= a.kv.table_stride) return -1;
  const int pg = a.kv.table[(long long)s * a.kv.table_stride + r / a.kv.page_size];
  if (pg < 0 || pg >= a.kv.n_pages) return -1;
  return ((long long)pg * a.kv.page_size + r % a.kv.page_size) * a.n_kv;
}

// The plain kernel: a warp a head of a token, a lane every 32nd pair, element
// by element.
template <typename TI>
__global__ void __launch_bounds__(32 * kRotWarps) rotary_plain_kernel(const __grid_constant__ RotParams p) {
  const tosk_rotary_args_t& a = p.a;
  const int lane = threadIdx.x & 31, hd = a.hd, rp = a.rot.turn ? a.rot.rot >> 1 : 0;
  const long long t = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  const int total = a.n_heads + (a.append ? 2 : 1) * a.n_kv;
  for (int g = blockIdx.y * kRotWarps + (threadIdx.x >> 5); g < total; g += gridDim.y * kRotWarps) {   // head: q, k, v
    const int kind = g < a.n_heads ? 0 : g < a.n_heads + a.n_kv ? 1 : 2;
    const int h = g - (kind == 0 ? 0 : kind == 1 ? a.n_heads : a.n_heads + a.n_kv);
    const tosk_rows_t& r = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const TI* src = reinterpret_cast<const TI*>(r.src) + t * r.sstride + (long long)h * hd;
    const float* w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float x[4], y[4], ss = 0.0f;
    int e0[4], e1[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = lane + 32 * c;
      const bool half = i < rp && a.rot.half;
      e0[c] = half ? i : 2 * i;
      e1[c] = half ? i + rp : 2 * i + 1;
      x[c] = i < hd >> 1 ? (float)src[e0[c]] : 0.0f;
      y[c] = i < hd >> 1 ? (float)src[e1[c]] : 0.0f;
      ss = fmaf(x[c], x[c], fmaf(y[c], y[c], ss));
    }
    if (w) {
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float rs = rsqrtf(fmaf(ss, 1.0f / (float)hd, a.eps));
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < hd >> 1) {
          x[c] = x[c] * rs * w[e0[c]];
          y[c] = y[c] * rs * w[e1[c]];
        }
    }
    void* dst = r.dst;
    long long off = t * r.dstride + (long long)h * hd;
    int dtype = r.dtype;
    if (a.append && kind > 0) {
      const long long row = cache_row(a, a.seq[t], a.slot[t]);
      if (row < 0) continue;
      dst = kind == 1 ? a.kv.k : a.kv.v;
      off = (row + h) * hd;
      dtype = a.kv.type;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = lane + 32 * c;
      if (i >= hd >> 1) break;
      if (kind < 2 && i < rp) {
        const float2 z = pair_turn(a.rot, i, a.pos[t]);
        const float u = x[c], v = y[c];
        x[c] = fmaf(u, z.x, -(v * z.y));
        y[c] = fmaf(v, z.x, u * z.y);
      }
      const float o0[1] = {x[c]}, o1[1] = {y[c]};
      store_n<1>(dst, dtype, off + e0[c], o0);
      store_n<1>(dst, dtype, off + e1[c], o1);
    }
  }
}

__device__ __forceinline__ void cp_piece(uint32_t dst, const void* src, int bytes, bool have) {
  const int n = have ? bytes : 0;
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

// The streaming kernel: V pairs a lane, whole lanes turn or do not.
template <typename TI, int V>
__global__ void __launch_bounds__(32 * kRotWarps, 7) rotary_stream_kernel(const __grid_constant__ RotParams p) {
  constexpr int PB = V * (int)sizeof(TI);             // bytes of a piece
  const tosk_rotary_args_t& a = p.a;
  __shared__ __align__(16) uint8_t s_in[kRotWarps][kAhead][2][32 * PB];
  __shared__ __align__(16) float s_c[kRotWarps][kMaxPairs], s_s[kRotWarps][kMaxPairs];   // magnitude * cos, -sin
  __shared__ __align__(16) float s_w[2][2 * kMaxPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (p.group - 1);
  const int per = 32 / p.group, slot = lane / p.group;
  const long long t = (long long)blockIdx.x * kRotWarps + warp;
  const int hd = a.hd, rp = a.rot.turn ? a.rot.rot >> 1 : 0;
  pdl_wait();
  pdl_trigger();
  const bool work = t < a.n_tokens;
  // this lane's pairs: where their elements lie, and whether they turn
  const int i0 = sub * V;
  const bool on = i0 < hd >> 1, turns = i0 < rp, half = turns && a.rot.half;
  const int e0 = half ? i0 : 2 * i0, e1 = half ? i0 + rp : 2 * i0 + V;
  const int nq = (a.n_heads + per - 1) / per, nk = (a.n_kv + per - 1) / per;
  const int rounds = nq + (a.append ? 2 : 1) * nk;
  const uint32_t in = smem_u32(&s_in[warp][0][0][0]) + lane * PB;
  int at = 0;                                          // ring place of the next round to be asked for
  auto ask = [&](int r) {
    if (r < rounds && work) {
      const int kind = r < nq ? 0 : r < nq + nk ? 1 : 2;
      const int h = (r - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk)) * per + slot;
      const tosk_rows_t& x = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
      const bool have = on && h < (kind == 0 ? a.n_heads : a.n_kv);
      const TI* src = reinterpret_cast<const TI*>(x.src) + (have ? t * x.sstride + (long long)h * hd : 0);
      cp_piece(in + at * 64 * PB, src + (have ? e0 : 0), PB, have);
      cp_piece(in + at * 64 * PB + 32 * PB, src + (have ? e1 : 0), PB, have);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    at = at + 1 == kAhead ? 0 : at + 1;
  };
#pragma unroll
  for (int i = 0; i < kAhead - 1; ++i) ask(blockIdx.y + i * p.parts);
  const bool normed = a.q_norm || a.k_norm;
  if (normed)
    for (int i = threadIdx.x; i < hd; i += 32 * kRotWarps) {
      s_w[0][i] = a.q_norm ? a.q_norm[i] : 0.0f;
      s_w[1][i] = a.k_norm ? a.k_norm[i] : 0.0f;
    }
  long long crow = -1;                                 // the cache row of this token (append), -1: none
  if (work) {
    int s = -1, r = -1;
    if (a.append) {
      s = a.seq[t];
      r = a.slot[t];
    }
    if (rp) {
      const long long pos = a.pos[t];
      for (int i = lane; i < rp; i += 32) {
        const float2 z = pair_turn(a.rot, i, pos);
        s_c[warp][i] = z.x;
        s_s[warp][i] = -z.y;
      }
    }
    if (a.append) crow = cache_row(a, s, r);
  }
  if (normed) __syncthreads();
  else __syncwarp();
  float c[V], ns[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    c[j] = turns ? s_c[warp][i0 + j] : 1.0f;
    ns[j] = turns ? s_s[warp][i0 + j] : 0.0f;
  }
  const float inv = 1.0f / (float)hd;
  int now = 0;
  for (int r = blockIdx.y; r < rounds; r += p.parts) {
    ask(r + (kAhead - 1) * p.parts);
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    float x[V], y[V];
    take_n<V>(reinterpret_cast<const TI*>(&s_in[warp][now][0][lane * PB]), x);
    take_n<V>(reinterpret_cast<const TI*>(&s_in[warp][now][1][lane * PB]), y);
    now = now + 1 == kAhead ? 0 : now + 1;
    const int kind = r < nq ? 0 : r < nq + nk ? 1 : 2;
    const int h = (r - (kind == 0 ? 0 : kind == 1 ? nq : nq + nk)) * per + slot;
    if (kind < 2 && (kind ? a.k_norm != nullptr : a.q_norm != nullptr)) {
      float ss = 0.0f, s1 = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss = fmaf(x[j], x[j], ss);
        s1 = fmaf(y[j], y[j], s1);
      }
      ss += s1;
      for (int o = p.group >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float rs = rsqrtf(fmaf(ss, inv, a.eps));
      if (on) {
        float w0[V], w1[V], rr[V];
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const float4 u = *reinterpret_cast<const float4*>(&s_w[kind][e0 + j]), v = *reinterpret_cast<const float4*>(&s_w[kind][e1 + j]);
          w0[j] = u.x; w0[j + 1] = u.y; w0[j + 2] = u.z; w0[j + 3] = u.w;
          w1[j] = v.x; w1[j + 1] = v.y; w1[j + 2] = v.z; w1[j + 3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) rr[j] = rs;
        mul_to(x, rr);
        mul_to(y, rr);
        mul_to(x, w0);
        mul_to(y, w1);
      }
    }
    if (kind < 2 && turns) {
      if (a.rot.half) {
        turn(x, y, c, ns);
      } else {
        // x then y hold 2V elements in a row, neighbours paired
        float g[V], k[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          g[j] = 2 * j < V ? x[2 * j % V] : y[2 * j % V];
          k[j] = 2 * j + 1 < V ? x[(2 * j + 1) % V] : y[(2 * j + 1) % V];
        }
        turn(g, k, c, ns);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = j & 1 ? k[j / 2] : g[j / 2];
          y[j] = (V + j) & 1 ? k[(V + j) / 2] : g[(V + j) / 2];
        }
      }
    }
    const bool cached = a.append && kind > 0;
    if (work && on && h < (kind == 0 ? a.n_heads : a.n_kv) && (!cached || crow >= 0)) {
      void* dst = kind == 0 ? a.q.dst : cached ? (kind == 1 ? a.kv.k : a.kv.v) : a.k.dst;
      const long long off = cached ? (crow + h) * hd : t * (kind == 0 ? a.q.dstride : a.k.dstride) + (long long)h * hd;
      const int dtype = kind == 0 ? a.q.dtype : cached ? a.kv.type : a.k.dtype;
      store_n<V>(dst, dtype, off + e0, x);
      store_n<V>(dst, dtype, off + e1, y);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace tos

using namespace tos;

namespace {
// n-element accesses at multiples of n elements are aligned (to 16 bytes at most)
bool fits(const void* p, long long stride, int type, int n) {
  const size_t b = (type == TOSK_F32 ? 4 : 2) * (size_t)n;
  return (reinterpret_cast<uintptr_t>(p) % (b < 16 ? b : 16)) == 0 && stride % n == 0;
}

bool takes(const tosk_rotary_args_t* a, int v) {
  const int rot = a->rot.turn ? a->rot.rot : 0;
  // whole lanes rotate or do not
  if (a->hd % (2 * v) || rot % (2 * v)) return false;
  const tosk_rows_t* rows[3] = {&a->q, &a->k, &a->v};
  for (const tosk_rows_t* r : rows) {
    if (r->src && !fits(r->src, r->sstride, r->stype, v)) return false;
    if (r->dst && !fits(r->dst, r->dstride, r->dtype, v)) return false;
  }
  return !a->append || (fits(a->kv.k, v, a->kv.type, v) && fits(a->kv.v, v, a->kv.type, v));
}

int launch_rot(const void* f, const RotParams& p, dim3 grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(32 * kRotWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<RotParams*>(&p)};
  return (int)cudaLaunchKernelExC(&cfg, f, args);
}
}  // namespace

extern "C" int tosk_rotary_rows(const tosk_rotary_args_t* a, cudaStream_t st) {
  RotParams p;
  p.a = *a;
  const bool f32 = (a->q.src ? a->q.stype : a->k.stype) == TOSK_F32;
  const int v = !f32 && takes(a, 8) ? 8 : takes(a, 4) ? 4 : 1;
  const int heads = a->n_heads + a->n_kv * (a->append ? 2 : 1);
  if (v == 1) {
    p.group = 32;
    p.parts = (heads + kRotWarps - 1) / kRotWarps;
    if (p.parts > 65535) p.parts = 65535;                // the grid's limit; warps go on to further heads
    return launch_rot(f32 ? (const void*)rotary_plain_kernel<float> : (const void*)rotary_plain_kernel<__half>, p,
                      dim3((unsigned)a->n_tokens, p.parts), st);
  }
  p.group = 2;
  while (p.group < a->hd / 2 / v) p.group *= 2;
  const int per = 32 / p.group;
  const int rounds = (a->n_heads + per - 1) / per + (a->n_kv + per - 1) / per * (a->append ? 2 : 1);
  // one warp a token once that fills the card's 148 SMs kRotDeep warps deep;
  // else a token's heads go to as many warps as they make rounds
  const long long want = 148ll * kRotDeep;
  long long parts = (want + a->n_tokens - 1) / a->n_tokens;
  if (parts > rounds) parts = rounds;
  p.parts = (int)parts;
  const unsigned gx = ((unsigned)a->n_tokens + kRotWarps - 1) / kRotWarps;
  const void* f = f32      ? (const void*)rotary_stream_kernel<float, 4>
                  : v == 8 ? (const void*)rotary_stream_kernel<__half, 8>
                           : (const void*)rotary_stream_kernel<__half, 4>;
  return launch_rot(f, p, dim3(gx, p.parts), st);
}
