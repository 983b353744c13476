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
// for fp32, 16-byte accesses; smaller where size, alignment or rot does not
// allow that), a group of lanes one head, a warp 32 / group heads at a time
// and one token at all times.  The warp computes the token's sines and cosines
// once, a pair a lane, into shared memory; they serve all its heads.  kBatch
// rounds of heads are loaded before the first is worked on, so a warp keeps
// 4 KB in flight; with one round at a time the long prompt ran at 2.5 TB/s.
// Few tokens: a token's heads are dealt to several warps.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tos_dev.cuh"
#include "tos_kernels.h"

namespace tos {

constexpr int kRotWarps = 8;   // warps per CTA
constexpr int kMaxPairs = 128; // of a head (head_dim <= 256)
constexpr int kBatch = 4;

// N consecutive elements as they lie, in 32-bit words (fp16, N odd: the last word half used)
template <typename T, int N>
struct Raw {
  static constexpr int kWords = (N * (int)sizeof(T) + 3) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (N * sizeof(T) == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N * sizeof(T) == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x; w[1] = v.y;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> (16 * (i & 1)))));
  }
};

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
  int parts;       // warps that share a token's heads
  int slots;       // heads of a token: q, k and (append) v
};

// V pairs a lane, NC rounds of group * V pairs a head
template <typename TI, int V, int NC>
__global__ void __launch_bounds__(32 * kRotWarps) rotary_rows_kernel(const RotParams p) {
  constexpr int B = NC == 1 ? kBatch : 1;
  const tosk_rotary_args_t& a = p.a;
  __shared__ float2 s_cs[kRotWarps][kMaxPairs];       // magnitude * (cos, sin) of the warp's token
  __shared__ __align__(16) float s_w[2][2 * kMaxPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (p.group - 1);
  const int per = 32 / p.group;                       // heads a warp takes at a time
  const long long w = (long long)blockIdx.x * kRotWarps + warp;
  const long long t = w / p.parts;
  const int part = (int)(w % p.parts);
  const int hd = a.hd, pairs = hd >> 1, rp = a.rot.turn ? a.rot.rot >> 1 : 0;
  pdl_wait();
  pdl_trigger();
  const bool work = t < a.n_tokens;
  long long crow = -1;                                // the cache row of this token (append), -1: none
  if (a.append && work) {
    const int s = a.seq[t], r = a.slot[t];
    if (s >= 0 && s < a.kv.n_seqs && r >= 0 && r / a.kv.page_size < a.kv.table_stride) {
      const int pg = a.kv.table[(long long)s * a.kv.table_stride + r / a.kv.page_size];
      if (pg >= 0 && pg < a.kv.n_pages) crow = ((long long)pg * a.kv.page_size + r % a.kv.page_size) * a.n_kv;
    }
  }
  if (rp && work) {
    const long long pos = a.pos[t];
    for (int i = lane; i < rp; i += 32) {
      const unsigned long long f = a.rot.turn[i] * (unsigned long long)pos;
      float s, c;
      sincospif((float)(int)(f >> 32) * 4.656612873077393e-10f, &s, &c);   // 2^-31: half turns
      s_cs[warp][i] = make_float2(c * a.rot.mag, s * a.rot.mag);
    }
  }
  const bool any_norm = a.q_norm || a.k_norm;
  if (any_norm) {
    for (int i = threadIdx.x; i < hd; i += 32 * kRotWarps) {
      s_w[0][i] = a.q_norm ? a.q_norm[i] : 0.0f;
      s_w[1][i] = a.k_norm ? a.k_norm[i] : 0.0f;
    }
    __syncthreads();
  }
  if (!work) return;
  __syncwarp();

  // this lane's pairs: where their elements lie, and whether they turn
  int e0[NC], e1[NC];
  bool on[NC], turns[NC];
  float2 cs[NC][V];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * p.group + sub) * V;            // first pair
    on[c] = i < pairs;
    turns[c] = i < rp;
    const bool half = turns[c] && a.rot.half;
    e0[c] = half ? i : 2 * i;
    e1[c] = half ? i + rp : 2 * i + V;
#pragma unroll
    for (int j = 0; j < V; ++j) cs[c][j] = turns[c] ? s_cs[warp][i + j] : make_float2(1.0f, 0.0f);
  }
  const float inv = 1.0f / (float)hd;
  const int stride = p.parts * per;
  for (int b0 = part * per; b0 < p.slots; b0 += B * stride) {
    Raw<TI, V> rx[B][NC], ry[B][NC];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      const int h = b0 + u * stride + lane / p.group;
      const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
      const int hh = is_q ? h : is_v ? h - a.n_heads - a.n_kv : h - a.n_heads;
      const void* base = is_q ? a.q.src : is_v ? a.v.src : a.k.src;
      const long long ss = is_q ? a.q.sstride : is_v ? a.v.sstride : a.k.sstride;
      const TI* src = reinterpret_cast<const TI*>(base) + t * ss + (long long)hh * hd;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        rx[u][c].zero();
        ry[u][c].zero();
        if (h < p.slots && on[c]) {
          rx[u][c].load(src + e0[c]);
          ry[u][c].load(src + e1[c]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (b0 + u * stride >= p.slots) break;
      const int h = b0 + u * stride + lane / p.group;
      const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
      const int hh = is_q ? h : is_v ? h - a.n_heads - a.n_kv : h - a.n_heads;
      void* dst = is_q ? a.q.dst : a.k.dst;
      long long off = t * (is_q ? a.q.dstride : a.k.dstride) + (long long)hh * hd;
      int dtype = is_q ? a.q.dtype : a.k.dtype;
      bool write = h < p.slots;
      if (a.append && !is_q) {
        dst = is_v ? a.kv.v : a.kv.k;
        off = (crow + hh) * hd;
        dtype = a.kv.type;
        write = write && crow >= 0;
      }
      const bool norm = !is_v && (is_q ? a.q_norm != nullptr : a.k_norm != nullptr);
      float rs = 1.0f;
      if (any_norm) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j)
            ss = fmaf(rx[u][c].get(j), rx[u][c].get(j), fmaf(ry[u][c].get(j), ry[u][c].get(j), ss));
        for (int o = p.group >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        rs = 1.0f / sqrtf(fmaf(ss, inv, a.eps));
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float x[V], y[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[j] = rx[u][c].get(j);
          y[j] = ry[u][c].get(j);
        }
        if (norm && on[c]) {
          const float* wt = s_w[is_q ? 0 : 1];
#pragma unroll
          for (int j = 0; j < V; ++j) {
            x[j] = x[j] * rs * wt[e0[c] + j];
            y[j] = y[j] * rs * wt[e1[c] + j];
          }
        }
        // (x, y) are the pairs themselves in the half layout; else x then y
        // hold 2V elements in a row, neighbours paired
        if (turns[c] && !is_v) {
          if (a.rot.half) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float g = x[j], k = y[j];
              x[j] = fmaf(g, cs[c][j].x, -(k * cs[c][j].y));
              y[j] = fmaf(k, cs[c][j].x, g * cs[c][j].y);
            }
          } else {
            float z[2 * V];
#pragma unroll
            for (int j = 0; j < V; ++j) { z[j] = x[j]; z[V + j] = y[j]; }
#pragma unroll
            for (int j = 0; j < V; ++j) {
              const float g = z[2 * j], k = z[2 * j + 1];
              z[2 * j] = fmaf(g, cs[c][j].x, -(k * cs[c][j].y));
              z[2 * j + 1] = fmaf(k, cs[c][j].x, g * cs[c][j].y);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) { x[j] = z[j]; y[j] = z[V + j]; }
          }
        }
        if (write && on[c]) {
          store_n<V>(dst, dtype, off + e0[c], x);
          store_n<V>(dst, dtype, off + e1[c], y);
        }
      }
    }
  }
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

int launch_rot(const void* f, const RotParams& p, unsigned grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
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
  const int lanes = v == 1 ? (a->hd / 2 + 3) / 4 : a->hd / 2 / v;    // V = 1 goes four rounds over a head
  p.group = 2;
  while (p.group < lanes) p.group *= 2;
  p.slots = a->n_heads + a->n_kv * (a->append ? 2 : 1);
  // one warp a token once that fills the card's 148 SMs three CTAs deep; else
  // a token's heads go to as many warps as they make rounds
  const int per = 32 / p.group, rounds = (p.slots + per - 1) / per;
  const long long want = 148ll * 3 * kRotWarps;
  long long parts = (want + a->n_tokens - 1) / a->n_tokens;
  if (parts > rounds) parts = rounds;
  p.parts = (int)parts;
  const long long grid = ((long long)a->n_tokens * parts + kRotWarps - 1) / kRotWarps;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  const void* f = f32 ? (v == 4 ? (const void*)rotary_rows_kernel<float, 4, 1> : (const void*)rotary_rows_kernel<float, 1, 4>)
                      : (v == 8   ? (const void*)rotary_rows_kernel<__half, 8, 1>
                         : v == 4 ? (const void*)rotary_rows_kernel<__half, 4, 1>
                                  : (const void*)rotary_rows_kernel<__half, 1, 4>);
  return launch_rot(f, p, (unsigned)grid, st);
}
