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
// Layout.  A lane holds V neighbouring pairs of a head (V = 4: eight elements,
// 16- or 32-byte accesses; V = 1 where size, alignment or rot does not allow
// that), a group of 4..32 lanes one head, a warp 32 / group heads at a time
// and one token at all times, so sine and cosine are computed once and serve
// all the token's heads.  Few tokens: a token's heads are dealt to several
// warps.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "tos_dev.cuh"
#include "tos_kernels.h"

namespace tos {

constexpr int kRotWarps = 8;   // warps per CTA

template <int N>
__device__ __forceinline__ void load_f(const float* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(p + i);
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}
template <int N>
__device__ __forceinline__ void load_f(const __half* p, float (&v)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint2 t = *reinterpret_cast<const uint2*>(p + i);
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&t.x));
      const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&t.y));
      v[i] = a.x; v[i + 1] = a.y; v[i + 2] = b.x; v[i + 3] = b.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __half2float(p[i]);
  }
}
template <int N>
__device__ __forceinline__ void store_f(void* base, int type, long long off, const float (&v)[N]) {
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
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const __half2 a = __floats2half2_rn(v[i], v[i + 1]), b = __floats2half2_rn(v[i + 2], v[i + 3]);
        uint2 t;
        t.x = *reinterpret_cast<const uint32_t*>(&a);
        t.y = *reinterpret_cast<const uint32_t*>(&b);
        *reinterpret_cast<uint2*>(p + i) = t;
      }
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
  const tosk_rotary_args_t& a = p.a;
  const int lane = threadIdx.x & 31, sub = lane & (p.group - 1);
  const int per = 32 / p.group;                       // heads a warp takes at a time
  const long long w = (long long)blockIdx.x * kRotWarps + (threadIdx.x >> 5);
  const long long t = w / p.parts;
  const int part = (int)(w % p.parts);
  pdl_wait();
  pdl_trigger();
  if (t >= a.n_tokens) return;
  const int hd = a.hd, pairs = hd >> 1, rp = a.rot.turn ? a.rot.rot >> 1 : 0;

  // this lane's pairs: where their elements lie, and the turn of each
  int e0[NC], e1[NC];
  bool on[NC], turns[NC];
  float cs[NC][V], sn[NC][V], wq[NC][2 * V], wk[NC][2 * V];
  const long long pos = a.rot.turn ? (long long)a.pos[t] : 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * p.group + sub) * V;            // first pair
    on[c] = i < pairs;
    turns[c] = i < rp;
    const bool half = turns[c] && a.rot.half;
    e0[c] = half ? i : 2 * i;
    e1[c] = half ? i + rp : 2 * i + V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      cs[c][j] = 1.0f;
      sn[c][j] = 0.0f;
      if (turns[c]) {
        const unsigned long long f = a.rot.turn[i + j] * (unsigned long long)pos;
        float s, k;
        sincospif((float)(int)(f >> 32) * 4.656612873077393e-10f, &s, &k);   // 2^-31: half turns
        cs[c][j] = k * a.rot.mag;
        sn[c][j] = s * a.rot.mag;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      wq[c][j] = on[c] && a.q_norm ? a.q_norm[e0[c] + j] : 0.0f;
      wq[c][V + j] = on[c] && a.q_norm ? a.q_norm[e1[c] + j] : 0.0f;
      wk[c][j] = on[c] && a.k_norm ? a.k_norm[e0[c] + j] : 0.0f;
      wk[c][V + j] = on[c] && a.k_norm ? a.k_norm[e1[c] + j] : 0.0f;
    }
  }
  // the cache row of this token (append), -1: none
  long long crow = -1;
  if (a.append) {
    const int s = a.seq[t], r = a.slot[t];
    if (s >= 0 && s < a.kv.n_seqs && r >= 0 && r / a.kv.page_size < a.kv.table_stride) {
      const int pg = a.kv.table[(long long)s * a.kv.table_stride + r / a.kv.page_size];
      if (pg >= 0 && pg < a.kv.n_pages) crow = ((long long)pg * a.kv.page_size + r % a.kv.page_size) * a.n_kv;
    }
  }
  const float inv = 1.0f / (float)hd;
  for (int h0 = part * per; h0 < p.slots; h0 += p.parts * per) {
    const int h = h0 + lane / p.group;
    const bool have = h < p.slots;
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv;
    const int hh = is_q ? h : is_v ? h - a.n_heads - a.n_kv : h - a.n_heads;
    const tosk_rows_t& r = is_q ? a.q : is_v ? a.v : a.k;
    const TI* src = reinterpret_cast<const TI*>(r.src) + t * r.sstride + (long long)hh * hd;
    void* dst = r.dst;
    long long off = t * r.dstride + (long long)hh * hd;
    int dtype = r.dtype;
    bool write = have;
    if (a.append && !is_q) {
      dst = is_v ? a.kv.v : a.kv.k;
      off = (crow + hh) * hd;
      dtype = a.kv.type;
      write = have && crow >= 0;
    }
    float x[NC][V], y[NC][V];
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[c][j] = y[c][j] = 0.0f;
      if (have && on[c]) {
        if (V == 4 && e1[c] == e0[c] + V) {           // eight elements in a row
          float b[2 * V];
          load_f<2 * V>(src + e0[c], b);
#pragma unroll
          for (int j = 0; j < V; ++j) { x[c][j] = b[j]; y[c][j] = b[V + j]; }
        } else {
          load_f<V>(src + e0[c], x[c]);
          load_f<V>(src + e1[c], y[c]);
        }
      }
#pragma unroll
      for (int j = 0; j < V; ++j) ss = fmaf(x[c][j], x[c][j], fmaf(y[c][j], y[c][j], ss));
    }
    const bool norm = !is_v && (is_q ? a.q_norm != nullptr : a.k_norm != nullptr);
    float rs = 1.0f;
    if (a.q_norm || a.k_norm) {
      for (int o = p.group >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      rs = 1.0f / sqrtf(fmaf(ss, inv, a.eps));
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      if (norm) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[c][j] = x[c][j] * rs * (is_q ? wq[c][j] : wk[c][j]);
          y[c][j] = y[c][j] * rs * (is_q ? wq[c][V + j] : wk[c][V + j]);
        }
      }
      // the two halves of a lane's pairs: (x, y) when e1 is the partner's
      // place, else x then y hold 2V elements in a row, neighbours paired
      if (turns[c] && !is_v) {
        if (a.rot.half) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float u = x[c][j], v = y[c][j];
            x[c][j] = fmaf(u, cs[c][j], -(v * sn[c][j]));
            y[c][j] = fmaf(v, cs[c][j], u * sn[c][j]);
          }
        } else {
          float b[2 * V];
#pragma unroll
          for (int j = 0; j < V; ++j) { b[j] = x[c][j]; b[V + j] = y[c][j]; }
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float u = b[2 * j], v = b[2 * j + 1];
            b[2 * j] = fmaf(u, cs[c][j], -(v * sn[c][j]));
            b[2 * j + 1] = fmaf(v, cs[c][j], u * sn[c][j]);
          }
#pragma unroll
          for (int j = 0; j < V; ++j) { x[c][j] = b[j]; y[c][j] = b[V + j]; }
        }
      }
      if (write && on[c]) {
        store_f<V>(dst, dtype, off + e0[c], x[c]);
        store_f<V>(dst, dtype, off + e1[c], y[c]);
      }
    }
  }
}

}  // namespace tos

using namespace tos;

namespace {
bool fits(const void* p, long long stride, int type, int n) {
  const size_t b = (type == TOSK_F32 ? 4 : 2) * (size_t)n;
  return (reinterpret_cast<uintptr_t>(p) % (b < 16 ? b : 16)) == 0 && stride % n == 0;
}

template <typename TI>
int launch_rot(const RotParams& p, bool v4, unsigned grid, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(32 * kRotWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)(v4 ? cudaLaunchKernelEx(&cfg, rotary_rows_kernel<TI, 4, 1>, p)
                  : cudaLaunchKernelEx(&cfg, rotary_rows_kernel<TI, 1, 4>, p));
}
}  // namespace

extern "C" int tosk_rotary_rows(const tosk_rotary_args_t* a, cudaStream_t st) {
  RotParams p;
  p.a = *a;
  const int rot = a->rot.turn ? a->rot.rot : 0;
  // four pairs a lane: whole lanes rotate or do not, and every access is
  // aligned to its four elements
  bool v4 = a->hd % 8 == 0 && rot % 8 == 0;
  const tosk_rows_t* rows[3] = {&a->q, &a->k, &a->v};
  for (const tosk_rows_t* r : rows) {
    if (r->src) v4 = v4 && fits(r->src, r->sstride, r->stype, 4);
    if (r->dst) v4 = v4 && fits(r->dst, r->dstride, r->dtype, 4);
  }
  if (a->append) v4 = v4 && fits(a->kv.k, 4, a->kv.type, 4) && fits(a->kv.v, 4, a->kv.type, 4);
  const int lanes = (a->hd / 2 + 3) / 4;   // four pairs a lane, at once or (V = 1) in four rounds
  p.group = 4;
  while (p.group < lanes) p.group *= 2;
  p.slots = a->n_heads + a->n_kv * (a->append ? 2 : 1);
  // one warp a token once that fills the card's 148 SMs four CTAs deep; else
  // a token's heads go to as many warps as they make rounds
  const int per = 32 / p.group, rounds = (p.slots + per - 1) / per;
  const long long want = 148ll * 4 * kRotWarps;
  long long parts = (want + a->n_tokens - 1) / a->n_tokens;
  if (parts > rounds) parts = rounds;
  p.parts = (int)parts;
  const long long grid = ((long long)a->n_tokens * parts + kRotWarps - 1) / kRotWarps;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  const int stype = a->q.src ? a->q.stype : a->k.stype;
  return stype == TOSK_F32 ? launch_rot<float>(p, v4, (unsigned)grid, st) : launch_rot<__half>(p, v4, (unsigned)grid, st);
}
