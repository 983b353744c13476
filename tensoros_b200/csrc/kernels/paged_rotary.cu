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

constexpr int kRotWarps = 4;   // warps per CTA
constexpr int kMaxPairs = 128; // of a head (head_dim <= 256)
constexpr int kBatch = 4;     // rounds of heads in flight (2: 25.3 us for the long prompt, 46 for the append; 4: 23.8 and 49)
constexpr int kRotDeep = 16;  // warps an SM before a token's heads are dealt to several (32: 27.5 us, 8: as 16)

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
  __device__ __forceinline__ void get(float (&v)[N]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (N > 1) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else {
      v[0] = __half2float(__ushort_as_half((unsigned short)w[0]));
    }
  }
};

// products and sums of two elements at a time where there are two
template <int N>
__device__ __forceinline__ void mul_to(float (&a)[N], const float (&b)[N]) {
  if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 r = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
      a[i] = r.x;
      a[i + 1] = r.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] *= b[i];
  }
}
// (a, b) <- (a c - b s, b c + a s); ns = -s
template <int N>
__device__ __forceinline__ void turn(float (&a)[N], float (&b)[N], const float (&c)[N], const float (&ns)[N]) {
  if constexpr (N % 2 == 0) {
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
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float x = a[i], y = b[i];
      a[i] = fmaf(x, c[i], y * ns[i]);
      b[i] = fmaf(y, c[i], -(x * ns[i]));
    }
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
  int k_first, v_first;   // rounds before k's and v's, modulo parts
};

// A lane's pairs of a head: where their elements lie, whether they turn, and
// their magnitude * (cos, -sin).
template <int V, int NC>
struct Pairs {
  int e0[NC], e1[NC];
  bool on[NC], turns[NC];
  float c[NC][V], s[NC][V];
};

// The heads of one kind (q, k or v) of a token: `n` heads, head h at src + h *
// hd, to dst + off + h * hd elements.  The token's rounds (32 / group heads
// each) are numbered through q, k, v; this warp takes every parts-th one from
// `first` on.
// `ready` runs once the first loads are on their way: what the values need.
template <typename TI, int V, int NC, typename F>
__device__ __forceinline__ void do_heads(const RotParams& p, const Pairs<V, NC>& pr, const TI* src, int n, void* dst,
                                         long long off, int dtype, bool write, const float* wt, bool rotate,
                                         int first, F ready) {
  constexpr int B = NC == 1 ? kBatch : 1;
  const int lane = threadIdx.x & 31, per = 32 / p.group, hd = p.a.hd, step = p.parts * per;
  float w0[NC][V], w1[NC][V];
  bool begun = false;
  const float inv = 1.0f / (float)hd;
  int h = first * per + lane / p.group;                    // this lane's head
  src += (long long)h * hd;
  off += (long long)h * hd;
  const long long adv = (long long)step * hd;
  for (; h - lane / p.group < n; h += B * step, src += B * adv, off += B * adv) {
    Raw<TI, V> rx[B][NC], ry[B][NC];
#pragma unroll
    for (int u = 0; u < B; ++u)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        rx[u][c].zero();
        ry[u][c].zero();
        if (h + u * step < n && pr.on[c]) {
          rx[u][c].load(src + u * adv + pr.e0[c]);
          ry[u][c].load(src + u * adv + pr.e1[c]);
        }
      }
    if (!begun) {
      begun = true;
      ready();
      if (wt) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            w0[c][j] = pr.on[c] ? wt[pr.e0[c] + j] : 0.0f;
            w1[c][j] = pr.on[c] ? wt[pr.e1[c] + j] : 0.0f;
          }
      }
    }
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (h - lane / p.group + u * step >= n) break;
      float x[NC][V], y[NC][V];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        rx[u][c].get(x[c]);
        ry[u][c].get(y[c]);
      }
      if (wt) {
        float ss = 0.0f, s1 = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            ss = fmaf(x[c][j], x[c][j], ss);
            s1 = fmaf(y[c][j], y[c][j], s1);
          }
        ss += s1;
        for (int o = p.group >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rs = rsqrtf(fmaf(ss, inv, p.a.eps));
        float r[V];
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = rs;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          mul_to(x[c], r);
          mul_to(y[c], r);
          mul_to(x[c], w0[c]);
          mul_to(y[c], w1[c]);
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        // (x, y) are the pairs themselves in the half layout; else x then y
        // hold 2V elements in a row, neighbours paired
        if (rotate && pr.turns[c]) {
          if (p.a.rot.half) {
            turn(x[c], y[c], pr.c[c], pr.s[c]);
          } else {
            float g[V], k[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
              g[j] = 2 * j < V ? x[c][2 * j % V] : y[c][2 * j % V];
              k[j] = 2 * j + 1 < V ? x[c][(2 * j + 1) % V] : y[c][(2 * j + 1) % V];
            }
            turn(g, k, pr.c[c], pr.s[c]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              x[c][j] = j & 1 ? k[j / 2] : g[j / 2];
              y[c][j] = (V + j) & 1 ? k[(V + j) / 2] : g[(V + j) / 2];
            }
          }
        }
        if (write && h + u * step < n && pr.on[c]) {
          store_n<V>(dst, dtype, off + u * adv + pr.e0[c], x[c]);
          store_n<V>(dst, dtype, off + u * adv + pr.e1[c], y[c]);
        }
      }
    }
  }
}

// V pairs a lane, NC rounds of group * V pairs a head
template <typename TI, int V, int NC>
__global__ void __launch_bounds__(32 * kRotWarps, 4) rotary_rows_kernel(const __grid_constant__ RotParams p) {
  const tosk_rotary_args_t& a = p.a;
  __shared__ float2 s_cs[kRotWarps][kMaxPairs];       // magnitude * (cos, -sin) of the warp's token
  __shared__ float s_w[2][2 * kMaxPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & (p.group - 1);
  const long long t = (long long)blockIdx.x * kRotWarps + warp;
  const int part = blockIdx.y;
  const int hd = a.hd, pairs = hd >> 1, rp = a.rot.turn ? a.rot.rot >> 1 : 0;
  pdl_wait();
  pdl_trigger();
  if (a.q_norm || a.k_norm) {
    for (int i = threadIdx.x; i < hd; i += 32 * kRotWarps) {
      s_w[0][i] = a.q_norm ? a.q_norm[i] : 0.0f;
      s_w[1][i] = a.k_norm ? a.k_norm[i] : 0.0f;
    }
    __syncthreads();
  }
  if (t >= a.n_tokens) return;
  Pairs<V, NC> pr;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * p.group + sub) * V;            // first pair
    pr.on[c] = i < pairs;
    pr.turns[c] = i < rp;
    const bool half = pr.turns[c] && a.rot.half;
    pr.e0[c] = half ? i : 2 * i;
    pr.e1[c] = half ? i + rp : 2 * i + V;
  }
  // the token's sines and cosines, and its cache row (append; -1: none)
  bool have = false;
  long long crow = -1;
  auto ready = [&]() {
    if (have) return;
    have = true;
    int s = -1, r = -1;
    if (a.append) {
      s = a.seq[t];
      r = a.slot[t];
    }
    if (rp) {
      const long long pos = a.pos[t];
      for (int i = lane; i < rp; i += 32) {
        const unsigned long long f = a.rot.turn[i] * (unsigned long long)pos;
        float sn, c;
        sincospif((float)(int)(f >> 32) * 4.656612873077393e-10f, &sn, &c);   // 2^-31: half turns
        s_cs[warp][i] = make_float2(c * a.rot.mag, -(sn * a.rot.mag));
      }
      __syncwarp();
    }
    if (s >= 0 && s < a.kv.n_seqs && r >= 0 && r / a.kv.page_size < a.kv.table_stride) {
      const int pg = a.kv.table[(long long)s * a.kv.table_stride + r / a.kv.page_size];
      if (pg >= 0 && pg < a.kv.n_pages) crow = ((long long)pg * a.kv.page_size + r % a.kv.page_size) * a.n_kv;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 v = pr.turns[c] ? s_cs[warp][(c * p.group + sub) * V + j] : make_float2(1.0f, 0.0f);
        pr.c[c][j] = v.x;
        pr.s[c][j] = v.y;
      }
  };
  // the first round of k and of v that is this warp's
  auto first = [&](int before) { return part >= before ? part - before : part - before + p.parts; };
  if (a.n_heads)
    do_heads<TI, V, NC>(p, pr, reinterpret_cast<const TI*>(a.q.src) + t * a.q.sstride, a.n_heads, a.q.dst,
                        t * a.q.dstride, a.q.dtype, true, a.q_norm ? s_w[0] : nullptr, true, part, ready);
  if (a.n_kv) {
    if (a.append) ready();                            // the row's place
    const bool write = !a.append || crow >= 0;
    do_heads<TI, V, NC>(p, pr, reinterpret_cast<const TI*>(a.k.src) + t * a.k.sstride, a.n_kv,
                        a.append ? a.kv.k : a.k.dst, a.append ? crow * hd : t * a.k.dstride,
                        a.append ? a.kv.type : a.k.dtype, write, a.k_norm ? s_w[1] : nullptr, true, first(p.k_first), ready);
    if (a.append)
      do_heads<TI, V, NC>(p, pr, reinterpret_cast<const TI*>(a.v.src) + t * a.v.sstride, a.n_kv, a.kv.v, crow * hd,
                          a.kv.type, write, nullptr, false, first(p.v_first), ready);
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
  const int lanes = v == 1 ? (a->hd / 2 + 3) / 4 : a->hd / 2 / v;    // V = 1 goes four rounds over a head
  p.group = 2;
  while (p.group < lanes) p.group *= 2;
  const int per = 32 / p.group, nq = (a->n_heads + per - 1) / per, nk = (a->n_kv + per - 1) / per;
  const int rounds = nq + nk * (a->append ? 2 : 1);
  // one warp a token once that fills the card's 148 SMs kRotDeep warps deep;
  // else a token's heads go to as many warps as they make rounds
  const long long want = 148ll * kRotDeep;
  long long parts = (want + a->n_tokens - 1) / a->n_tokens;
  if (parts > rounds) parts = rounds;
  p.parts = (int)parts;
  p.k_first = nq % p.parts;
  p.v_first = (nq + nk) % p.parts;
  const unsigned gx = ((unsigned)a->n_tokens + kRotWarps - 1) / kRotWarps;
  const void* f = f32 ? (v == 4 ? (const void*)rotary_rows_kernel<float, 4, 1> : (const void*)rotary_rows_kernel<float, 1, 4>)
                      : (v == 8   ? (const void*)rotary_rows_kernel<__half, 8, 1>
                         : v == 4 ? (const void*)rotary_rows_kernel<__half, 4, 1>
                                  : (const void*)rotary_rows_kernel<__half, 1, 4>);
  return launch_rot(f, p, dim3(gx, p.parts), st);
}
