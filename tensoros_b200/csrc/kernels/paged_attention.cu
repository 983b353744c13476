// paged_attention.cu - attention over a paged K/V cache: the general kernel
// (any head dimension up to 256, fp32 or fp16 cache, any page size), the
// joining of a split key axis, and the launch plans.
//
//   o_r = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q_r.k_j - m),  c = scale log2 e
//
// in one pass over the keys with a running maximum m and sum per row; a new
// maximum scales what was summed so far by 2^(m_old - m_new).
//
// general kernel.  A CTA takes R packed rows (token, query head of the group)
// of one sequence and one key/value head, so a K/V row read serves all of the
// group's heads, and walks the keys in tiles of 64 staged in shared memory as
// fp32.  256 threads as 16 x 16: thread (ty, tx) owns rows ty + 16 i and, for
// the scores, keys tx + 16 j, for the sums, dims 4 tx + 64 j.  All arithmetic
// is fp32 FMA (packed, two at a time).  R = 64 for prompts, 16 where a sequence
// brings few rows.  It serves what the faster kernels refuse.  One prompt of 2048
// tokens, 32 / 8 heads x 128, fp32 cache: 1.1 ms, 31 TFLOP/s, bound by shared
// memory reads (70% busy, the FMA pipe 48%).  R = 128 reads less a product: 1.0 ms
// there, but 700 tokens of 16 heads take 197 us instead of 117, so 64 is the most.
#include <cuda_runtime.h>

#include "paged_common.cuh"
#include "paged_tc.cuh"

namespace tos {

constexpr int kKT = 64;      // keys a tile
constexpr int kGenThreads = 256;

__device__ __forceinline__ float4 load4(const void* p, int type, long long i, bool vec) {
  if (type == TOSK_F32) {
    const float* f = reinterpret_cast<const float*>(p) + i;
    if (vec) return *reinterpret_cast<const float4*>(f);
    return make_float4(f[0], f[1], f[2], f[3]);
  }
  const __half* h = reinterpret_cast<const __half*>(p) + i;
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(h);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    return make_float4(a.x, a.y, b.x, b.y);
  }
  return make_float4(__half2float(h[0]), __half2float(h[1]), __half2float(h[2]), __half2float(h[3]));
}
// four elements from i on of a row of hd, zeros behind its end
__device__ __forceinline__ float4 load4_tail(const void* p, int type, long long row, int d, int hd, bool vec) {
  if (d + 4 <= hd) return load4(p, type, row + d, vec);
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < hd) v.x = load_elem(p, type, row + d);
  if (d + 1 < hd) v.y = load_elem(p, type, row + d + 1);
  if (d + 2 < hd) v.z = load_elem(p, type, row + d + 2);
  return v;
}

struct GenArgs {
  PagedProblem p;
  int rtiles;                // row tiles of the longest sequence
  int q_vec, kv_vec;         // four-element accesses are aligned
};

// The values that this thread has just put into a tile, of keys that not all rows
// see (row r of the tile is key at + r of those): what is not finite becomes
// zero, and its key is noted.
template <int NJ>
static __device__ __noinline__ void clean_values(float* sv, int at, uint32_t* s_odd) {
#pragma unroll 1
  for (int i = threadIdx.x; i < kKT * 16 * NJ; i += kGenThreads) {
    const int r = i / (16 * NJ), c = i % (16 * NJ);
    uint4* u = reinterpret_cast<uint4*>(sv + r * (64 * NJ + 4) + 4 * c);
    uint4 x = *u;
    if (at + r < 0 || !clean_piece<float>(x)) continue;
    *u = x;
    atomicOr(&s_odd[(at + r) >> 5], 1u << ((at + r) & 31));
  }
}
// Sum of the values that were left out, of dim d at keys [some, lim).
static __device__ __noinline__ float left_out(const PagedProblem& p, const int* table, int kvh, const uint32_t* s_odd,
                                              int some, int lim, int d) {
  float s = 0.0f;
  for (int key = some; key < lim && d < p.hd; ++key)
    if (s_odd[(key - some) >> 5] >> ((key - some) & 31) & 1) {
      const float x = load_elem(p.v, p.kv_type, kv_off(p, table, key, kvh) + d);
      if (not_finite(x)) s += x;
    }
  return s;
}

template <int R, int NJ>
__global__ void __launch_bounds__(kGenThreads) paged_attn_general_kernel(const __grid_constant__ GenArgs a) {
  constexpr int RI = R / 16, LD = 64 * NJ + 4, LP = kKT + 4;
  constexpr int NL = kKT * 16 * NJ / kGenThreads;      // 16-byte pieces of K, and of V, a thread a tile
  constexpr bool AHEAD = NJ <= 2;                      // the next tile waits in registers while this one is worked on
  extern __shared__ float sm[];
  float* sq = sm;                       // [R][LD]
  float* sk = sq + R * LD;              // [kKT][LD]
  float* sv = sk + kKT * LD;            // [kKT][LD]
  float* sp = sv + kKT * LD;            // [R][LP]
  __shared__ uint32_t s_odd[2];         // keys from `some` on with values that are not finite, which were left out
  __shared__ long long s_off[2][kKT];   // where the rows of a tile lie
  const PagedProblem& p = a.p;
  pdl_wait();
  pdl_trigger();
  int b = blockIdx.x;
  const int kvh = b % p.n_kv;
  b /= p.n_kv;
  const int seq = b % p.n_seqs;
  b /= p.n_seqs;
  const int split = p.splits ? b % p.splits : 0;
  const int rt = a.rtiles - 1 - (p.splits ? b / p.splits : b);   // long rows first
  const SeqTask t = seq_task(p, seq);
  const int rows = t.qn * p.group, r0 = rt * R;
  if (r0 >= rows) return;
  const int nr = min(R, rows - r0);
  const int first = seen(p, t, r0 / p.group);          // keys that all rows see
  int k0 = 0, k1 = seen(p, t, (r0 + nr - 1) / p.group);
  if (p.splits) {
    k0 = split * p.chunk;
    k1 = min(k1, k0 + p.chunk);
    if (k0 >= k1) return;               // no row of the tile sees a key of this split
  }
  // from here on not all rows see a key (of at most 63, a row tile's tokens); none: far behind
  const int some = first < k1 ? max(first, k0) : 0x7fff0000;
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int hd4 = (p.hd + 3) / 4;
  auto place = [&](int kt, int buf) {
    if (tid < kKT) s_off[buf][tid] = kt + tid < k1 ? kv_off(p, t.table, kt + tid, kvh) : -1;
  };
  float4 rk[AHEAD ? NL : 1], rv[AHEAD ? NL : 1];
  auto piece = [&](int i, int buf, float4& kx, float4& vx) {
    const int r = i / (16 * NJ), c = i % (16 * NJ);
    const long long off = s_off[buf][r];
    kx = vx = make_float4(0.f, 0.f, 0.f, 0.f);
    if (off >= 0 && c < hd4) {
      kx = load4_tail(p.k, p.kv_type, off, 4 * c, p.hd, a.kv_vec);
      vx = load4_tail(p.v, p.kv_type, off, 4 * c, p.hd, a.kv_vec);
    }
  };
  auto put = [&](int i, const float4& kx, const float4& vx) {
    const int r = i / (16 * NJ), c = i % (16 * NJ);
    *reinterpret_cast<float4*>(sk + r * LD + 4 * c) = kx;
    *reinterpret_cast<float4*>(sv + r * LD + 4 * c) = vx;
  };
  place(k0, 0);
  if (tid < 2) s_odd[tid] = 0;
#pragma unroll 4
  for (int i = tid; i < R * 16 * NJ; i += kGenThreads) {
    const int r = i / (16 * NJ), c = i % (16 * NJ);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < nr && c < hd4) {
      const int rr = r0 + r;
      v = load4_tail(p.q, p.type, (long long)(t.q0 + rr / p.group) * p.q_stride +
                                      (long long)(kvh * p.group + rr % p.group) * p.hd, 4 * c, p.hd, a.q_vec);
    }
    *reinterpret_cast<float4*>(sq + r * LD + 4 * c) = v;
  }
  int lim[RI];
  float m[RI], l[RI], o[RI][NJ][4];
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    const int r = ty + 16 * i;
    lim[i] = r < nr ? min(k1, seen(p, t, (r0 + r) / p.group)) : 0;
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][j][e] = 0.0f;
  }
  __syncthreads();
  if (AHEAD) {
#pragma unroll
    for (int x = 0; x < NL; ++x) piece(tid + x * kGenThreads, 0, rk[AHEAD ? x : 0], rv[AHEAD ? x : 0]);
  }
  int buf = 0;
  for (int kt = k0; kt < k1; kt += kKT, buf ^= 1) {
    place(kt + kKT, buf ^ 1);
#pragma unroll
    for (int x = 0; x < NL; ++x) {
      if (AHEAD) {
        put(tid + x * kGenThreads, rk[AHEAD ? x : 0], rv[AHEAD ? x : 0]);
      } else {
        float4 kx, vx;
        piece(tid + x * kGenThreads, buf, kx, vx);
        put(tid + x * kGenThreads, kx, vx);
      }
    }
    if (kt + kKT > some) clean_values<NJ>(sv, kt - some, s_odd);
    __syncthreads();
    if (AHEAD && kt + kKT < k1) {
#pragma unroll
      for (int x = 0; x < NL; ++x) piece(tid + x * kGenThreads, buf ^ 1, rk[AHEAD ? x : 0], rv[AHEAD ? x : 0]);
    }
    float2 s2[RI][4];                           // even and odd dims apart: packed FMAs
    float s[RI][4];
#pragma unroll
    for (int i = 0; i < RI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s2[i][j] = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int c = 0; c < hd4; ++c) {
      float4 kx[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) kx[j] = *reinterpret_cast<const float4*>(sk + (tx + 16 * j) * LD + 4 * c);
#pragma unroll
      for (int i = 0; i < RI; ++i) {
        const float4 qx = *reinterpret_cast<const float4*>(sq + (ty + 16 * i) * LD + 4 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s2[i][j] = __ffma2_rn(make_float2(qx.x, qx.y), make_float2(kx[j].x, kx[j].y), s2[i][j]);
          s2[i][j] = __ffma2_rn(make_float2(qx.z, qx.w), make_float2(kx[j].z, kx[j].w), s2[i][j]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < RI; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = kt + tx + 16 * j < lim[i] ? (s2[i][j].x + s2[i][j].y) * p.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int x = 8; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.0f : mn;
      const float c = exp2f(m[i] - base);       // 2^-inf = 0 on a row's first keys
      m[i] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float w = exp2f(s[i][j] - base);
        sum += w;
        sp[(ty + 16 * i) * LP + tx + 16 * j] = w;
      }
      l[i] = fmaf(l[i], c, sum);                // this thread's keys; joined at the end
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][j][e] *= c;
    }
    __syncwarp();                               // a row's weights come from its own half warp
    const int kn = min(kKT, k1 - kt);           // the rows behind are zeros, with weights of zero
#pragma unroll 2
    for (int kk = 0; kk < kn; kk += 4) {
      float4 w[RI];
#pragma unroll
      for (int i = 0; i < RI; ++i) w[i] = *reinterpret_cast<const float4*>(sp + (ty + 16 * i) * LP + kk);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const float4 vx = *reinterpret_cast<const float4*>(sv + (kk + e) * LD + 4 * tx + 64 * j);
#pragma unroll
          for (int i = 0; i < RI; ++i) {
            const float we = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
            const float2 w2 = make_float2(we, we);
            const float2 a0 = __ffma2_rn(w2, make_float2(vx.x, vx.y), make_float2(o[i][j][0], o[i][j][1]));
            const float2 a1 = __ffma2_rn(w2, make_float2(vx.z, vx.w), make_float2(o[i][j][2], o[i][j][3]));
            o[i][j][0] = a0.x; o[i][j][1] = a0.y;
            o[i][j][2] = a1.x; o[i][j][3] = a1.y;
          }
        }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < RI; ++i) {
    float sum = l[i];
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const int r = ty + 16 * i;
    if (r >= nr) continue;
    const int rr = r0 + r, tok = t.q0 + rr / p.group, h = kvh * p.group + rr % p.group;
    if (s_odd[0] | s_odd[1]) {
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[i][j][e] += left_out(p, t.table, kvh, s_odd, some, lim[i], 4 * tx + 64 * j + e);
    }
    if (p.splits) {
      const long long row = (long long)(p.slot0 + split) * p.total_q * p.heads + (long long)tok * p.heads + h;
      if (tx == 0) p.part_ml[row] = make_float2(m[i], sum);
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * tx + 64 * j + e < p.hd) p.part_o[row * p.hd + 4 * tx + 64 * j + e] = o[i][j][e];
    } else {
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const long long oo = (long long)tok * p.out_stride + (long long)h * p.hd;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * tx + 64 * j + e < p.hd) store_elem(p.out, p.type, oo + 4 * tx + 64 * j + e, o[i][j][e] * inv);
    }
  }
}

// Joins the partial rows of a split key axis: o = sum_s 2^(m_s - M) o_s /
// sum_s 2^(m_s - M) l_s.  A warp a row; the slots of the prefix come first.
struct JoinArgs {
  PagedProblem p;              // of the sequences' own keys; splits: slots they have
  int pre_splits;              // slots of the prefix, all of them written
  int out_vec;                 // four-element stores to out are aligned
  const int* counts;           // NULL, or partial rows of every row; where it has one, it is not one but done
};

// V elements a lane a round, N rounds.  A warp waits on its slots' rows: eight
// CTAs an SM hide more of that than 94 registers a thread gain (700 tokens of 64
// heads, 4 slots: 42 us, so 33; with more elements a lane the registers are worth more).
template <int V, int N>
__global__ void __launch_bounds__(128, V * N <= 4 ? 8 : 1) paged_attn_join_kernel(const __grid_constant__ JoinArgs a) {
  constexpr int U = V * N <= 4 ? 8 : 4;       // slots whose rows are in flight together
  const PagedProblem& p = a.p;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int seq = blockIdx.y;
  const SeqTask t = seq_task(p, seq);
  const int w = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (w >= t.qn * p.heads) return;
  const int r = w / p.heads, h = w % p.heads, tok = t.q0 + r;
  const int n = seen(p, t, r);
  const long long row = (long long)tok * p.heads + h, step = (long long)p.total_q * p.heads;
  const int cnt = a.counts ? a.counts[row] : a.pre_splits + (n + p.chunk - 1) / p.chunk;
  if (a.counts && cnt <= 1) return;
  // running over rounds of 32 slots, lane i has slot s0 + i
  float M = -INFINITY, L = 0.0f, o[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) o[i][e] = 0.0f;
  for (int s0 = 0; s0 < cnt; s0 += 32) {
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (s0 + lane < cnt) ml = p.part_ml[(s0 + lane) * step + row];
    float mx = ml.x;
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    const float mn = fmaxf(M, mx), base = mn == -INFINITY ? 0.0f : mn;
    const float f = exp2f(M - base), c = exp2f(ml.x - base);
    M = mn;
    L = fmaf(L, f, ml.y * c);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) o[i][e] *= f;
    const int m = min(32, cnt - s0);
    for (int s = 0; s < m; s += U) {
      float x[U][N][V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* src = p.part_o + ((s0 + s + u) * step + row) * p.hd;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int d = (lane + 32 * i) * V;
          const bool have = s + u < m && d < p.hd;
          if constexpr (V == 4) {
            const float4 q = have ? *reinterpret_cast<const float4*>(src + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[u][i][0] = q.x; x[u][i][1] = q.y; x[u][i][2] = q.z; x[u][i][3] = q.w;
          } else {
            x[u][i][0] = have ? src[d] : 0.0f;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float cu = __shfl_sync(0xffffffffu, c, (s + u) & 31);
        if (s + u < m) {
#pragma unroll
          for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) o[i][e] = fmaf(x[u][i][e], cu, o[i][e]);
        }
      }
    }
  }
  for (int x = 16; x > 0; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  const long long oo = (long long)tok * p.out_stride + (long long)h * p.hd;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = (lane + 32 * i) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) o[i][e] = L == 0.0f ? 0.0f : o[i][e] * inv;
    if (d >= p.hd) continue;
    if constexpr (V == 4) {
      if (a.out_vec && p.type == TOSK_F32) {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + oo + d) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
        continue;
      }
      if (a.out_vec) {
        const __half2 x = __floats2half2_rn(o[i][0], o[i][1]), y = __floats2half2_rn(o[i][2], o[i][3]);
        uint2 u;
        u.x = *reinterpret_cast<const uint32_t*>(&x);
        u.y = *reinterpret_cast<const uint32_t*>(&y);
        *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p.out) + oo + d) = u;
        continue;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) store_elem(p.out, p.type, oo + d + e, o[i][e]);
  }
}

}  // namespace tos

using namespace tos;

namespace {
constexpr int kSms = 148;

int launch(const void* func, dim3 grid, int threads, size_t smem, const void* arg, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {const_cast<void*>(arg)};
  return (int)cudaLaunchKernelExC(&cfg, func, args);
}

PagedProblem problem_of(const tosk_paged_attn_t* a) {
  PagedProblem p = {};
  p.out = a->out; p.q = a->q;
  p.out_stride = a->out_stride; p.q_stride = a->q_stride;
  p.type = a->type;
  p.k = a->kv.k; p.v = a->kv.v;
  p.kv_type = a->kv.type; p.n_pages = a->kv.n_pages; p.page_size = a->kv.page_size;
  p.n_kv = a->kv.n_kv; p.hd = a->kv.hd;
  p.heads = a->n_heads; p.group = a->n_heads / a->kv.n_kv;
  p.gshift = p.pshift = -1;
  for (int i = 0; i < 31; ++i) {
    if (p.group == 1 << i) p.gshift = i;
    if (p.page_size == 1 << i) p.pshift = i;
  }
  p.table = a->kv.table; p.table_stride = a->kv.table_stride;
  p.cu_q = a->cu_q; p.kv_len = a->kv_len;
  p.n_seqs = a->n_seqs; p.total_q = a->total_q; p.max_q = a->max_q;
  p.max_kv = a->room > 0 && a->room < a->max_kv ? a->room : a->max_kv;
  p.fixed_kv = -1;
  p.causal = 1;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.err = a->err;
  return p;
}

// ------------------------------------------------------------ general kernel
bool aligned4(const void* p, long long stride, int type, int hd) {
  return ((uintptr_t)p & (type == TOSK_F32 ? 15 : 7)) == 0 && stride % 4 == 0 && hd % 4 == 0;
}

template <int R, int NJ>
int general_launch(const GenArgs& g, long long grid, cudaStream_t st) {
  const size_t smem = ((size_t)(R + 2 * kKT) * (64 * NJ + 4) + (size_t)R * (kKT + 4)) * 4;
  const void* f = (const void*)paged_attn_general_kernel<R, NJ>;
  // per call: the attribute belongs to the device, and setting it is a host-side store
  const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return (int)e;
  return launch(f, dim3((unsigned)grid), kGenThreads, smem, &g, st);
}

template <int R>
int general_rows(const PagedProblem& p, cudaStream_t st) {
  GenArgs g;
  g.p = p;
  const long long rows = (long long)(p.fixed_kv >= 0 ? p.total_q : p.max_q) * p.group;
  g.rtiles = (int)((rows + R - 1) / R);
  g.q_vec = aligned4(p.q, p.q_stride, p.type, p.hd);
  g.kv_vec = aligned4(p.k, 4, p.kv_type, p.hd) && aligned4(p.v, 4, p.kv_type, p.hd);
  const long long grid = (long long)g.rtiles * (p.splits ? p.splits : 1) * p.n_seqs * p.n_kv;
  if (grid > 0x7fffffffll) return (int)cudaErrorInvalidValue;
  if (p.hd <= 64) return general_launch<R, 1>(g, grid, st);
  if (p.hd <= 128) return general_launch<R, 2>(g, grid, st);
  return general_launch<R, 4>(g, grid, st);
}

int run_general(const PagedProblem& p, cudaStream_t st) {
  const long long rows = (long long)(p.fixed_kv >= 0 ? p.total_q : p.max_q) * p.group;
  return rows <= 32 ? general_rows<16>(p, st) : general_rows<64>(p, st);
}

// Splits of a key axis: `rounds` CTAs for every SM, at least `least` keys each.
int plan_splits(long long tiles, int keys, int rounds, int least) {
  const long long want = (rounds * kSms + tiles - 1) / tiles;
  const long long most = (keys + least - 1) / least;
  const long long s = want < most ? want : most;
  return s < 1 ? 1 : (int)s;
}
// Keys a split, a multiple of the tensor-core kernel's tile.
int chunk_of(int keys, int splits) { return ((keys + splits - 1) / splits + 127) / 128 * 128; }

struct DecodePlan {
  int own, own_chunk, pre, pre_chunk;   // own 0: whole rows, the prefix's added to them
};
DecodePlan plan_decode(int n_seqs, int max_kv, int prefix_len, int heads, int n_kv) {
  DecodePlan d;
  const long long rows = (long long)n_seqs * (heads / n_kv);
  d.pre = prefix_len > 0 ? plan_splits((rows + 255) / 256 * n_kv, prefix_len, 1, 256) : 0;
  d.pre_chunk = d.pre ? chunk_of(prefix_len, d.pre) : 0;
  if (d.pre) d.pre = (prefix_len + d.pre_chunk - 1) / d.pre_chunk;
  d.own = max_kv > 0 ? plan_splits((long long)n_seqs * n_kv, max_kv, 4, 512) : 1;
  d.own_chunk = max_kv > 0 ? chunk_of(max_kv, d.own) : 128;
  if (max_kv > 0) d.own = (max_kv + d.own_chunk - 1) / d.own_chunk;
  if (d.own == 1) d.own = 0;
  return d;
}

int run_join(const PagedProblem& own, int pre, cudaStream_t st, const int* counts = nullptr) {
  JoinArgs j;
  j.p = own;
  j.counts = counts;
  j.pre_splits = pre;
  const long long gx = ((long long)own.max_q * own.heads + 3) / 4;
  if (gx > 0x7fffffffll || own.n_seqs > 65535) return (int)cudaErrorInvalidValue;
  j.out_vec = aligned4(own.out, own.out_stride, own.type, own.hd);
  const void* f = own.hd % 4   ? (const void*)paged_attn_join_kernel<1, 8>
                  : own.hd <= 128 ? (const void*)paged_attn_join_kernel<4, 1>
                                  : (const void*)paged_attn_join_kernel<4, 2>;
  return launch(f, dim3((unsigned)gx, own.n_seqs), 128, 0, &j, st);
}

// A workspace: `slots` slots of partial rows, then the tensor-core kernel's sums.
size_t slots_bytes(int slots, int total_q, int heads, int hd) {
  const size_t rows = (size_t)slots * total_q * heads;
  return slots ? ((rows * hd * 4 + 15) & ~(size_t)15) + ((rows * 8 + 15) & ~(size_t)15) : 0;
}
void part_views(PagedProblem& p, void* ws, int slots, size_t fold) {
  const size_t rows = (size_t)slots * p.total_q * p.heads;
  uint8_t* b = reinterpret_cast<uint8_t*>(ws);
  p.part_o = reinterpret_cast<float*>(b);
  p.part_ml = reinterpret_cast<float2*>(b + ((rows * p.hd * 4 + 15) & ~(size_t)15));
  p.fold = fold ? reinterpret_cast<float*>(b + slots_bytes(slots, p.total_q, p.heads, p.hd)) : nullptr;
}

// Which kernel takes a problem with several rows a sequence.  The few-rows
// kernels start faster, but read each K/V row once for every 8 (16) rows; how
// much of that they may do before the others are ahead is measured, in MB (one
// sequence, us, others / few rows):
//   fp32 cache     32 x 128: 67 MB 26.0 / 17.7, 268 MB 44.6 / 45.4
//                   6 x 48:  75 MB 42.7 / 24.7, 302 MB 48.7 / 80.0
//   fp16 cache      6 x 48:  38 MB 14.5 / 13.2, 151 MB 20.7 / 26.7
//     fp32 rows    32 x 128:  8 MB 12.3 / 11.1,  34 MB 12.8 / 13.2, 134 MB 17.8 / 25.3
//     fp16 rows    32 x 128:  1 MB  8.9 / 10.8
// Dims between those, groups and several sequences go by the same rule,
// unmeasured; max_kv stands for every sequence's length, so a ragged batch
// counts as if all were the longest.
// A shared prefix goes by its rows a key/value head (all tokens' together), one
// row tile for fp16 caches; a decode call behind 4096 and 16384 keys (us):
//   fp32 cache  32 x 128,   8 rows: 142, 576 / 56, 177;  32 rows: 202, 912 / 140, 480;
//               128 rows: 386 / 493 at 4096;  8 heads, 32 rows: 62, 177 / 50, 120
//   fp16 cache  32 x 128,   8 rows, fp32: 54, 194 / 32, 73;   fp16: 36, 112 / 32, 73
//               32 rows, fp32: 71, 206 / 73, 187;  fp16: 52, 124 / 67, 179
bool few_rows(const PagedProblem& p) {
  if (!paged_decode_ok(p)) return false;
  const bool f16 = p.kv_type == TOSK_F16;
  if (p.fixed_kv >= 0) return p.total_q * (long long)p.group <= (f16 && paged_tc_ok(p) ? 8 : 32);
  const long long mb = !f16 ? 150 : p.hd <= 64 ? 40 : p.type == TOSK_F32 ? 30 : 0;
  // the tensor cores refuse what the few-rows kernel takes (odd pages, 256 dims): the general kernel is the other then
  const long long most = (f16 && !paged_tc_ok(p) ? 150 : mb) * 1000000;
  return (long long)p.total_q * p.heads / 8 * p.max_kv * p.hd * (f16 ? 4 : 8) <= most;
}
int run_tiles(const PagedProblem& p, cudaStream_t st) {
  if (few_rows(p)) return paged_decode_run(p, 0, st);
  return paged_tc_ok(p) ? paged_tc_run(p, st) : run_general(p, st);
}

// Splits of a prompt call's keys (0: none).  Up to two rounds of row tiles over
// the SMs, the keys are cut into the number of splits with the shortest
// schedule, counted in key tiles of 128: rounds over the SMs, each its share
// of the keys and ~3.5 tiles' worth of starting and ending a piece; the joining
// ~2, and a tile's worth for every 1.1 M elements of partial rows.  (A key tile
// takes 2.0 us with fp16 rows, 4.0 with fp32 rows.)  A sequence has a row tile
// of its own, however short: 16 sequences of 8 tokens behind 4096 keys take
// 76 us, 106 where only packed rows are counted; 20 of 16, 122, unsplit 139.
// The estimate does not see that a causal prompt's row tiles differ in length:
// 1200 tokens behind 4000 keys, fp16, 169 us, unsplit 160.
int plan_prompt(int n_seqs, int total_q, int max_kv, int heads, int n_kv, int hd) {
  const long long packed = ((long long)total_q * (heads / n_kv) + 255) / 256;
  const long long tiles = (packed > n_seqs ? packed : n_seqs) * n_kv;
  if (tiles >= 2 * kSms) return 0;
  const float keys = max_kv / 128.0f, rows = (float)total_q * heads * hd / 1.1e6f;
  int best = 1;
  float cost = (float)((tiles + kSms - 1) / kSms) * (keys + 3.5f);
  for (int s = 2; s <= 16 && s <= max_kv / 512; ++s) {
    const float c = (float)((s * tiles + kSms - 1) / kSms) * (keys / s + 3.5f) + 2.0f + s * rows;
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  return best > 1 ? best : 0;
}
}  // namespace

// Keys of one piece of a prompt's work.
int prompt_keys(int splits, int max_kv) { return splits ? chunk_of(max_kv, splits) : max_kv; }

extern "C" size_t tosk_paged_prompt_ws_bytes(int n_seqs, int total_q, int max_kv, int n_heads, int n_kv, int hd) {
  const int splits = plan_prompt(n_seqs, total_q, max_kv, n_heads, n_kv, hd);
  return slots_bytes(splits, total_q, n_heads, hd) + paged_tc_fold_bytes(prompt_keys(splits, max_kv));
}

extern "C" size_t tosk_paged_decode_ws_bytes(int n_seqs, int max_kv, int prefix_len, int n_heads, int n_kv, int hd) {
  const DecodePlan d = plan_decode(n_seqs, max_kv, prefix_len, n_heads, n_kv);
  // the general kernel does not add a prefix: its rows take a slot
  const int slots = d.pre && !d.own ? d.pre + 1 : d.own + d.pre;
  return slots_bytes(slots, n_seqs, n_heads, hd) + paged_tc_fold_bytes(d.pre_chunk);
}

extern "C" int tosk_paged_prompt(const tosk_paged_attn_t* a, cudaStream_t st) {
  PagedProblem p = problem_of(a);
  p.splits = plan_prompt(a->n_seqs, a->total_q, a->max_kv, a->n_heads, a->kv.n_kv, a->kv.hd);
  p.chunk = prompt_keys(p.splits, a->max_kv);
  part_views(p, a->ws, p.splits, paged_tc_fold_bytes(p.chunk));
  const int e = run_tiles(p, st);
  return e || !p.splits ? e : run_join(p, 0, st);
}

extern "C" int tosk_paged_decode(const tosk_paged_attn_t* a, cudaStream_t st) {
  PagedProblem p = problem_of(a);
  DecodePlan d = plan_decode(a->n_seqs, a->max_kv, a->prefix_len, a->n_heads, a->kv.n_kv);
  const bool fast = paged_decode_ok(p);
  if (!fast && d.pre && !d.own) d.own = 1;
  part_views(p, a->ws, d.own + d.pre, paged_tc_fold_bytes(d.pre_chunk));
  if (d.pre) {
    PagedProblem x = p;
    x.table = a->prefix_table;
    x.n_seqs = 1;
    x.cu_q = nullptr;
    x.max_q = p.total_q;
    x.fixed_kv = a->prefix_len;
    x.causal = 0;
    x.splits = d.pre;
    x.chunk = d.pre_chunk;
    const int e = run_tiles(x, st);
    if (e) return e;
  }
  p.splits = d.own;
  p.chunk = d.own_chunk;
  p.slot0 = d.pre;
  const int e = fast ? paged_decode_run(p, d.pre, st) : run_general(p, st);
  if (e || !d.own) return e;
  return run_join(p, d.pre, st);
}

namespace tos {
// What the 8-bit cache's decode kernel (paged8_decode.cu) shares.
PagedProblem paged_problem(const tosk_paged_attn_t* a) { return problem_of(a); }
size_t paged_slots_bytes(int slots, int total_q, int heads, int hd) { return slots_bytes(slots, total_q, heads, hd); }
void paged_part_views(PagedProblem& p, void* ws, int slots) { part_views(p, ws, slots, 0); }
int paged_join(const PagedProblem& p, const int* counts, cudaStream_t st) { return run_join(p, 0, st, counts); }
}  // namespace tos
