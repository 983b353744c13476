// paged_common.cuh - what the paged attention kernels share: the problem as
// the kernels see it, partial results of a split key axis, and the plain
// recomputation of single rows.
#pragma once
#include <cuda_fp16.h>

#include "tos_dev.cuh"
#include "tos_kernels.h"

namespace tos {

// One attention problem: n_seqs sequences, the query rows of sequence i being
// tokens q0..q0+qn of q.  A decode step has one token a sequence (cu_q NULL);
// its shared prefix is one "sequence" of all tokens over the prefix's pages,
// not causal.
struct PagedProblem {
  void* out;
  const void* q;
  long long out_stride, q_stride;
  int type;                    // of q and out
  const void *k, *v;
  int kv_type, n_pages, page_size, n_kv, hd, heads, group;   // group = heads / n_kv
  int gshift, pshift;          // log2 of a group, a page size that is a power of two, else -1
  const int *table, *cu_q, *kv_len;
  int n_seqs, total_q, max_q, max_kv, table_stride;
  int fixed_kv;                // >= 0: every sequence's key count (prefix)
  int causal;
  float scale_log2;            // scale * log2(e): the softmax runs in base 2
  // split key axis: split s takes keys [s * chunk, (s + 1) * chunk); partial
  // rows go to slots slot0 .. of part_o / part_ml; splits 0: straight to out
  int splits, chunk, slot0;
  float* part_o;               // [slot][total_q * heads][hd], not normalised
  float2* part_ml;             // [slot][total_q * heads]: running maximum (base 2), sum
  float* fold;                 // tensor-core kernel, fp32 rows, many keys: every CTA's own sums so far
  int* err;
};

// Token and head of packed row r; a division only where the group needs one.
__device__ __forceinline__ int row_token(const PagedProblem& p, int r) { return p.gshift >= 0 ? r >> p.gshift : r / p.group; }
__device__ __forceinline__ int row_head(const PagedProblem& p, int r) {
  return p.gshift >= 0 ? r & (p.group - 1) : r % p.group;
}

struct SeqTask {
  int q0, qn, kvn, off;        // first token, tokens, keys; row r sees keys < off + r + 1 (causal) or kvn
  const int* table;
};

__device__ __forceinline__ SeqTask seq_task(const PagedProblem& p, int s) {
  SeqTask t;
  if (p.fixed_kv >= 0) {       // the prefix: every token, all its keys
    t.q0 = 0;
    t.qn = p.total_q;
    t.kvn = p.fixed_kv;
  } else {
    if (p.cu_q) {
      const int a = p.cu_q[s], b = p.cu_q[s + 1];
      t.q0 = max(a, 0);
      t.qn = min(min(b, p.total_q) - t.q0, p.max_q);
      t.off = b - a;
    } else {
      t.q0 = s;
      t.qn = 1;
      t.off = 1;
    }
    const int len = p.kv_len[s];
    t.kvn = min(len, p.max_kv);
    if ((long long)t.kvn > (long long)p.table_stride * p.page_size) t.kvn = p.table_stride * p.page_size;
    t.off = len - t.off;       // position of row 0; negative: rows that see nothing
  }
  if (p.fixed_kv >= 0) t.off = 0;
  t.kvn = max(t.kvn, 0);
  t.qn = max(t.qn, 0);
  t.table = p.table + (long long)s * p.table_stride;
  return t;
}

// Keys that row r (a token of the sequence) sees.
__device__ __forceinline__ int seen(const PagedProblem& p, const SeqTask& t, int r) {
  return p.causal ? max(0, min(t.kvn, t.off + r + 1)) : t.kvn;
}

// Element offset of key j's row (head kvh) in the cache, -1 where its page is
// not one.
__device__ __forceinline__ long long kv_off(const PagedProblem& p, const int* table, int j, int kvh) {
  const int pg = table[j / p.page_size];
  if (pg < 0 || pg >= p.n_pages) return -1;
  return (((long long)pg * p.page_size + j % p.page_size) * p.n_kv + kvh) * p.hd;
}

__device__ __forceinline__ float load_elem(const void* p, int type, long long i) {
  return type == TOSK_F32 ? reinterpret_cast<const float*>(p)[i] : __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int type, long long i, float v) {
  if (type == TOSK_F32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// One output row by one warp, key by key and seen keys only.  The tiled
// kernels multiply whole key tiles with weights that are zero where a row
// does not see a key; 0 * inf or 0 * NaN of an unseen value then shows as NaN
// in the row.  Such rows are computed again here, where an unseen key is not
// read at all (a row with a NaN of its own gets it again).  prefix: keys
// before the sequence's own (decode).
static __device__ __noinline__ void attn_row_plain(const PagedProblem& p, const int* prefix_table, int prefix_len,
                                            const int* table, int n, int tok, int h) {
  const int lane = threadIdx.x & 31;
  const long long qo = (long long)tok * p.q_stride + (long long)h * p.hd;
  const int kvh = h / p.group;
  float o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.0f;
  for (int seg = 0; seg < 2; ++seg) {
    const int* tb = seg ? table : prefix_table;
    const int cnt = seg ? n : prefix_len;
    for (int j = 0; j < cnt; ++j) {
      const long long ko = kv_off(p, tb, j, kvh);
      float s = 0.0f;
      if (ko >= 0)
        for (int d = lane; d < p.hd; d += 32) s = fmaf(load_elem(p.q, p.type, qo + d), load_elem(p.k, p.kv_type, ko + d), s);
      for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s *= p.scale_log2;
      const float mn = fmaxf(m, s);
      const float c = mn == -INFINITY ? 1.0f : exp2f(m - mn);
      const float w = mn == -INFINITY ? 0.0f : exp2f(s - mn);
      l = fmaf(l, c, w);
      m = mn;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = lane + 32 * i;
        if (d < p.hd) o[i] = fmaf(o[i], c, ko >= 0 ? w * load_elem(p.v, p.kv_type, ko + d) : 0.0f);
      }
    }
  }
  const long long oo = (long long)tok * p.out_stride + (long long)h * p.hd;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d < p.hd) store_elem(p.out, p.type, oo + d, l == 0.0f ? 0.0f : o[i] / l);
  }
}

}  // namespace tos
