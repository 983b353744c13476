// paged_tc.cuh - tcgen05 wrappers and operand descriptors of the paged
// attention kernel (PTX ISA 8.7, sm_100a), and the kernel's launcher.
#pragma once
#include <cuda.h>
#include <cudaTypedefs.h>

#include "paged_common.cuh"

// gemm_tc.cu: cuTensorMapEncodeTiled through the runtime's entry point
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace tos {

bool paged_tc_ok(const PagedProblem& p);
int paged_tc_run(const PagedProblem& p, cudaStream_t st);
size_t paged_tc_fold_bytes(int keys);
long long paged_tc_tiles(int n_seqs, int total_q, int max_q, int group);
// paged_decode.cu
bool paged_decode_ok(const PagedProblem& p);
// pre_slots: partial rows of a shared prefix that a kernel launched just before
// brings, at the slots before the problem's own.
int paged_decode_run(const PagedProblem& p, int pre_slots, cudaStream_t st);

#ifdef __CUDACC__
// Shared-memory operands, rows of 128 bytes swizzled 128 B, eight rows every
// 1024 bytes (the stride offset): the descriptors differ in their low word
// only, and an address within the tile is added to that.  K-major (Q, K: the
// contraction runs along the row) has no leading offset; N-major (V: down the
// rows) has the next 64 columns `lead` bytes on.
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_k(uint32_t saddr) { return (saddr >> 4) | 1u << 16; }
__device__ __forceinline__ uint32_t desc_mn(uint32_t saddr, uint32_t lead) { return (saddr >> 4) | (lead >> 4) << 16; }
// One lane of a converged warp.  The tensor instructions take their operands
// from uniform registers; behind this predicate the compiler knows that one
// thread runs and moves them there directly (with the descriptors' low words above,
// packed fp16 prompts 208 us; lane == 0 and whole descriptors 235).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}
// D (tensor memory) = A B or += A B; A and B in shared memory, or A in tensor
// memory
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b), "r"(idesc), "r"((uint32_t)acc), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Byte offset of 16-byte chunk c (0..7) of row r in a swizzled tile of 128-byte rows.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two floats as packed fp16 high parts and what they leave
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 H = __floats2half2_rn(x, y);
  const float2 f = __half22float2(H);
  const __half2 L = __floats2half2_rn(x - f.x, y - f.y);
  hi = *reinterpret_cast<const uint32_t*>(&H);
  lo = *reinterpret_cast<const uint32_t*>(&L);
}
// Power of two 2^k with m * 2^k in [2^13, 2^14) (m > 0 finite), else 1.
__device__ __forceinline__ float pow2_to_2p13(float m) {
  const int eb = (int)((__float_as_uint(m) >> 23) & 0xFF);
  if (!(m > 0.0f) || eb == 255) return 1.0f;
  const int k = max(-126, min(126, 13 - (eb - 127)));
  return __uint_as_float((uint32_t)(k + 127) << 23);
}
// 1 / s of such a power of two (exponents -126 .. 126)
__device__ __forceinline__ float pow2_inverse(float s) {
  return __uint_as_float((254u << 23) - __float_as_uint(s));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
#endif

}  // namespace tos
