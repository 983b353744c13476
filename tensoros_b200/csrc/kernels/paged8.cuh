// paged8.cuh - a paged cache in 8 bits: its formats and where its rows lie.
//
// `block` neighbouring rows of a sequence share one scale a head, K and V apart,
// a power of two.  So whatever a block stands for is an fp16 number (whole
// numbers up to 127, or e4m3, times 2^e within the limits below): kernels that
// read it round nothing, and a scale that grows when rows arrive shifts what is
// there.  It costs at most one bit of the 8 that a scale of any value would use.
#pragma once
#include <cuda_fp16.h>
#include <string.h>

#include "paged_common.cuh"

namespace tos {

// The exponents' limits keep the smallest step a subnormal fp16 and the largest
// value a finite one.
template <int TYPE>
struct Fmt8;
template <>
struct Fmt8<TOSK_I8> {
  static constexpr int kMinExp = -24, kMaxExp = 9;
  static constexpr uint32_t kTop = 0x42fe0000u;                 // 127.0f
};
template <>
struct Fmt8<TOSK_F8> {
  static constexpr int kMinExp = -15, kMaxExp = 7;
  static constexpr uint32_t kTop = 0x43e00000u;                 // 448.0f
};

// 2^e, e the least with which a magnitude (its fp32 bits) fits; NaN where it is
// not finite.
template <int TYPE>
__device__ __forceinline__ float scale_for(uint32_t amax) {
  if (amax >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
  constexpr uint32_t top = Fmt8<TYPE>::kTop;
  int e = (int)(amax >> 23) - (int)(top >> 23) + ((amax & 0x7fffffu) > (top & 0x7fffffu));
  e = min(max(e, Fmt8<TYPE>::kMinExp), Fmt8<TYPE>::kMaxExp);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Four elements of 8 bits to two half2, as they are (no scale).
// I8: the byte, its sign flipped, becomes the low mantissa bits of 1024 + u.
template <int TYPE>
__device__ __forceinline__ void cvt_word(uint32_t w, uint32_t& a, uint32_t& b) {
  if constexpr (TYPE == TOSK_I8) {
    w ^= 0x80808080u;
    const uint32_t x = prmt(w, 0x64646464u, 0x4140u), y = prmt(w, 0x64646464u, 0x4342u);
    const __half2 off = __float2half2_rn(1152.0f);
    const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&x), off);
    const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&y), off);
    a = *reinterpret_cast<const uint32_t*>(&p);
    b = *reinterpret_cast<const uint32_t*>(&q);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(a), "=r"(b)
        : "r"(w));
  }
}

// Four floats, scaled to the type's range, to its bytes.
template <int TYPE>
__device__ __forceinline__ uint32_t pack_word(float x0, float x1, float x2, float x3) {
  if constexpr (TYPE == TOSK_I8) {
    const int a = min(max(__float2int_rn(x0), -127), 127), b = min(max(__float2int_rn(x1), -127), 127);
    const int c = min(max(__float2int_rn(x2), -127), 127), d = min(max(__float2int_rn(x3), -127), 127);
    return prmt(prmt(a, b, 0x0040u), prmt(c, d, 0x0040u), 0x5410u);
  } else {
    uint32_t w;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(w)
        : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
    return w;
  }
}
// One element of 8 bits as a float.
template <int TYPE>
__device__ __forceinline__ float elem8(uint8_t b) {
  uint32_t x, y;
  cvt_word<TYPE>(b, x, y);
  return __half2float(__ushort_as_half((unsigned short)(x & 0xffffu)));
}

// Where a sequence's rows lie.  Divisions only where page sizes need them.
struct Pool8 {
  uint8_t *k, *v;
  float *ks, *vs;
  int n_pages, page_size, pshift, bshift, bpp;   // blocks of 2^bshift rows, bpp a page
  int n_kv, hd;
  const int* table;
  int n_seqs, table_stride;
};
struct Row8 {
  long long at, scale;        // element of head 0, its scale; at < 0: the page is none
};
__device__ __forceinline__ int page_index(const Pool8& c, int slot) {
  return c.pshift >= 0 ? slot >> c.pshift : slot / c.page_size;
}
// page: the table's entry for page_index(slot)
__device__ __forceinline__ Row8 row8(const Pool8& c, int slot, int page) {
  if (page < 0 || page >= c.n_pages) return {-1, 0};
  const int r = c.pshift >= 0 ? slot & (c.page_size - 1) : slot % c.page_size;
  return {((long long)page * c.page_size + r) * c.n_kv * c.hd, ((long long)page * c.bpp + (r >> c.bshift)) * c.n_kv};
}

// The last of n sequences whose start (ascending, start(0) <= u taken as given)
// is at most u, by a warp.
template <typename F>
__device__ __forceinline__ int find_seq(int n, int u, F start) {
  const int lane = threadIdx.x & 31;
  int lo = 0;
  while (n > 1) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const uint32_t hit = __ballot_sync(0xffffffffu, lane * step < n && start(i) <= u);
    // the first lane that fails; garbage that does not ascend still ends in range
    const int c = max(0, (hit == 0xffffffffu ? 32 : __ffs(~hit) - 1) - 1);
    lo += c * step;
    n = min(step, n - c * step);
  }
  return lo;
}

Pool8 pool8_of(const tosk_paged8_t& kv);      // paged8_store.cu
// paged_attention.cu: the problem of a call, its partial rows in a workspace,
// and their joining
PagedProblem paged_problem(const tosk_paged_attn_t* a);
size_t paged_slots_bytes(int slots, int total_q, int heads, int hd);
void paged_part_views(PagedProblem& p, void* ws, int slots);
int paged_join(const PagedProblem& p, const int* counts, cudaStream_t st);   // counts: see JoinArgs

}  // namespace tos
