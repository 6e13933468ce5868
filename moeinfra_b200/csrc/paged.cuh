// What the paged-cache kernels share: element types, the cache's description,
// mma.sync / ldmatrix / cp.async wrappers.
//
// A paged cache holds the keys (and, in a second array of the same shape, the
// values) of every sequence in pages [num_pages, kv_heads, page_size, head_dim]
// of contiguous rows (pages may be further apart than their size).  Row b of
// the block table lists sequence b's pages in order: position p is row
// p % page_size of page table[b][p / page_size].
#pragma once

#include "common.cuh"

namespace moe {

struct F16 {
  static constexpr bool kBf16 = false;
  // Probabilities are rounded to 16 bits for the product with V.  fp16 has its
  // smallest normal at 2^-14: times 2^10 a probability keeps all 11 bits down
  // to 2^-24 of the row's largest.  bf16 has fp32's exponents and needs none.
  static constexpr float kProbShift = 10.f;
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint16_t one(float v) { return f2h(v); }
};
struct BF16 {
  static constexpr bool kBf16 = true;
  static constexpr float kProbShift = 0.f;
  static __device__ __forceinline__ float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
  }
  static __device__ __forceinline__ uint16_t one(float v) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
};

struct KvPages {
  uint16_t* k;
  uint16_t* v;
  int64_t k_stride, v_stride;  // elements from one page to the next
  int64_t num_pages;
  const int32_t* table;        // [seqs, max_pages], rows table_stride apart
  int64_t table_stride;
  int seqs, max_pages, page_size, kv_heads;
};

// The cache as a call describes it; MOE_OK, or what is wrong with it.
inline int check_pages(const moe_kv_pages_t& c) {
  if (c.seqs < 0 || c.seqs > INT32_MAX || c.max_pages < 0 || c.max_pages > INT32_MAX ||
      c.kv_heads < 1 || c.kv_heads > 4096 ||
      c.num_pages < 0 || c.page_size < 1 || c.page_size > (1 << 20))
    return MOE_ERR_INVALID_ARG;
  if ((c.dtype != MOE_DTYPE_F16 && c.dtype != MOE_DTYPE_BF16) ||
      (c.head_dim != 64 && c.head_dim != 128) || c.max_pages * c.page_size > INT32_MAX)
    return MOE_ERR_UNSUPPORTED;
  const int64_t page = c.kv_heads * c.page_size * c.head_dim;
  if (c.table_stride < c.max_pages ||
      (c.num_pages > 1 && (c.k_page_stride < page || c.v_page_stride < page)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(c.k_pages) || !aligned16(c.v_pages) || ((c.k_page_stride | c.v_page_stride) & 7))
    return MOE_ERR_ALIGNMENT;
  return MOE_OK;
}
inline KvPages pages_of(const moe_kv_pages_t& c) {
  return KvPages{c.k_pages, c.v_pages, c.k_page_stride, c.v_page_stride, c.num_pages,
                 c.block_table, c.table_stride, (int)c.seqs, (int)c.max_pages, (int)c.page_size,
                 (int)c.kv_heads};
}

// d += a . b for one 16 x 8 x 16 tile, fp32 accumulation.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (T::kBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The 8 x 8 tile of 16-bit values that the warp holds, transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 16 bytes global -> shared, asynchronously; zeros when !take (src is not read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(take ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// 2^x, the hardware's approximation (2 ulp; flushes results below 2^-126).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace moe
