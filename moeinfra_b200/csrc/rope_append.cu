// Rotary embedding of q and k and the append of k and v to a paged cache, in
// one pass over the rows of a fused q/k/v projection.
//
// For the head x of a token at position p (h = head_dim / 2, i < h):
//   y[i]     = x[i] cos[p,i] - x[i+h] sin[p,i]
//   y[i + h] = x[i+h] cos[p,i] + x[i] sin[p,i]
// in fp32, rounded once; k and v rows land at the token's slot of its page
// (v bit for bit), q rows are returned packed.  No reference counterpart: the
// reference's cache is a growing DynamicCache (engine/engine.py:326-378).
//
// Bound by memory: each element is read once and written once.  A thread
// takes 8 elements of a head's first half and the 8 that rotate with them, so
// every access is 16 bytes and a head of 128 is 8 neighbouring threads.
#include "paged.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

struct RopeArgs {
  const uint16_t* qkv;
  int64_t qkv_stride;
  const float *cos, *sin;
  int64_t max_pos;
  const int32_t *positions, *seq_ids;
  KvPages kv;
  uint16_t* q_out;
  int heads;
};

constexpr int kRopeThreads = 256;

template <typename T, int HD>
__global__ void __launch_bounds__(kRopeThreads) k_rope_append(const RopeArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int kPer = HD / 16;  // threads a head takes
  const int64_t t = blockIdx.x;
  const int32_t pos = a.positions[t];
  const int32_t seq = a.seq_ids ? a.seq_ids[t] : static_cast<int32_t>(t);
  // The token's slot: page >= 0, or -1 for a padding token (position < 0) and
  // for one whose position, sequence or page is out of range (error bit set).
  int64_t page = -1;
  if (pos >= 0) {
    const int entry = pos / a.kv.page_size;
    if (pos < a.max_pos && seq >= 0 && seq < a.kv.seqs && entry < a.kv.max_pages) {
      const int32_t p = a.kv.table[seq * a.kv.table_stride + entry];
      if (p >= 0 && p < a.kv.num_pages) page = p;
    }
    if (page < 0 && threadIdx.x == 0) set_device_error(kErrPage);
  }
  const int slot = page < 0 ? 0 : pos % a.kv.page_size;
  const int items = (a.heads + 2 * a.kv.kv_heads) * kPer;
  for (int i = threadIdx.x; i < items; i += kRopeThreads) {
    const int head = i / kPer, c = (i % kPer) * 8;
    const int kv_head = head - a.heads;  // < 0: a query head; >= kv_heads: a value head
    uint16_t* dst;
    if (kv_head < 0) {
      dst = a.q_out + (t * a.heads + head) * HD;
    } else {
      if (page < 0) continue;
      const bool val = kv_head >= a.kv.kv_heads;
      const int j = val ? kv_head - a.kv.kv_heads : kv_head;
      dst = (val ? a.kv.v + page * a.kv.v_stride : a.kv.k + page * a.kv.k_stride) +
            ((int64_t)j * a.kv.page_size + slot) * HD;
    }
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (page >= 0) {
      const uint16_t* src = a.qkv + t * a.qkv_stride + (int64_t)head * HD + c;
      lo = *reinterpret_cast<const uint4*>(src);
      hi = *reinterpret_cast<const uint4*>(src + HD / 2);
      if (kv_head < a.kv.kv_heads) {
        const float4* cp = reinterpret_cast<const float4*>(a.cos + (int64_t)pos * (HD / 2) + c);
        const float4* sp = reinterpret_cast<const float4*>(a.sin + (int64_t)pos * (HD / 2) + c);
        uint32_t* l = reinterpret_cast<uint32_t*>(&lo);
        uint32_t* h = reinterpret_cast<uint32_t*>(&hi);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const float4 cs = __ldg(cp + v), sn = __ldg(sp + v);
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const float c0 = w ? cs.z : cs.x, c1 = w ? cs.w : cs.y;
            const float s0 = w ? sn.z : sn.x, s1 = w ? sn.w : sn.y;
            const float2 x = T::unpack(l[2 * v + w]), y = T::unpack(h[2 * v + w]);
            l[2 * v + w] = T::pack(x.x * c0 - y.x * s0, x.y * c1 - y.y * s1);
            h[2 * v + w] = T::pack(y.x * c0 + x.x * s0, y.y * c1 + x.y * s1);
          }
        }
      }
    }
    *reinterpret_cast<uint4*>(dst + c) = lo;
    *reinterpret_cast<uint4*>(dst + c + HD / 2) = hi;
  }
}

template <typename T, int HD>
int launch_rope(const RopeArgs& a, int64_t tokens, cudaStream_t s) {
  if (launch_pdl(k_rope_append<T, HD>, dim3(static_cast<unsigned>(tokens)), dim3(kRopeThreads), 0,
                 s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

}  // namespace
}  // namespace moe

extern "C" int moe_rope_append(const uint16_t* qkv, int64_t qkv_stride, const float* cos,
                               const float* sin, int64_t max_pos, const int32_t* positions,
                               const int32_t* seq_ids, int64_t tokens, uint16_t* k_pages,
                               uint16_t* v_pages, int64_t k_page_stride, int64_t v_page_stride,
                               int64_t num_pages, int page_size, const int32_t* block_table,
                               int64_t table_stride, int seqs, int max_pages, int heads,
                               int kv_heads, int head_dim, int dtype, uint16_t* q_out,
                               void* stream) {
  using namespace moe;
  if (tokens < 0 || tokens > INT32_MAX || seqs < 0 || max_pages < 0 || heads < 1 || kv_heads < 1 ||
      heads > 1024 || kv_heads > 1024 || num_pages < 0 || max_pos < 0 || max_pos > INT32_MAX || page_size < 1)
    return MOE_ERR_INVALID_ARG;
  if (dtype != MOE_DTYPE_F16 && dtype != MOE_DTYPE_BF16) return MOE_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return MOE_ERR_UNSUPPORTED;
  const int64_t page_elems = (int64_t)kv_heads * page_size * head_dim;
  if (qkv_stride < (int64_t)(heads + 2 * kv_heads) * head_dim || table_stride < max_pages ||
      (num_pages > 1 && (k_page_stride < page_elems || v_page_stride < page_elems)))
    return MOE_ERR_INVALID_ARG;
  if (tokens == 0) return MOE_OK;
  if (!qkv || !cos || !sin || !positions || !k_pages || !v_pages || !block_table || !q_out)
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(qkv) || !aligned16(cos) || !aligned16(sin) || !aligned16(k_pages) ||
      !aligned16(v_pages) || !aligned16(q_out) || (qkv_stride & 7) || (k_page_stride & 7) ||
      (v_page_stride & 7))
    return MOE_ERR_ALIGNMENT;
  RopeArgs a{qkv, qkv_stride, cos, sin, max_pos, positions, seq_ids,
             KvPages{k_pages, v_pages, k_page_stride, v_page_stride, num_pages, block_table,
                     table_stride, seqs, max_pages, page_size, kv_heads},
             q_out, heads};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MOE_DTYPE_F16)
    return head_dim == 64 ? launch_rope<F16, 64>(a, tokens, s) : launch_rope<F16, 128>(a, tokens, s);
  return head_dim == 64 ? launch_rope<BF16, 64>(a, tokens, s) : launch_rope<BF16, 128>(a, tokens, s);
}
