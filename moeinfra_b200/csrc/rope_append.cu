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
// every access is 16 bytes and a head of 128 is 8 neighbouring threads; a block
// is one token, whose row is requested before the token's slot is looked up.
// Measured, 32 / 8 heads of 128 fp16: 64 prompts (21527 tokens, 530 MB) 95 us, 5.6
// TB/s (with 2, 3, 4 tokens a block 110, 103, 100 us); one token 1.9 us.
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
  uint16_t* k_out;  // the rotated keys packed too (prompts attend to them), or null
  int heads;
  const int32_t* slots;  // the positions' places in their sequence, or null: themselves
};

constexpr int kMaxThreads = 512;

template <typename T, int HD>
__global__ void __launch_bounds__(kMaxThreads) k_rope_append(const RopeArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int kPer = HD / 16;  // threads a head takes
  const int64_t t = blockIdx.x;
  const int items = (a.heads + 2 * a.kv.kv_heads) * kPer;
  // The first row pieces are on their way while the position, then the page
  // and the angles are looked up.
  const uint16_t* row = a.qkv + t * a.qkv_stride;
  auto source = [&](int i) { return row + (int64_t)(i / kPer) * HD + i % kPer * 8; };
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  if (threadIdx.x < items) {
    lo = *reinterpret_cast<const uint4*>(source(threadIdx.x));
    hi = *reinterpret_cast<const uint4*>(source(threadIdx.x) + HD / 2);
  }
  const int32_t pos = a.positions[t];
  const int32_t seq = a.seq_ids ? a.seq_ids[t] : static_cast<int32_t>(t);
  // The token's slot: page >= 0, or -1 for a padding token (position < 0) and
  // for one whose position, slot, sequence or page is out of range (error bit set).
  int64_t page = -1;
  const int32_t place = a.slots ? a.slots[t] : pos;
  if (pos >= 0) {
    const int entry = place / a.kv.page_size;
    if (pos < a.max_pos && place >= 0 && seq >= 0 && seq < a.kv.seqs && entry < a.kv.max_pages) {
      const int32_t p = a.kv.table[seq * a.kv.table_stride + entry];
      if (p >= 0 && p < a.kv.num_pages) page = p;
    }
    if (page < 0 && threadIdx.x == 0) set_device_error(kErrPage);
  }
  const int slot = page < 0 ? 0 : place % a.kv.page_size;
  for (int i = threadIdx.x; i < items; i += blockDim.x) {
    if (i != threadIdx.x) {
      lo = *reinterpret_cast<const uint4*>(source(i));
      hi = *reinterpret_cast<const uint4*>(source(i) + HD / 2);
    }
    const int head = i / kPer, c = (i % kPer) * 8;
    const int kv_head = head - a.heads;  // < 0: a query head; >= kv_heads: a value head
    uint16_t *dst, *copy = nullptr;
    if (kv_head < 0) {
      dst = a.q_out + (t * a.heads + head) * HD;
    } else {
      const bool val = kv_head >= a.kv.kv_heads;
      if (a.k_out && !val) copy = a.k_out + (t * a.kv.kv_heads + kv_head) * HD;
      if (page < 0 && !copy) continue;
      const int j = val ? kv_head - a.kv.kv_heads : kv_head;
      const int64_t at = page < 0 ? 0 : page;
      dst = (val ? a.kv.v + at * a.kv.v_stride : a.kv.k + at * a.kv.k_stride) +
            ((int64_t)j * a.kv.page_size + slot) * HD;
    }
    if (page < 0) {
      lo = hi = make_uint4(0, 0, 0, 0);
    } else if (kv_head < a.kv.kv_heads) {
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
    if (copy) {
      *reinterpret_cast<uint4*>(copy + c) = lo;
      *reinterpret_cast<uint4*>(copy + c + HD / 2) = hi;
      if (page < 0) continue;  // padding: a zero row there, nothing appended
    }
    *reinterpret_cast<uint4*>(dst + c) = lo;
    *reinterpret_cast<uint4*>(dst + c + HD / 2) = hi;
  }
}

template <typename T, int HD>
int launch_rope(const RopeArgs& a, int64_t tokens, cudaStream_t s) {
  // A thread per piece of the row and equal rounds: 32 + 16 heads of 128 are one
  // round of 384 threads.
  const int items = (a.heads + 2 * a.kv.kv_heads) * (HD / 16);
  const int rounds = (items + kMaxThreads - 1) / kMaxThreads;
  const int threads = ((items + rounds - 1) / rounds + 31) / 32 * 32;
  if (launch_pdl(k_rope_append<T, HD>, dim3(static_cast<unsigned>(tokens)), dim3(threads), 0, s, a) !=
      cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

}  // namespace
}  // namespace moe

extern "C" int moe_rope_append_slots(const moe_rope_append_args_t* args, const int32_t* slots) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_rope_append_args_t& c = *args;
  if (const int st = check_pages(c.kv); st != MOE_OK) return st;
  if (c.tokens < 0 || c.tokens > INT32_MAX || c.heads < 1 || c.heads > 4096 || c.max_pos < 0 ||
      c.max_pos > INT32_MAX || c.qkv_stride < (c.heads + 2 * c.kv.kv_heads) * c.kv.head_dim)
    return MOE_ERR_INVALID_ARG;
  if (c.tokens == 0) return MOE_OK;
  if (!c.qkv || !c.cos || !c.sin || !c.positions || !c.kv.k_pages || !c.kv.v_pages ||
      !c.kv.block_table || !c.q_out)
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(c.qkv) || !aligned16(c.cos) || !aligned16(c.sin) || !aligned16(c.q_out) ||
      !aligned16(c.k_out) || (c.qkv_stride & 7))
    return MOE_ERR_ALIGNMENT;
  const RopeArgs a{c.qkv, c.qkv_stride, c.cos, c.sin, c.max_pos, c.positions, c.seq_ids,
                   pages_of(c.kv), c.q_out, c.k_out, (int)c.heads, slots};
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (c.kv.dtype == MOE_DTYPE_F16)
    return c.kv.head_dim == 64 ? launch_rope<F16, 64>(a, c.tokens, s)
                               : launch_rope<F16, 128>(a, c.tokens, s);
  return c.kv.head_dim == 64 ? launch_rope<BF16, 64>(a, c.tokens, s)
                             : launch_rope<BF16, 128>(a, c.tokens, s);
}

extern "C" int moe_rope_append(const moe_rope_append_args_t* args) {
  return moe_rope_append_slots(args, nullptr);
}
