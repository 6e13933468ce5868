// moe_paged_attention: attention of one new token per sequence over its pages (the
// kernel: paged_line.cuh).
#include "paged.cuh"

namespace moe {
namespace {
MOE_DEFINE_ERROR_WORD()
}  // namespace
}  // namespace moe

#include "paged_line.cuh"

namespace moe {
namespace {

template <typename T, int HD>
int launch_wide(PagedArgs& a, const Shape& sh, cudaStream_t s) {
  return sh.nt == 1 ? launch_tile<T, HD, 1, false>(a, sh, s) : launch_tile<T, HD, 2, false>(a, sh, s);
}

}  // namespace
}  // namespace moe

extern "C" size_t moe_paged_attention_workspace_size(int64_t seqs, int64_t max_pages,
                                                     int64_t page_size, int64_t heads,
                                                     int64_t kv_heads, int64_t head_dim) {
  using namespace moe;
  if (seqs < 1 || kv_heads < 1 || heads < kv_heads || max_pages < 0 || page_size < 1 ||
      (head_dim != 64 && head_dim != 128) || seqs > kMaxSeqs || heads > 4096)
    return 0;
  const Shape sh = shape_of(seqs, kv_heads, heads / kv_heads, max_pages * page_size);
  return workspace_size(sh, static_cast<int>(head_dim));
}

extern "C" int moe_paged_attention(const moe_paged_attention_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_paged_attention_args_t& c = *args;
  if (const int st = check_pages(c.kv); st != MOE_OK) return st;
  const int64_t hd = c.kv.head_dim;
  const float scale = static_cast<float>(c.scale);
  if (c.heads < 1 || c.heads > 4096 || c.heads % c.kv.kv_heads || !(scale > 0.f && scale < INFINITY) ||
      c.q_stride < c.heads * hd)
    return MOE_ERR_INVALID_ARG;
  if (c.kv.page_size % kChunk || c.kv.seqs > kMaxSeqs) return MOE_ERR_UNSUPPORTED;
  if (c.kv.seqs == 0) return MOE_OK;
  if (!c.q || !c.lengths || !c.out ||
      (c.kv.max_pages > 0 &&
       (!c.kv.k_pages || !c.kv.v_pages || !c.kv.block_table || c.kv.num_pages < 1)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(c.q) || !aligned16(c.out) || (c.q_stride & 7)) return MOE_ERR_ALIGNMENT;
  const Shape sh = shape_of(c.kv.seqs, static_cast<int>(c.kv.kv_heads),
                            static_cast<int>(c.heads / c.kv.kv_heads), c.kv.max_pages * c.kv.page_size);
  if (sh.units * sh.chunks > kMostChunks) return MOE_ERR_UNSUPPORTED;
  if (!c.workspace || c.workspace_bytes < (int64_t)workspace_size(sh, static_cast<int>(hd)))
    return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  PagedArgs a{};
  a.q = c.q;
  a.q_stride = c.q_stride;
  a.out = c.out;
  a.lengths = c.lengths;
  a.kv = pages_of(c.kv);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.heads = static_cast<int>(c.heads);
  a.per_seq = static_cast<int>(c.kv.kv_heads) * sh.parts;
  a.tile = sh.tile;
  a.parts = sh.parts;
  a.page_chunks = a.kv.page_size / kChunk;
  a.page_shift = -1;
  for (int i = 0; i < 27; ++i)
    if (a.page_chunks == 1 << i) a.page_shift = i;
  a.counts = static_cast<int*>(c.workspace);
  a.warp_part = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + kCountBytes);
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (c.kv.dtype == MOE_DTYPE_F16)
    return hd == 64 ? launch_wide<F16, 64>(a, sh, s) : launch_wide<F16, 128>(a, sh, s);
  return hd == 64 ? launch_wide<BF16, 64>(a, sh, s) : launch_wide<BF16, 128>(a, sh, s);
}
