// moe_tree_attention for small trees: at most 16 rows (nodes x heads of a group) to a KV
// head, by the kernel for one token per sequence (paged_line.cuh), bound by memory as there: a
// unit's keys and values are read once for all its rows.  The tcgen05 kernel's 128-row tiles would
// be seven eighths empty, and a unit's start and end (TMEM, barriers, the join's kernel) would cost
// more than its keys: see kMostRows for both kernels' times.
#include "tree.cuh"

namespace moe {
namespace {
MOE_DEFINE_ERROR_WORD()
}  // namespace
}  // namespace moe

#include "paged_line.cuh"

namespace moe {
namespace {

Shape few_shape(const TreeRows& r) {
  Shape s;
  s.parts = 1;
  s.tile = r.nodes * r.group;
  s.nt = s.tile <= 8 ? 1 : 2;
  s.units = (int64_t)r.kv.seqs * r.kv.kv_heads;
  s.chunks = ceil_div((int64_t)r.kv.max_pages * r.kv.page_size, kChunk);
  s.whole = true;
  s.ctas = static_cast<int>(s.units);
  return s;
}

template <typename T, int HD>
int launch_few(PagedArgs& a, const Shape& sh, cudaStream_t s) {
  return sh.nt == 1 ? launch_tile<T, HD, 1, true>(a, sh, s) : launch_tile<T, HD, 2, true>(a, sh, s);
}

// Rows, and the table's width in chunks of 16 keys where each unit has a place of its own on the
// GPU, and where there are more units: a unit is one CTA's here.  In a graph (32 / 8 heads of 128
// unless said, us; this kernel / the tcgen05 one):
//   64 x 512..640 cached keys, 1 node 32.0 / 43.7, 2 nodes 33.4 / 44.2, 4 nodes 38.8 / 44.2; heads of
//   64, 4 nodes 28.7 / 38.9; 32 KV heads, 8 nodes 104 / 130, 16 nodes 128 / 131; of 64, 64 x 20..40,
//   4 nodes 31.8 / 54.4, 16 nodes 52.9 / 54.7; 1 x 72, 2 nodes 6.2 / 9.4, 4 nodes 8.5 / 9.4;
//   4 nodes over 1 x 600 12.4 / 12.9, over 8 x 600 12.7 / 14.8.
// Not for 17 to 32 rows (64 x 512..640, 8 nodes: 77 / 44: four column tiles' sums leave the
// registers), nor for longer tables (4 nodes over 1 x 800 14.7 / 13.2, over 20 x 500..2000 38.3 /
// 31.6, over 64 x 500..2000 69.7 / 68.0; but 64 x 250..1000 42.7 / 44.8).
constexpr int kMostRows = 16, kChunksAlone = 40, kMostChunksOfMany = 64;

}  // namespace

bool tree_is_few(const TreeRows& r) {
  const Shape sh = few_shape(r);
  return sh.tile <= kMostRows && sh.chunks <= (sh.units <= sm_count() ? kChunksAlone : kMostChunksOfMany);
}

int tree_attention_few(const TreeRows& r, int hd, bool bf16, cudaStream_t s) {
  const Shape sh = few_shape(r);
  PagedArgs a{};
  a.lengths = r.lengths;
  a.kv = r.kv;
  a.scale_log2 = r.scale_log2;
  a.heads = r.heads;
  a.per_seq = r.kv.kv_heads;
  a.tile = sh.tile;
  a.parts = 1;
  a.page_chunks = r.kv.page_size / kChunk;
  a.page_shift = -1;
  for (int i = 0; i < 27; ++i)
    if (a.page_chunks == 1 << i) a.page_shift = i;
  a.tree = r;
  if (bf16) return hd == 64 ? launch_few<BF16, 64>(a, sh, s) : launch_few<BF16, 128>(a, sh, s);
  return hd == 64 ? launch_few<F16, 64>(a, sh, s) : launch_few<F16, 128>(a, sh, s);
}

}  // namespace moe
