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
  s.whole = whole_units(s.units, s.chunks);
  s.ctas = static_cast<int>(s.units);
  return s;
}

template <typename T, int HD>
int launch_few(PagedArgs& a, const Shape& sh, cudaStream_t s) {
  return sh.nt == 1 ? launch_tile<T, HD, 1, true>(a, sh, s) : launch_tile<T, HD, 2, true>(a, sh, s);
}

// Measured in a graph (bf16, 32 heads of 128 unless said, us; this kernel / the tcgen05 one):
//   64 x 576 cached keys, 1 node 32.2 / 55.8, 2 nodes 33.7 / 55.6, 4 nodes 39.1 / 56.9;
//   1 x 72, 2 nodes 6.7 / 10.5, 4 nodes 8.9 / 10.5; 1 x 600 12.8 / 17.4; 8 x 600 12.9 / 19.5;
//   heads of 64, 64 x 576, 4 nodes 28.8 / 47.5; 32 KV heads, 8 nodes 105 / 172, 16 nodes 130 / 166.
// Not for 17 to 32 rows (64 x 576, 8 nodes: 77 / 57: four column tiles' sums leave the
// registers), nor where the even cut of paged_line.cuh would have to share units out
// (1 x 4000: 26.7 / 17.8, 64 x about 2050 114.6 / 108.8, 2 x about 100000 177 / 167).
constexpr int kMostRows = 16;

}  // namespace

bool tree_is_few(const TreeRows& r) {
  return (int64_t)r.nodes * r.group <= kMostRows && few_shape(r).whole;
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
