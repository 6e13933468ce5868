// The pages of a cache whose sequences branch: rows of the block table fork,
// end and grow (k_fork_tables, k_fork_copy), and the accepted nodes of a
// verified tree move to the end of their sequence (k_keep_nodes).
//
// Pages are counted: refs[g] is how many rows list page g, 0 means free.  A
// fork is new lines in the block table; keys and values are copied only where
// a row is about to write into a page that others list too, and there only the
// positions that are filled.  No counterpart in the reference (one sequence
// over a growing DynamicCache, engine/engine.py:326-378).
// Measured in a graph (8 KV heads of 128, fp16 but for 8 layers): fork of 1 x 4 rows, 32 layers 8.6 us, of
// 16 x 4, pages of 64 35.8 us (180 MB, 5.0 TB/s), of 32 x 8 rows, 8 layers bf16 44 us, 11 of them the
// tables; nodes of 1 sequence, 32 layers 3.0 us, of 64 9.6 us (34 MB).
#include "paged.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

struct Layers {
  uint16_t *k, *v;
  int64_t k_page, v_page;    // elements from one page to the next
  int64_t k_layer, v_layer;  // and from one layer to the next
  int page_size, kv_heads, layers;
};

constexpr int kMaxRows = 8192;    // of a block table that forks
constexpr int kForkThreads = 1024;
constexpr int kCopyThreads = 256;

struct ForkArgs {
  Layers kv;
  int64_t num_pages;
  int32_t* table;
  int64_t table_stride;
  int rows, max_pages;
  int col_shift;            // log2 of the columns of a CTA
  int32_t* lengths;
  const int32_t* parents;
  int32_t* refs;
  int64_t room;
  int entries;              // pages that `room` positions touch at most
  uint32_t* done;           // CTAs done: zero between calls
  int4* list;               // [0].x: copies; then source, destination, positions of each
};

// Exclusive sum of v over the block's threads; total in every thread.
__device__ __forceinline__ int block_scan(int v, int* s_warp, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  const int w = lane < (int)blockDim.x / 32 ? s_warp[lane] : 0;
  int y = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  total = __shfl_sync(0xffffffffu, y, 31);
  const int before = __shfl_sync(0xffffffffu, y - w, warp);
  __syncthreads();
  return before + x - v;
}

// Rows take their parents' lines, a CTA some columns of all rows (so that a
// line may be read and overwritten in place); then the last CTA to finish gives
// out pages, as if row after row asked for its own:
//   missing page                       the lowest-numbered free one
//   page that other rows list too      the same, its filled positions copied; the
//                                      old page loses the row
// Only entries that change touch the counts: what siblings share stays.
__global__ void __launch_bounds__(kForkThreads) k_fork_tables(const ForkArgs a) {
  extern __shared__ int s_mem[];
  __shared__ int s_warp[32], s_free[kForkThreads], s_copies, s_last;
  __shared__ __align__(16) int s_held[kForkThreads];
  __shared__ int64_t s_cursor;
  const int S = a.rows, tid = threadIdx.x, threads = blockDim.x, cols = 1 << a.col_shift;
  int *s_par = s_mem, *s_old = s_mem + S, *s_tile = s_mem + 2 * S;
  pdl_trigger();
  pdl_wait();
  auto listed = [&](int g) { return g >= 0 && g < a.num_pages; };
  const int c0 = blockIdx.x << a.col_shift;
  // The first entries are on their way while the parents are looked at.
  constexpr int kFirst = 4;
  auto entry_at = [&](int e) {
    const int i = e >> a.col_shift, col = c0 + (e & (cols - 1));
    return e < S << a.col_shift && col < a.max_pages ? a.table[i * a.table_stride + col] : -1;
  };
  int first[kFirst];
#pragma unroll
  for (int u = 0; u < kFirst; ++u) first[u] = entry_at(tid + u * threads);
  for (int i = tid; i < S; i += threads) {
    int p = a.parents[i];
    s_old[i] = a.lengths[i];  // written by the last CTA alone, after all have read
    if (p >= S) {
      set_device_error(kErrPage);
      p = -1;
    }
    s_par[i] = max(p, -1);
  }
#pragma unroll
  for (int u = 0; u < kFirst; ++u)
    if (tid + u * threads < S << a.col_shift) s_tile[tid + u * threads] = first[u];
#pragma unroll 4
  for (int e = tid + kFirst * threads; e < S << a.col_shift; e += threads) s_tile[e] = entry_at(e);
  __syncthreads();
  for (int e = tid; e < S << a.col_shift; e += threads) {
    const int i = e >> a.col_shift, c = e & (cols - 1), p = s_par[i];
    const int was = s_tile[e], is = p >= 0 ? s_tile[(p << a.col_shift) + c] : -1;
    if (is == was || c0 + c >= a.max_pages) continue;
    a.table[i * a.table_stride + c0 + c] = is;
    if (listed(was)) atomicSub(a.refs + was, 1);
    if (listed(is)) atomicAdd(a.refs + is, 1);
  }
  const bool alone = gridDim.x == 1;  // the whole table passes through this CTA's shared memory
  if (!alone) __threadfence();
  __syncthreads();
  if (tid == 0) {
    s_last = alone || atomicAdd(a.done, 1) == gridDim.x - 1;
    s_copies = 0;
    s_cursor = 0;
  }
  __syncthreads();
  if (!s_last) return;
  if (!alone) {
    __threadfence();
    if (tid == 0) *a.done = 0;
  }

  const int page = a.kv.page_size;
  int* s_len = s_tile + (alone ? S << a.col_shift : 0);
  for (int i = tid; i < S; i += threads) {
    int n = s_par[i] >= 0 ? s_old[s_par[i]] : 0;  // negative: no sequence, which is given no page
    if (n > a.max_pages * page) {  // no table's row holds so many
      set_device_error(kErrPage);
      n = a.max_pages * page;
    }
    s_len[i] = n;
    a.lengths[i] = n;
  }
  __syncthreads();
  auto first_of = [&](int i) { return s_len[i] / page; };
  auto last_of = [&](int i) {
    const int64_t c = (s_len[i] + a.room - 1) / page;
    return static_cast<int>(c < a.max_pages ? c : a.max_pages - 1);
  };
  const int64_t asked = (int64_t)S * a.entries;
  for (int64_t base = 0; base < asked; base += threads) {
    const int64_t at = base + tid;
    const int i = static_cast<int>(min(at / a.entries, (int64_t)S - 1));
    const int64_t col = first_of(i) + (at - (int64_t)i * a.entries);
    const bool use = at < asked && s_par[i] >= 0 && s_len[i] >= 0 && col <= last_of(i);
    int32_t* entry = a.table + i * a.table_stride + (use ? col : 0);
    int g = -1;
    if (use) g = alone && base == 0 ? s_tile[(s_par[i] << a.col_shift) + (int)col] : __ldcg(entry);
    if (g >= a.num_pages) {
      set_device_error(kErrPage);
      g = -1;
    }
    const int holders = use && g >= 0 ? __ldcg(a.refs + g) : 0;
    // The counts where the search for free pages goes on come with it.
    constexpr int kLook = 8;  // that a thread looks at in a go
    int32_t r[kLook];
    auto look = [&](int64_t from) {
#pragma unroll
      for (int u = 0; u < kLook; ++u) r[u] = from + u < a.num_pages ? __ldcg(a.refs + from + u) : 1;
    };
    const int64_t ahead = s_cursor;
    look(ahead + tid * kLook);
    // Of the rows that ask in this round and list a page, those before one leave it to
    // it (those of earlier rounds have): the last keeps it.
    const int held = holders > 1 ? g : -1 - tid;
    s_held[tid] = held;
    __syncthreads();
    int before = __popc(__match_any_sync(0xffffffffu, held) & ((1u << (tid & 31)) - 1));
    if (holders > 1) {
      const int4* s4 = reinterpret_cast<const int4*>(s_held);
#pragma unroll 4
      for (int j = 0; j < (tid & ~31) / 4; ++j) {
        const int4 v = s4[j];
        before += (v.x == g) + (v.y == g) + (v.z == g) + (v.w == g);
      }
    }
    const bool copy = holders > 1 && holders - before > 1;
    const bool need = use && (copy || g < 0);
    int wanted, found = 0;
    const int turn = block_scan(need, s_warp, wanted);
    while (found < wanted && s_cursor < a.num_pages) {
      const int64_t from = s_cursor + tid * kLook;
      if (s_cursor != ahead) look(from);
      int mine = 0, more;
#pragma unroll
      for (int u = 0; u < kLook; ++u) mine += r[u] == 0;
      int place = found + block_scan(mine, s_warp, more);
      if (tid == 0) s_cursor += threads * kLook;
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kLook; ++u) {
        if (r[u] != 0) continue;
        if (place < wanted) s_free[place] = static_cast<int>(from + u);
        if (place == wanted - 1) s_cursor = from + u + 1;
        ++place;
      }
      found = min(found + more, wanted);
      __syncthreads();
    }
    if (need) {
      int dst = -1;
      if (turn < found) {
        dst = s_free[turn];
        a.refs[dst] = 1;
      } else {
        set_device_error(kErrPage);  // no page left: the row has none there
      }
      *entry = dst;
      if (copy) {
        atomicSub(a.refs + g, 1);
        const int64_t filled = s_len[i] - col * page;
        if (dst >= 0 && filled > 0) a.list[1 + atomicAdd(&s_copies, 1)] = make_int4(g, dst, (int)filled, 0);
      }
    }
    __syncthreads();
  }
  if (tid == 0) a.list[0].x = s_copies;
}

// The listed pages' filled positions, 4 KB of a (layer, keys or values, head) to
// a warp: eight 16-byte loads of a lane are in flight before the first store.
template <int HD>
__global__ void __launch_bounds__(kCopyThreads) k_fork_copy(const ForkArgs a) {
  constexpr int kLoads = 8, kRows = kLoads * 32 / (HD / 8);  // positions of a warp's turn
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int layer = blockIdx.y >> 1, heads = a.kv.kv_heads;
  const bool is_v = blockIdx.y & 1;
  uint16_t* pages = is_v ? a.kv.v + layer * a.kv.v_layer : a.kv.k + layer * a.kv.k_layer;
  const int64_t stride = is_v ? a.kv.v_page : a.kv.k_page;
  const uint32_t chunks = (a.kv.page_size + kRows - 1) / kRows;
  const uint32_t items = a.list[0].x * heads * chunks;
  for (uint32_t x = blockIdx.x * (kCopyThreads / 32) + threadIdx.x / 32; x < items;
       x += gridDim.x * (kCopyThreads / 32)) {
    const uint32_t c = x % chunks, ch = x / chunks, head = ch % heads;
    const int4 job = a.list[1 + ch / heads];
    const int from = c * kRows, n = (min(job.z, from + kRows) - from) * (HD / 8);
    if (n <= 0) continue;
    const int64_t in = ((int64_t)head * a.kv.page_size + from) * HD;
    const uint4* src = reinterpret_cast<const uint4*>(pages + job.x * stride + in);
    uint4* dst = reinterpret_cast<uint4*>(pages + job.y * stride + in);
    uint4 r[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (u * 32 + lane < n) r[u] = src[u * 32 + lane];
#pragma unroll
    for (int u = 0; u < kLoads; ++u)
      if (u * 32 + lane < n) dst[u * 32 + lane] = r[u];
  }
}

struct KeepArgs {
  Layers kv;
  int64_t num_pages;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  const int32_t *lengths, *keep;
  int64_t keep_stride;
  int most;                 // entries of a sequence's list
  int parts;                // CTAs of a sequence
  int32_t* new_lengths;
};

constexpr int kKeepThreads = 128, kPieces = 2;

// A thread has kPieces 16-byte pieces of (layer, keys or values, head) rows and
// moves them for every kept node of its sequence: lists rise, so a node's place is
// never read after it was written, and pieces have nothing to do with each other.
// Bound by latency (length and list, pages, rows) and by how many rows are on their way: 64
// sequences x 32 layers x 8 heads of 128 take 2048 CTAs, 8 to an SM at once, 9.6 us; 10.1 without the
// bound on registers, 11.4 with CTAs of 256, 11.4 with one piece a thread.
template <int HD>
__global__ void __launch_bounds__(kKeepThreads, 8) k_keep_nodes(const KeepArgs a) {
  __shared__ int4 s_move[kKeepThreads];  // source page and slot, destination page and slot
  __shared__ int s_warp[32], s_end, s_bad;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, b = blockIdx.x / (uint32_t)a.parts;
  const int part = blockIdx.x - b * a.parts, page = a.kv.page_size;
  const int32_t *list = a.keep + b * a.keep_stride, *table = a.table + b * a.table_stride;
  // The list's start comes with the length, not after it.
  int node = tid < a.most ? list[tid] : -1, node_before = tid > 0 && tid < a.most ? list[tid - 1] : -1;
  const int len = a.lengths[b];
  // This thread's pieces.
  constexpr int kPer = HD / 8;
  const uint16_t* from[kPieces];
  int64_t stride[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int64_t x = ((int64_t)part * kPieces + i) * kKeepThreads + tid, row = x / kPer;
    const int64_t lk = row / a.kv.kv_heads;
    const int head = static_cast<int>(row - lk * a.kv.kv_heads), layer = static_cast<int>(lk >> 1);
    const bool is_v = lk & 1;
    stride[i] = is_v ? a.kv.v_page : a.kv.k_page;
    from[i] = layer >= a.kv.layers ? nullptr
                                   : (is_v ? a.kv.v + layer * a.kv.v_layer : a.kv.k + layer * a.kv.k_layer) +
                                         (int64_t)head * page * HD + x % kPer * 8;
  }
  int kept = 0;
  for (int base_j = 0; len >= 0 && base_j < a.most; base_j += kKeepThreads) {
    if (tid == 0) s_end = s_bad = kKeepThreads;
    const int j = base_j + tid;
    if (base_j > 0) {
      node = j < a.most ? list[j] : -1;
      node_before = j < a.most ? list[j - 1] : -1;
    }
    __syncthreads();
    if (node < 0) atomicMin(&s_end, tid);
    __syncthreads();
    int4 move = make_int4(-1, 0, 0, 0);
    if (tid < s_end) {  // a list that falls or leaves the table ends there
      const int64_t src = (int64_t)len + node, dst = (int64_t)len + j;
      bool ok = node > node_before && src < (int64_t)a.max_pages * page;
      if (ok) {
        move = make_int4(table[src / page], src % page, table[dst / page], dst % page);
        ok = move.x >= 0 && move.x < a.num_pages && move.z >= 0 && move.z < a.num_pages;
      }
      if (!ok) atomicMin(&s_bad, tid);
    }
    __syncthreads();
    if (tid == 0 && part == 0 && s_bad < s_end) set_device_error(kErrPage);
    const int end = min(s_end, s_bad);
    const bool moves = tid < end && node != j;
    int n;
    const int at = block_scan(moves, s_warp, n);
    if (moves) s_move[at] = move;
    __syncthreads();
    kept += end;
    constexpr int kAhead = 4;
    for (int m = 0; m < n; m += kAhead) {
      uint4 r[kPieces][kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (m + u >= n) continue;
        const int4 mv = s_move[m + u];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          if (from[i]) r[i][u] = *reinterpret_cast<const uint4*>(from[i] + mv.x * stride[i] + mv.y * HD);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (m + u >= n) continue;
        const int4 mv = s_move[m + u];
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
          if (from[i])
            *reinterpret_cast<uint4*>(const_cast<uint16_t*>(from[i]) + mv.z * stride[i] + mv.w * HD) = r[i][u];
      }
    }
    __syncthreads();
    if (end < kKeepThreads) break;
  }
  if (part == 0 && tid == 0) a.new_lengths[b] = len + kept;
}

// The cache with its layers; MOE_OK, or what is wrong with it.
int check_layers(const moe_kv_pages_t& c, int64_t layers, int64_t k_layer, int64_t v_layer) {
  if (const int st = check_pages(c); st != MOE_OK) return st;
  if (layers < 1 || layers > 16384 || (layers > 1 && (k_layer < 1 || v_layer < 1)))
    return MOE_ERR_INVALID_ARG;
  if ((k_layer | v_layer) & 7) return MOE_ERR_ALIGNMENT;
  return c.num_pages > INT32_MAX ? MOE_ERR_UNSUPPORTED : MOE_OK;
}
Layers layers_of(const moe_kv_pages_t& c, int64_t layers, int64_t k_layer, int64_t v_layer) {
  return Layers{c.k_pages, c.v_pages, c.k_page_stride, c.v_page_stride, k_layer, v_layer,
                (int)c.page_size, (int)c.kv_heads, (int)layers};
}

constexpr int64_t kListAt = 4096;  // behind the counters that every call leaves zero

bool fork_attr() {
  return cudaFuncSetAttribute(k_fork_tables, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              3 * kMaxRows * 4 + 64 * 1024) == cudaSuccess;
}

template <int HD>
int launch_fork(const ForkArgs& a, cudaStream_t s) {
  if (!once_per_device(reinterpret_cast<const void*>(&fork_attr), &fork_attr)) return MOE_ERR_CUDA;
  const int cols = 1 << a.col_shift;
  // A barrier of 1024 threads costs twice that of 256, and there are a dozen; a large tile
  // wants them all the same (64 rows x 16 columns: 7.0 us with 256, 8.1 with 1024; 256 x 16: 13.6, 10.0).
  const int threads = a.rows * cols <= 2048 && a.entries <= 2 ? 256 : kForkThreads;
  const size_t smem = (size_t)a.rows * 4 * (3 + cols);
  if (launch_pdl(k_fork_tables, dim3((unsigned)ceil_div(a.max_pages, cols)), dim3(threads), smem, s,
                 a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  if (a.entries == 0) return MOE_OK;
  const int slices = 2 * a.kv.layers, per = (8 * sm_count() + slices - 1) / slices;
  if (launch_pdl(k_fork_copy<HD>, dim3(per, slices), dim3(kCopyThreads), 0, s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <int HD>
int launch_keep(const KeepArgs& a, int64_t seqs, cudaStream_t s) {
  if (launch_pdl(k_keep_nodes<HD>, dim3(static_cast<unsigned>(seqs * a.parts)), dim3(kKeepThreads), 0,
                 s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

}  // namespace
}  // namespace moe

extern "C" size_t moe_fork_pages_workspace_size(int64_t rows) {
  return rows < 0 || rows > moe::kMaxRows ? 0 : moe::kListAt + 16 * (rows + 1);
}

extern "C" int moe_fork_pages(const moe_fork_pages_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_fork_pages_args_t& c = *args;
  if (const int st = check_layers(c.kv, c.layers, c.k_layer_stride, c.v_layer_stride); st != MOE_OK)
    return st;
  if (c.room < 0 || c.room > INT32_MAX) return MOE_ERR_INVALID_ARG;
  if (c.kv.seqs > kMaxRows) return MOE_ERR_UNSUPPORTED;
  if (c.kv.seqs == 0 || c.kv.max_pages == 0) return MOE_OK;
  if (!c.kv.block_table || !c.lengths || !c.parents || !c.refs || !c.kv.k_pages || !c.kv.v_pages)
    return MOE_ERR_INVALID_ARG;
  const int hd = static_cast<int>(c.kv.head_dim), chunk = 8 * 32 * 8 / hd;
  if (c.kv.seqs * c.kv.kv_heads > INT32_MAX / ceil_div(c.kv.page_size, chunk))
    return MOE_ERR_UNSUPPORTED;
  if (!c.workspace || c.workspace_bytes < (int64_t)moe_fork_pages_workspace_size(c.kv.seqs))
    return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  ForkArgs a{};
  a.kv = layers_of(c.kv, c.layers, c.k_layer_stride, c.v_layer_stride);
  a.num_pages = c.kv.num_pages;
  a.table = const_cast<int32_t*>(c.kv.block_table);  // the one call that writes it
  a.table_stride = c.kv.table_stride;
  a.rows = static_cast<int>(c.kv.seqs);
  a.max_pages = static_cast<int>(c.kv.max_pages);
  // Columns of a CTA: 32 (a line of memory), fewer where there are many rows or columns.
  a.col_shift = 0;
  while (a.col_shift < 5 && (2 << a.col_shift) * a.rows <= 16384 && (1 << a.col_shift) < a.max_pages)
    ++a.col_shift;
  a.lengths = c.lengths;
  a.parents = c.parents;
  a.refs = c.refs;
  a.room = c.room;
  const int64_t touched = c.room == 0 ? 0 : (c.room + c.kv.page_size - 2) / c.kv.page_size + 1;
  a.entries = static_cast<int>(touched < a.max_pages ? touched : a.max_pages);
  a.done = static_cast<uint32_t*>(c.workspace);
  a.list = reinterpret_cast<int4*>(static_cast<char*>(c.workspace) + kListAt);
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  return hd == 64 ? launch_fork<64>(a, s) : launch_fork<128>(a, s);
}

extern "C" int moe_keep_nodes(const moe_keep_nodes_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_keep_nodes_args_t& c = *args;
  if (const int st = check_layers(c.kv, c.layers, c.k_layer_stride, c.v_layer_stride); st != MOE_OK)
    return st;
  if (c.most < 0 || c.most > (1 << 20) || c.keep_stride < c.most) return MOE_ERR_INVALID_ARG;
  if (c.kv.seqs == 0) return MOE_OK;
  if (!c.lengths || !c.new_lengths || (c.most > 0 && (!c.keep || !c.kv.block_table)) ||
      (c.most > 0 && (!c.kv.k_pages || !c.kv.v_pages)))
    return MOE_ERR_INVALID_ARG;
  // A sequence's CTAs read its length while one of them writes the new one.
  if (overlap(c.lengths, 4 * c.kv.seqs, c.new_lengths, 4 * c.kv.seqs)) return MOE_ERR_INVALID_ARG;
  KeepArgs a{};
  a.kv = layers_of(c.kv, c.layers, c.k_layer_stride, c.v_layer_stride);
  a.num_pages = c.kv.num_pages;
  a.table = c.kv.block_table;
  a.table_stride = c.kv.table_stride;
  a.max_pages = static_cast<int>(c.kv.max_pages);
  a.lengths = c.lengths;
  a.keep = c.keep;
  a.keep_stride = c.keep_stride;
  a.most = static_cast<int>(c.most);
  const int64_t parts = ceil_div(2 * c.layers * c.kv.kv_heads * (c.kv.head_dim / 8),
                                kPieces * kKeepThreads);
  if (parts > INT32_MAX / c.kv.seqs) return MOE_ERR_UNSUPPORTED;
  a.parts = static_cast<int>(c.most > 0 ? parts : 1);
  a.new_lengths = c.new_lengths;
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  return c.kv.head_dim == 64 ? launch_keep<64>(a, c.kv.seqs, s) : launch_keep<128>(a, c.kv.seqs, s);
}
