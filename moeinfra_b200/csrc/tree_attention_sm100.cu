// Attention of a tree of drafted tokens per sequence over its paged keys and
// values, on the 5th-generation tensor cores.
//
//   o[b,t,h] = sum_j softmax_j(scale q[b,t,h] . k_j) v_j
//
// over sequence b's first lengths[b] positions and those of its nodes (position
// lengths[b] + i is node i) that node t sees: bit i of visible[b,t].  Query head h
// reads KV head h / (heads / kv_heads).  A chain of nodes is a chunk of a prompt.
//
// Bound by memory where a KV head's rows (nodes x heads of its group) are fewer
// than what the tensor cores do in the time a key takes to arrive (250 rows), so
// every key is read once for all rows, up to 256, and the keys are cut evenly over
// the GPU whatever the lengths are:
//   * A unit is a (sequence, KV head, block of rows): two tiles of 128 rows at most.
//     Its keys come in steps of 64.  All units' steps form one line, which is cut
//     evenly over persistent CTAs, one to an SM; the cuts are found on the device
//     from the lengths, so a captured graph follows them.
//   * A CTA's pieces run through two pipelines, each with its own rows Q, scores
//     S, probabilities P and result O in tensor memory: both take the same keys
//     where a unit has two tiles; else they take turns, so that one's start and end
//     lie under the other's steps.
//     warps 0-3, 4-7  softmax of pipeline 0 and 1, one thread per row: S -> registers,
//                     maximum, p = 2^(c s - c m), P (16 bits) -> tensor memory
//     warp 8          loads Q, K and V with TMA (no multicast), pages by the table
//     warps 9, 10     tcgen05.mma of pipeline 0 and 1: S = Q K^T, O += P V
//     warp 11         zeros V past a sequence's end in shared memory: what lies in a
//                     page there has no effect
//   * A unit that several CTAs share is joined by the last of them to finish, in the
//     order of its keys; the order of all sums depends on the shapes, the lengths and
//     the GPU only.
//
// O is rescaled only when a row's maximum grew by more than 2^8 since the reference
// in use: probabilities stay below 2^8, O and l are sums of the same factor.
// Every wait is bounded: on a timeout the error word is set, the roles stop, and
// the CTA waits (bounded) for what it issued before it frees its tensor memory.
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

constexpr int kM = 128;        // rows of a tile
constexpr int kN = 64;         // keys of a step
constexpr int kSoftWarps = 8, kTmaWarp = 8, kMmaWarp = 9, kTailWarp = 11;
constexpr int kThreads = 12 * 32;
constexpr int kMaxSeqs = 2048, kMaxNodes = 1024;
constexpr float kLazy = 8.f;   // log2 of what a row's maximum may grow before O is rescaled
// fp16 probabilities, up to 2^kLazy, take 2^7 on top: 2^15 fits, normal down to 2^-21.
template <typename T>
constexpr float prob_shift() { return T::kBf16 ? 0.f : 7.f; }
// Smallest share of a CTA in steps.
constexpr int kMinShare = 2;

template <int HD>
struct Cfg {
  // A tile's 64 dims: rows of 128 bytes, in swizzled groups of 8 (1024 bytes).
  static constexpr int kHalves = HD / 64;
  static constexpr uint32_t kHalfQ = kM * 128, kHalfK = kN * 128;
  static constexpr uint32_t kTileQ = kHalfQ * kHalves, kTileK = kHalfK * kHalves;
  static constexpr int kStages = 8 * 2 / kHalves;  // K and V tiles in flight: 128 KB
  static constexpr uint32_t kRing = kStages * kTileK;
  static constexpr uint32_t smem(int seqs) { return 2 * kTileQ + kRing + 1024 + (3 * seqs + 1) * 4; }
  // TMEM columns of pipeline 0, and how much further pipeline 1's are.
  static constexpr uint32_t kS = 0, kS1 = kN, kP = 2 * kN, kP1 = kN / 2, kO = 3 * kN, kO1 = HD;
  static_assert(kO + 2 * HD <= 512, "TMEM columns");
  // Floats of a piece: O [HD / 4][2 kM rows][4], then m and l per row.
  static constexpr int kPiece = 2 * kM * (HD + 2);
};

struct TreeArgs {
  KvPages kv;
  const uint16_t* q;
  int64_t q_seq, q_node;        // elements from one sequence's (node's) queries to the next
  uint16_t* out;                // [seqs, nodes, heads, HD]
  const int32_t *lengths, *counts;
  const uint64_t* visible;      // [seqs, nodes, words]
  int64_t vis_seq, vis_node;
  int nodes, words, heads, group;
  int parts, tile_heads;        // a group's heads in tiles: parts x tile_heads
  int tokens;                   // nodes of a tile
  int blocks;                   // blocks of rows (two tiles) of a KV head's part
  int per_seq;                  // units of a sequence
  int box;                      // rows of a K or V box: they lie in one page
  float scale_log2;
  uint32_t* counters;           // [CTAs]: pieces written of the unit that starts there; zero between calls
  float* part;                  // [CTAs][2] pieces
  uint64_t wait_ns;
};

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  return mbar_poll_or(bar, parity, limit_ns, [] { set_device_error(kErrWaitTimeout); });
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x,
                                            int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// fp32 accumulate, M = 128; b_rows: B is stored along N (V) instead of K.
template <typename T>
__device__ __forceinline__ uint32_t instr_desc(int n, bool b_rows) {
  const uint32_t ab = T::kBf16 ? ((1u << 7) | (1u << 10)) : 0u;
  return (1u << 4) | ab | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kM >> 4) << 24);
}
// acc + 0 * v for two 16-bit values: NaN once one was infinite or NaN, else +0.
template <typename T>
__device__ __forceinline__ uint32_t trace_odd(uint32_t v, uint32_t acc) {
  if constexpr (T::kBf16)
    asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc) : "r"(v), "r"(0));
  return acc;
}

// What shared memory knows of the sequences: prefix sums of the steps of one
// unit, cached positions, positions with the nodes.
struct Line {
  const int *prefix, *len, *keys;
};

// A CTA's pieces in order: steps [s0, s1) of unit u of sequence b, which has n.
struct Piece {
  int b, u, s0, s1, n;
  int tiles;   // bit t: pipeline t has a tile of it
  int ones;    // pieces of one tile so far: they take the pipelines in turn
  int at, end; // places in the line: this piece's end, the CTA's end

  __device__ __forceinline__ void shape(const TreeArgs& a) {
    s1 = min(n, s0 + end - at);
    at += s1 - s0;
    const int block = u % a.blocks;
    const bool two = a.nodes - block * 2 * a.tokens > a.tokens;
    tiles = two ? 3 : 1 << (ones & 1);
    ones += !two;
  }
  __device__ __forceinline__ bool start(const TreeArgs& a, const Line& line, int lo, int hi) {
    at = lo;
    end = hi;
    ones = 0;
    if (lo >= hi) return false;
    int x = 0, y = a.kv.seqs;  // last b with prefix[b] * per_seq <= lo
    while (y - x > 1) {
      const int mid = (x + y) >> 1;
      if (line.prefix[mid] * a.per_seq <= lo) x = mid;
      else y = mid;
    }
    b = x;
    n = line.prefix[b + 1] - line.prefix[b];
    const int r = lo - line.prefix[b] * a.per_seq;
    u = r / n;
    s0 = r - u * n;
    shape(a);
    return true;
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, const Line& line) {
    if (at >= end) return false;
    s0 = 0;
    if (++u == a.per_seq) {
      u = 0;
      do ++b;
      while (line.prefix[b + 1] == line.prefix[b]);
      n = line.prefix[b + 1] - line.prefix[b];
    }
    shape(a);
    return true;
  }
};

// A row of a unit: its node and head; node < 0: no row.
struct Row {
  int node, head;
};
__device__ __forceinline__ Row row_of(const TreeArgs& a, int u, int second, int r, int have) {
  const int kp = u / a.blocks, block = u - kp * a.blocks;  // KV head and part, block
  const int in = r / a.tile_heads;
  Row w;
  w.node = (block * 2 + second) * a.tokens + in;
  w.head = kp * a.tile_heads + r - in * a.tile_heads;
  if (in >= a.tokens || w.node >= have) w.node = -1;
  return w;
}
// Which of the 64 keys from j0 on a node sees.
__device__ __forceinline__ uint64_t seen_keys(const TreeArgs& a, int b, int node, int len, int keys,
                                              int j0) {
  uint64_t mask = ~0ull;
  const int off = len - j0;  // keys of the cache among them
  if (off < 64) {
    const uint64_t* w = a.visible + b * a.vis_seq + node * a.vis_node;
    const int i0 = off > 0 ? 0 : -off, word = i0 >> 6, sh = i0 & 63;
    mask = word < a.words ? w[word] >> sh : 0;
    if (sh && word + 1 < a.words) mask |= w[word + 1] << (64 - sh);
    if (off > 0) mask = mask << off | ((1ull << off) - 1);
  }
  const int real = keys - j0;
  return real >= 64 ? mask : real <= 0 ? 0 : mask & ((1ull << real) - 1);
}

__device__ __forceinline__ int64_t page_at(const TreeArgs& a, int b, int entry) {
  const int64_t page = entry < a.kv.max_pages ? a.kv.table[b * a.kv.table_stride + entry] : -1;
  if (page >= 0 && page < a.kv.num_pages) return page;
  set_device_error(kErrPage);
  return 0;
}

// One row by the formula, by one warp: 32 keys a step, one to a lane, then the
// values of those that the node sees, HD / 32 dims to a lane.  For rows that met an
// infinity or NaN among the values of a node they do not see (a probability of 0
// does not silence it).  131072 keys take some 10 ms; the other warps' waits end after 2 s.
template <typename T, int HD>
__device__ __noinline__ void redo_row(const TreeArgs& a, int b, int node, int head, int len, int keys) {
  constexpr int kWords = HD / 64;
  const int lane = threadIdx.x & 31, kv_head = head / a.group, page = a.kv.page_size;
  const uint16_t* q = a.q + b * a.q_seq + node * a.q_node + head * HD;
  float m = -INFINITY, l = 0.f;
  float2 acc[kWords] = {};
  for (int j0 = 0; j0 < keys; j0 += 32) {
    const int j = j0 + lane;
    const bool sees = seen_keys(a, b, node, len, keys, j0) >> lane & 1;
    int64_t row_v = 0;
    float s = -INFINITY;
    if (sees) {
      const int64_t p = page_at(a, b, j / page), in = ((int64_t)kv_head * page + j % page) * HD;
      const uint16_t* k = a.kv.k + p * a.kv.k_stride + in;
      row_v = p * a.kv.v_stride + in;
      s = 0.f;
#pragma unroll 4
      for (int d = 0; d < HD; d += 8) {
        const uint4 ks = *reinterpret_cast<const uint4*>(k + d);
        const uint4 qs = *reinterpret_cast<const uint4*>(q + d);
        const uint32_t kw[4] = {ks.x, ks.y, ks.z, ks.w}, qw[4] = {qs.x, qs.y, qs.z, qs.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = T::unpack(qw[i]), y = T::unpack(kw[i]);
          s = fmaf(x.x, y.x, fmaf(x.y, y.y, s));
        }
      }
      s *= a.scale_log2;
    }
    float top = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float nm = fmaxf(m, top), f = m == nm ? 1.f : exp2_approx(m - nm);
    m = nm;
    const float p = exp2_approx(s - (nm == -INFINITY ? 0.f : nm));
    l = l * f + warp_sum(p);
#pragma unroll
    for (int w = 0; w < kWords; ++w) acc[w] = make_float2(acc[w].x * f, acc[w].y * f);
    uint32_t todo = __ballot_sync(0xffffffffu, sees);
    while (todo) {
      const int i = __ffs(todo) - 1;
      todo &= todo - 1;
      const float pi = __shfl_sync(0xffffffffu, p, i);
      const uint16_t* v = a.kv.v + __shfl_sync(0xffffffffu, row_v, i);
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const float2 x = T::unpack(*reinterpret_cast<const uint32_t*>(v + w * 64 + lane * 2));
        acc[w] = make_float2(fmaf(pi, x.x, acc[w].x), fmaf(pi, x.y, acc[w].y));
      }
    }
  }
  const float inv = 1.f / l;
  uint16_t* out = a.out + (((int64_t)b * a.nodes + node) * a.heads + head) * HD;
#pragma unroll
  for (int w = 0; w < kWords; ++w)
    *reinterpret_cast<uint32_t*>(out + w * 64 + lane * 2) = T::pack(acc[w].x * inv, acc[w].y * inv);
}

// A warp's rows whose result is not finite (odd): computed again where a value of a
// node that the row does not see is not.
template <typename T, int HD>
__device__ __noinline__ void mend_rows(const TreeArgs& a, uint32_t odd, int b, Row mine, int len,
                                       int keys) {
  const int lane = threadIdx.x & 31, page = a.kv.page_size;
  __syncwarp();
  while (odd) {
    const int r = __ffs(odd) - 1;
    odd &= odd - 1;
    const int node = __shfl_sync(0xffffffffu, mine.node, r);
    const int head = __shfl_sync(0xffffffffu, mine.head, r);
    uint32_t met = 0;
    for (int j = len; j < keys; ++j) {
      if (seen_keys(a, b, node, len, keys, j) & 1) continue;
      const uint16_t* v = a.kv.v + page_at(a, b, j / page) * a.kv.v_stride +
                          ((int64_t)(head / a.group) * page + j % page) * HD;
#pragma unroll
      for (int w = 0; w < HD / 64; ++w)
        met = trace_odd<T>(*reinterpret_cast<const uint32_t*>(v + w * 64 + lane * 2), met);
    }
    if (__any_sync(0xffffffffu, met)) redo_row<T, HD>(a, b, node, head, len, keys);
  }
}

// 32 columns of a finished row, divided by its sum.  `odd` gathers products: not
// finite once an element is not.
template <typename T>
__device__ __forceinline__ void put_columns(uint16_t* dst, const uint32_t (&o)[32], float inv,
                                            bool blind, float& odd) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[e] = __uint_as_float(o[i + e]);
      odd = fmaf(f[e], 0.f, odd);
      f[e] = blind ? 0.f : f[e] * inv;
    }
    *reinterpret_cast<uint4*>(dst + i) = make_uint4(T::pack(f[0], f[1]), T::pack(f[2], f[3]),
                                                    T::pack(f[4], f[5]), T::pack(f[6], f[7]));
  }
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    k_tree_attention(const __grid_constant__ TreeArgs a, const __grid_constant__ CUtensorMap map_q,
                     const __grid_constant__ CUtensorMap map_k,
                     const __grid_constant__ CUtensorMap map_v) {
  using C = Cfg<HD>;
  constexpr int NS = C::kStages;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t s_qfull[2], s_qempty[2], s_full[NS], s_empty[NS], s_tail[NS],
      s_sfull[2], s_sfree[2], s_pready[2], s_pvdone[2], s_drain[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[kThreads / 32];
  __shared__ int4 s_join[2];
  __shared__ volatile int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (saddr(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_at = base, ring = base + 2 * C::kTileQ;
  int* prefix = reinterpret_cast<int*>(smem_raw + (base - saddr(smem_raw)) + 2 * C::kTileQ + C::kRing);
  int *s_len = prefix + a.kv.seqs + 1, *s_keys = s_len + a.kv.seqs;
  const Line line{prefix, s_len, s_keys};

  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(saddr(&s_qfull[t]), 1);
      mbar_init(saddr(&s_qempty[t]), 1);
      mbar_init(saddr(&s_sfull[t]), 1);
      mbar_init(saddr(&s_sfree[t]), 4);
      mbar_init(saddr(&s_pready[t]), 4);
      mbar_init(saddr(&s_pvdone[t]), 1);
      mbar_init(saddr(&s_drain[t]), 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(saddr(&s_full[i]), 1);
      mbar_init(saddr(&s_empty[i]), 2);
      mbar_init(saddr(&s_tail[i]), 1);
    }
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     saddr(&s_tmem)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_trigger();
  pdl_wait();
  // The line: steps of a unit of each sequence, and their running sum.
  int run = 0;
  const int64_t most = (int64_t)a.kv.max_pages * a.kv.page_size;
  for (int b0 = 0; b0 < a.kv.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    int steps = 0;
    if (b < a.kv.seqs) {
      const int len = a.lengths[b];
      int have = a.counts ? a.counts[b] : a.nodes;
      if (have > a.nodes || (len >= 0 && (int64_t)len + max(have, 0) > most)) {
        if (blockIdx.x == 0) set_device_error(kErrPage);
        have = min(have, a.nodes);
      }
      // No sequence, or none of its nodes are there: nothing to compute.
      const bool none = len < 0 || have <= 0;
      const int keys = none ? 0 : static_cast<int>(min((int64_t)len + have, most));
      s_len[b] = none ? 0 : min(len, keys);
      s_keys[b] = keys;
      steps = (keys + kN - 1) / kN;
    }
    int inc = steps;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int before = run, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += s_scan[w];
      all += s_scan[w];
    }
    if (b < a.kv.seqs) prefix[b] = before + inc - steps;
    run += all;
    __syncthreads();
  }
  if (tid == 0) prefix[a.kv.seqs] = run;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int total = run * a.per_seq;
  const int share = max((int)(((uint32_t)total + gridDim.x - 1) / gridDim.x), kMinShare);
  const int lo = (int)min((int64_t)blockIdx.x * share, (int64_t)total), hi = (int)min((int64_t)lo + share, (int64_t)total);
  // A sequence's nodes that are there: rows of the others are zeros.
  auto have_of = [&](int b) { return min(s_keys[b] - s_len[b], a.nodes); };
  float* parts = a.part + (int64_t)blockIdx.x * 2 * C::kPiece;

  Piece it;
  bool more = it.start(a, line, lo, hi);
  if (warp < kSoftWarps) {
    // ---------------- softmax: one thread per row of pipeline t ----------------
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + C::kS + t * C::kS1 + lane_base;
    const uint32_t p_at = tmem + C::kP + t * C::kP1 + lane_base;
    const uint32_t o_at = tmem + C::kO + t * C::kO1 + lane_base;
    uint32_t n_s = 0, n_pv = 0;  // phases of s_full and pv_done
    bool ok = true;
    for (; more && ok; more = it.next(a, line)) {
      if (!(it.tiles >> t & 1)) continue;
      const int second = it.tiles == 3 ? t : 0, len = s_len[it.b], keys = s_keys[it.b];
      const Row me = row_of(a, it.u, second, row, have_of(it.b));
      const bool idle = !__any_sync(0xffffffffu, me.node >= 0);  // no row of this warp is one
      float m = -INFINITY, l = 0.f;
      for (int j = it.s0; j < it.s1; ++j) {
        if (!(ok = warp_wait(saddr(&s_sfull[t]), n_s++ & 1, a.wait_ns))) break;
        tc_fence_after();
        uint32_t s[kN];
        if (!idle) {
          tmem_ld32(s_at, s);
          tmem_ld32(s_at + 32, s + 32);
          tmem_wait_ld();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_sfree[t]));
        float top = -INFINITY;
        if (!idle) {
          if (j * kN + kN > len) {
            const uint64_t mask = me.node >= 0 ? seen_keys(a, it.b, me.node, len, keys, j * kN) : 0;
            const uint32_t mlo = (uint32_t)mask, mhi = (uint32_t)(mask >> 32);
#pragma unroll
            for (int c = 0; c < 32; ++c) {
              if (!(mlo >> c & 1)) s[c] = 0xff800000u;
              if (!(mhi >> c & 1)) s[c + 32] = 0xff800000u;
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < kN; c += 2)
            mx[c / 2 & 3] = max3(mx[c / 2 & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
          top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
        }
        // P's columns and O are free once the previous product is done.
        if (j > it.s0) {
          if (!(ok = warp_wait(saddr(&s_pvdone[t]), n_pv++ & 1, a.wait_ns))) break;
          tc_fence_after();
        }
        if (!idle) {
          if (__any_sync(0xffffffffu, top > m + (m == -INFINITY ? 0.f : kLazy))) {
            const float nm = fmaxf(m, top);
            const float f = m == nm ? 1.f : exp2_approx(m - nm);
            m = nm;
            l *= f;
            if (j > it.s0) {
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(o_at + c, o);
              }
            }
          }
          const float ref = (m == -INFINITY ? 0.f : m) - prob_shift<T>();
          const uint64_t c2 = pair(a.scale_log2, a.scale_log2), r2 = pair(-ref, -ref);
          uint64_t sum[2] = {0, 0};
          uint32_t p[kN / 2];
#pragma unroll
          for (int c = 0; c < kN; c += 2) {
            const uint64_t x = fma2(pair(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), c2, r2);
            const uint64_t e = pair(exp2_approx(lo_of(x)), exp2_approx(hi_of(x)));
            sum[c / 2 & 1] = add2(sum[c / 2 & 1], e);
            p[c / 2] = T::pack(lo_of(e), hi_of(e));
          }
          tmem_st32(p_at, p);
          tmem_wait_st();
          sum[0] = add2(sum[0], sum[1]);
          l += lo_of(sum[0]) + hi_of(sum[0]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_pready[t]));
      }
      if (ok) ok = warp_wait(saddr(&s_pvdone[t]), n_pv++ & 1, a.wait_ns);
      if (!ok) break;
      tc_fence_after();
      if (!idle) {
        const bool real = me.node >= 0;
        if (it.s0 == 0 && it.s1 == it.n) {
          // The whole unit.  A row without keys is zeros; one with keys has l above 0, unless every
          // score is -inf (0 / 0), and NaN where one is NaN or +inf: the row then is NaN.
          bool blind = false;
          if (real && l == 0.f) {
            blind = len == 0;
            for (int j = 0; j < keys && blind; j += 64)
              blind = seen_keys(a, it.b, me.node, len, keys, j) == 0;
          }
          const float inv = __fdividef(1.f, l);
          uint16_t* dst = a.out + (((int64_t)it.b * a.nodes + max(me.node, 0)) * a.heads + me.head) * HD;
          float odd = 0.f;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_at + c, o);
            tmem_wait_ld();
            if (real) put_columns<T>(dst + c, o, inv, blind, odd);
          }
          const uint32_t again = __ballot_sync(0xffffffffu, real && !blind && odd != 0.f);
          if (again) mend_rows<T, HD>(a, again, it.b, me, len, keys);
        } else {
          // A piece: the unit's start (its end is another CTA's) or what follows it.
          float* dst = parts + (it.s0 == 0 ? C::kPiece : 0);
          const int r = second * kM + row;
#pragma unroll 1
          for (int c = 0; c < HD; c += 32) {
            uint32_t o[32];
            tmem_ld32(o_at + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              reinterpret_cast<uint4*>(dst)[((c + i) / 4) * 2 * kM + r] =
                  make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
          dst[2 * kM * HD + r] = m;
          dst[2 * kM * (HD + 1) + r] = l;
        }
      }
      tc_fence_before();
    }
    if (!ok) s_abort = 1;
  } else if (warp == kTmaWarp) {
    // ---------------- TMA producer ----------------
    // Q, K(0), then K(j + 1), V(j): the order of use.
    uint32_t g = 0, n_q[2] = {0, 0};
    bool ok = true;
    const int boxes = kN / a.box, my_box = lane / C::kHalves, half = lane % C::kHalves;
    // Pages of 32 boxes of the sequence from w_base on, one per lane, and of the 32 after them.
    int w_base = 0, w_page = 0, w_next = 0;
    auto look = [&](int x) -> int {  // the page of box x
      const int j = x * a.box;
      return j < s_keys[it.b] ? (int)page_at(a, it.b, j / a.kv.page_size) : 0;
    };
    int cur_page = 0, cur_y = 0, nxt_page = 0, nxt_y = 0;
    auto find = [&](int j) {  // this lane's box of step j
      const int x = j * boxes + my_box;
      if (j * boxes >= w_base + 32) {
        w_base += 32;
        w_page = w_next;
        w_next = look(w_base + 32 + lane);
      }
      nxt_page = __shfl_sync(0xffffffffu, w_page, (x - w_base) & 31);
      nxt_y = x * a.box % a.kv.page_size;
    };
    auto load = [&](bool is_v, int j, int page, int y, int kv_head) {
      const int s = g % NS;
      ok = ok && warp_wait(saddr(&s_empty[s]), ((g / NS) & 1) ^ 1, a.wait_ns);
      if (__any_sync(0xffffffffu, s_abort)) ok = false;
      if (!ok) return;
      ++g;
      const int rows = s_keys[it.b] - j * kN;
      const int count = min(boxes, (rows + a.box - 1) / a.box);
      const uint32_t bar = saddr(is_v && rows < kN ? &s_tail[s] : &s_full[s]);
      if (lane == 0) mbar_expect_tx(bar, count * a.box * 128 * C::kHalves);
      __syncwarp();
      if (my_box < count)
        tma_load_4d(ring + s * C::kTileK + half * C::kHalfK + my_box * a.box * 128,
                    is_v ? &map_v : &map_k, bar, half * 64, y, kv_head, page);
    };
    for (; more && ok; more = it.next(a, line)) {
      const int kp = it.u / a.blocks, block = it.u - kp * a.blocks, kv_head = kp / a.parts;
      w_base = it.s0 * boxes / 32 * 32;
      w_page = look(w_base + lane);
      w_next = look(w_base + 32 + lane);
      for (int t = 0; t < 2 && ok; ++t) {
        if (!(it.tiles >> t & 1)) continue;
        ok = warp_wait(saddr(&s_qempty[t]), (n_q[t]++ & 1) ^ 1, a.wait_ns);
        if (!ok) break;
        if (lane == 0) {
          const uint32_t bar = saddr(&s_qfull[t]);
          mbar_expect_tx(bar, a.tokens * a.tile_heads * 128 * C::kHalves);
          for (int hf = 0; hf < C::kHalves; ++hf)
            tma_load_4d(q_at + t * C::kTileQ + hf * C::kHalfQ, &map_q, bar, hf * 64, kp * a.tile_heads,
                        (block * 2 + (it.tiles == 3 ? t : 0)) * a.tokens, it.b);
        }
      }
      if (!ok) break;
      find(it.s0);
      cur_page = nxt_page;
      cur_y = nxt_y;
      load(false, it.s0, cur_page, cur_y, kv_head);
      for (int j = it.s0; j < it.s1 && ok; ++j) {
        if (j + 1 < it.s1) {
          find(j + 1);
          load(false, j + 1, nxt_page, nxt_y, kv_head);
        }
        load(true, j, cur_page, cur_y, kv_head);
        cur_page = nxt_page;
        cur_y = nxt_y;
      }
    }
    if (!ok) s_abort = 1;
    // After a timeout copies may be in flight: let them land (a tail's on its own barrier).
    if (!ok && lane == 0) {
      for (uint32_t j = g > (uint32_t)NS ? g - NS : 0; j < g; ++j) {
        const uint32_t bar = saddr(&s_full[j % NS]);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_poll(bar, (j / NS) & 1) && globaltimer_ns() - t0 < 1000000) {}
      }
      for (int t = 0; t < 2; ++t) {
        const uint64_t t0 = globaltimer_ns();
        while (n_q[t] && !mbar_poll(saddr(&s_qfull[t]), (n_q[t] - 1) & 1) &&
               globaltimer_ns() - t0 < 1000000) {}
      }
    }
  } else if (warp == kTailWarp) {
    // ---------------- V past a sequence's end becomes zeros ----------------
    uint32_t g = 0, phases = 0;  // tiles so far; a bit per stage: parity of its next tail
    for (; more; more = it.next(a, line)) {
      g += 2 * (it.s1 - it.s0);
      const int rows = s_keys[it.b] - (it.s1 - 1) * kN;
      if (rows >= kN) continue;
      const uint32_t s = (g - 1) % NS;
      if (!warp_wait(saddr(&s_tail[s]), phases >> s & 1, a.wait_ns)) {
        s_abort = 1;
        break;
      }
      phases ^= 1u << s;
      const uint32_t dst = ring + s * C::kTileK;
      for (int hf = 0; hf < C::kHalves; ++hf)
        for (uint32_t z = rows * 128 + lane * 16; z < C::kHalfK; z += 512)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + hf * C::kHalfK + z),
                       "r"(0)
                       : "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(saddr(&s_full[s]));
    }
  } else {
    // ---------------- MMA issuers: one warp per pipeline ----------------
    // The whole warp walks the loop and one elected lane issues: addresses and
    // descriptors are then uniform over the warp and stay in uniform registers.
    const int t = warp - kMmaWarp;
    const uint32_t d_qk = instr_desc<T>(kN, false), d_pv = instr_desc<T>(HD, true);
    const uint32_t leader = elect_one();
    const uint64_t desc_q = smem_desc(q_at + t * C::kTileQ), desc_k = smem_desc(ring);
    const uint64_t desc_v = smem_desc_mn(ring, C::kHalfK);
    const uint32_t s_col = tmem + C::kS + t * C::kS1, p_col = tmem + C::kP + t * C::kP1;
    const uint32_t o_col = tmem + C::kO + t * C::kO1;
    uint32_t slot = 0, turn = 0;  // of the ring: the next tile, and the parity of its barrier
    uint32_t n_q = 0, n_qk = 0, n_pv = 0;
    bool ok = true;
    auto next = [&]() {  // waits for the ring's next tile and takes its slot
      const uint32_t at = slot;
      ok = ok && warp_wait(saddr(&s_full[slot]), turn, a.wait_ns);
      if (++slot == NS) {
        slot = 0;
        turn ^= 1;
      }
      return at;
    };
    // A slot is released by both warps, by one that uses it after its product.
    for (; more && ok; more = it.next(a, line)) {
      const int steps = __shfl_sync(0xffffffffu, it.s1 - it.s0, 0);
      if (!(__shfl_sync(0xffffffffu, it.tiles, 0) >> t & 1)) {
        for (int i = 0; i < 2 * steps && ok; ++i) {
          const uint32_t at = next();
          if (ok && lane == 0) mbar_arrive(saddr(&s_empty[at]));
        }
        continue;
      }
      ok = warp_wait(saddr(&s_qfull[t]), n_q++ & 1, a.wait_ns);
      for (int j = -1; j < steps && ok; ++j) {  // Q K^T of step j + 1, P V of step j
        if (j + 1 < steps) {
          const uint32_t k = next();
          // S, once the last one is read.
          if (n_qk > 0) ok = ok && warp_wait(saddr(&s_sfree[t]), (n_qk - 1) & 1, a.wait_ns);
          if (!ok) break;
          ++n_qk;
          tc_fence_after();
          const uint64_t kd = desc_k + k * (C::kTileK >> 4);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            tc_mma_if(leader, s_col, desc_q + ((kk / 4 * C::kHalfQ + kk % 4 * 32) >> 4),
                      kd + ((kk / 4 * C::kHalfK + kk % 4 * 32) >> 4), d_qk, kk != 0);
          tc_commit_if(leader, saddr(&s_sfull[t]));
          tc_commit_if(leader, saddr(&s_empty[k]));
          if (j + 2 == steps) tc_commit_if(leader, saddr(&s_qempty[t]));
        }
        if (j < 0) continue;
        const uint32_t v = next();
        ok = ok && warp_wait(saddr(&s_pready[t]), n_pv & 1, a.wait_ns);
        if (!ok) break;
        ++n_pv;
        tc_fence_after();
        const uint64_t vd = desc_v + v * (C::kTileK >> 4);
        tc_mma_ta_if(leader, o_col, p_col, vd, d_pv, j == 0 ? 0 : 1);
#pragma unroll
        for (int kk = 1; kk < kN / 16; ++kk)
          tc_mma_ta_if(leader, o_col, p_col + kk * 8, vd + (kk * 2048 >> 4), d_pv, 1);
        tc_commit_if(leader, saddr(&s_pvdone[t]));
        tc_commit_if(leader, saddr(&s_empty[v]));
      }
    }
    if (!ok) s_abort = 1;
    // After a timeout, wait (bounded) for the MMAs already issued.
    if (__any_sync(0xffffffffu, s_abort)) {
      tc_commit_if(leader, saddr(&s_drain[t]));
      warp_wait(saddr(&s_drain[t]), 0, a.wait_ns);
    }
  }

  // Rows of nodes that are not there: zeros.
  for (int b = blockIdx.x; b < a.kv.seqs; b += gridDim.x) {
    const int row = a.heads * HD / 8;
    uint4* o = reinterpret_cast<uint4*>(a.out) + (int64_t)b * a.nodes * row;
    for (int i = have_of(b) * row + tid; i < a.nodes * row; i += kThreads) o[i] = make_uint4(0, 0, 0, 0);
  }

  tc_fence_before();
  __threadfence();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u)
                 : "memory");
  }
  // ---- join the CTAs' pieces: the last CTA of a unit to get here does it ----
  // A unit is counted at the CTA that holds its start.  Whoever finds the count
  // full sees every piece (each CTA's are fenced before its count) and sets the
  // counter back to zero for the next launch.
  if (tid < 2) {
    int4 job = make_int4(0, 0, 0, 0);  // b, u, first CTA, pieces (0: not the last)
    Piece p;
    if (lo < hi) {
      // 0: the unit that the CTA's first step belongs to; 1: that of its last.
      p.start(a, line, tid ? hi - 1 : lo, hi);
      const int from = prefix[p.b] * a.per_seq + p.u * p.n, to = from + p.n;
      const int c0 = from / share, pieces = (to - 1) / share - c0 + 1;
      // One unit over the whole CTA is counted once.
      const bool mine = pieces > 1 && (tid == 0 ? from < lo || to > hi : from > lo);
      if (mine && atomicAdd(a.counters + c0, 1) == (uint32_t)pieces - 1) {
        a.counters[c0] = 0;
        job = make_int4(p.b, p.u, c0, pieces);
      }
    }
    s_join[tid] = job;
  }
  __syncthreads();
  if (warp >= kSoftWarps) return;
  for (int w = 0; w < 2; ++w) {
    const int4 job = s_join[w];
    if (job.w == 0 || s_abort) continue;
    __threadfence();
    const int second = warp >> 2, row = (warp & 3) * 32 + lane, r = second * kM + row;
    const int len = s_len[job.x], keys = s_keys[job.x];
    const Row me = row_of(a, job.y, second, row, have_of(job.x));
    const bool real = me.node >= 0;
    if (!__any_sync(0xffffffffu, real)) continue;
    // Piece 0 is CTA c0's second, the others the first of the CTAs after it.
    const float* first = a.part + (int64_t)job.z * 2 * C::kPiece;
    auto piece = [&](int k) { return first + (int64_t)(k == 0 ? 1 : 2 * k) * C::kPiece; };
    float m = -INFINITY, l = 0.f;
    for (int k = 0; k < job.w; ++k) m = fmaxf(m, __ldcg(piece(k) + 2 * kM * HD + r));
    auto factor = [&](int k) {
      const float mk = __ldcg(piece(k) + 2 * kM * HD + r);
      return mk == m ? 1.f : exp2_approx(mk - m);
    };
    for (int k = 0; k < job.w; ++k) l += factor(k) * __ldcg(piece(k) + 2 * kM * (HD + 1) + r);
    bool blind = false;
    if (real && l == 0.f) {
      blind = len == 0;
      for (int j = 0; j < keys && blind; j += 64) blind = seen_keys(a, job.x, me.node, len, keys, j) == 0;
    }
    const float inv = __fdividef(1.f, l);
    uint16_t* dst = a.out + (((int64_t)job.x * a.nodes + max(me.node, 0)) * a.heads + me.head) * HD;
    float odd = 0.f;
#pragma unroll 1
    for (int c = 0; c < HD; c += 32) {
      float acc[32] = {};
#pragma unroll 1
      for (int k = 0; k < job.w; ++k) {
        const float f = factor(k);
        const float4* src = reinterpret_cast<const float4*>(piece(k)) + (c / 4) * 2 * kM + r;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 x = __ldcg(src + i * 2 * kM);
          acc[4 * i] += f * x.x;
          acc[4 * i + 1] += f * x.y;
          acc[4 * i + 2] += f * x.z;
          acc[4 * i + 3] += f * x.w;
        }
      }
      uint32_t o[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(acc[i]);
      if (real) put_columns<T>(dst + c, o, inv, blind, odd);
    }
    const uint32_t again = __ballot_sync(0xffffffffu, real && !blind && odd != 0.f);
    if (again) mend_rows<T, HD>(a, again, job.x, me, len, keys);
  }
}

// Four dimensions, boxes of box[1] x box[2] rows of 64 elements, 128-byte swizzle.
bool make_map(CUtensorMap* map, const uint16_t* x, bool bf16, const cuuint64_t (&dims)[4],
              const int64_t (&stride)[3], const cuuint32_t (&box)[4]) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t strides[3] = {(cuuint64_t)stride[0] * 2, (cuuint64_t)stride[1] * 2,
                                 (cuuint64_t)stride[2] * 2};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<uint16_t*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
bool tree_attr() {
  return cudaFuncSetAttribute(k_tree_attention<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Cfg<HD>::smem(kMaxSeqs)) == cudaSuccess;
}

template <typename T, int HD>
int launch_tree(const TreeArgs& a, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v,
                int grid, cudaStream_t s) {
  if (!once_per_device(reinterpret_cast<const void*>(&tree_attr<T, HD>), &tree_attr<T, HD>))
    return MOE_ERR_CUDA;
  if (launch_pdl(k_tree_attention<T, HD>, dim3(grid), dim3(kThreads), Cfg<HD>::smem(a.kv.seqs), s, a, q,
                 k, v) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

constexpr int64_t kPartAt = 4096;  // behind the counters that every call leaves zero

}  // namespace
}  // namespace moe

extern "C" size_t moe_tree_attention_workspace_size(int64_t head_dim) {
  using namespace moe;
  if (head_dim != 64 && head_dim != 128) return 0;
  return kPartAt + (size_t)sm_count() * 2 * 4 * (head_dim == 64 ? Cfg<64>::kPiece : Cfg<128>::kPiece);
}

extern "C" int moe_tree_attention(const moe_tree_attention_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_tree_attention_args_t& c = *args;
  if (const int st = check_pages(c.kv); st != MOE_OK) return st;
  const int64_t hd = c.kv.head_dim;
  const float scale = static_cast<float>(c.scale);
  if (c.heads < 1 || c.heads > 4096 || c.heads % c.kv.kv_heads || c.nodes < 0 ||
      !(scale > 0.f && scale < INFINITY) || c.q_node_stride < c.heads * hd || c.q_seq_stride < 0 ||
      (c.kv.seqs > 1 && c.q_seq_stride < c.heads * hd) || c.visible_seq_stride < 0 ||
      c.visible_node_stride < 0)
    return MOE_ERR_INVALID_ARG;
  if (c.kv.page_size % 16 || c.kv.seqs > kMaxSeqs || c.nodes > kMaxNodes || c.kv.num_pages > INT32_MAX)
    return MOE_ERR_UNSUPPORTED;
  if (c.kv.seqs == 0 || c.nodes == 0) return MOE_OK;
  if (!c.q || !c.lengths || !c.visible || !c.out ||
      (c.kv.max_pages > 0 &&
       (!c.kv.k_pages || !c.kv.v_pages || !c.kv.block_table || c.kv.num_pages < 1)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(c.q) || !aligned16(c.out) || ((c.q_seq_stride | c.q_node_stride) & 7) ||
      (reinterpret_cast<uintptr_t>(c.visible) & 7))
    return MOE_ERR_ALIGNMENT;
  TreeArgs a{};
  a.kv = pages_of(c.kv);
  a.q = c.q;
  a.q_seq = c.q_seq_stride;
  a.q_node = c.q_node_stride;
  a.out = c.out;
  a.lengths = c.lengths;
  a.counts = c.counts;
  a.visible = reinterpret_cast<const uint64_t*>(c.visible);
  a.vis_seq = c.visible_seq_stride;
  a.vis_node = c.visible_node_stride;
  a.nodes = static_cast<int>(c.nodes);
  a.words = (a.nodes + 63) / 64;
  a.heads = static_cast<int>(c.heads);
  a.group = a.heads / a.kv.kv_heads;
  // A tile's rows are the heads of a group for neighbouring nodes; a group above 128
  // heads is cut.
  a.parts = (a.group + kM - 1) / kM;
  while (a.group % a.parts) ++a.parts;
  a.tile_heads = a.group / a.parts;
  a.tokens = kM / a.tile_heads;
  a.blocks = (a.nodes + 2 * a.tokens - 1) / (2 * a.tokens);
  const int64_t per_seq = (int64_t)a.kv.kv_heads * a.parts * a.blocks;
  const int64_t steps = ceil_div(c.kv.max_pages * c.kv.page_size, kN);
  if (per_seq > INT32_MAX || c.kv.seqs * per_seq > INT32_MAX / (steps > 0 ? steps : 1) - 4096)
    return MOE_ERR_UNSUPPORTED;
  a.per_seq = static_cast<int>(per_seq);
  a.box = 16;
  while (a.box < kN && a.kv.page_size % (2 * a.box) == 0) a.box *= 2;
  a.scale_log2 = scale * 1.4426950408889634f;
  const size_t need = moe_tree_attention_workspace_size(hd);
  if (!c.workspace || c.workspace_bytes < (int64_t)need) return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  a.counters = static_cast<uint32_t*>(c.workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + kPartAt);
  a.wait_ns = wait_limit_ns();
  const bool bf16 = c.kv.dtype == MOE_DTYPE_BF16;
  const bool none = c.kv.max_pages == 0;  // no keys at all: the maps describe q
  CUtensorMap mq, mk, mv;
  const cuuint64_t q_dims[4] = {(cuuint64_t)hd, (cuuint64_t)c.heads, (cuuint64_t)c.nodes,
                                (cuuint64_t)c.kv.seqs};
  const int64_t q_strides[3] = {hd, c.q_node_stride, c.kv.seqs > 1 ? c.q_seq_stride : c.q_node_stride * c.nodes};
  const cuuint32_t q_box[4] = {64, (cuuint32_t)a.tile_heads, (cuuint32_t)a.tokens, 1};
  const cuuint64_t kv_dims[4] = {(cuuint64_t)hd, (cuuint64_t)c.kv.page_size, (cuuint64_t)c.kv.kv_heads,
                                 (cuuint64_t)c.kv.num_pages};
  const int64_t in_page = c.kv.page_size * hd, whole = in_page * c.kv.kv_heads;
  const cuuint32_t kv_box[4] = {64, (cuuint32_t)a.box, 1, 1};
  auto kv_map = [&](CUtensorMap* m, const uint16_t* x, int64_t page_stride) {
    if (none) return make_map(m, c.q, bf16, q_dims, q_strides, q_box);
    return make_map(m, x, bf16, kv_dims, {hd, in_page, c.kv.num_pages > 1 ? page_stride : whole}, kv_box);
  };
  if (!make_map(&mq, c.q, bf16, q_dims, q_strides, q_box) ||
      !kv_map(&mk, c.kv.k_pages, c.kv.k_page_stride) || !kv_map(&mv, c.kv.v_pages, c.kv.v_page_stride))
    return MOE_ERR_CUDA;
  const int64_t line = c.kv.seqs * per_seq * steps, most = ceil_div(line, kMinShare);
  const int sms = sm_count(), grid = static_cast<int>(most < 1 ? 1 : most < sms ? most : sms);
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (bf16)
    return hd == 64 ? launch_tree<BF16, 64>(a, mq, mk, mv, grid, s)
                    : launch_tree<BF16, 128>(a, mq, mk, mv, grid, s);
  return hd == 64 ? launch_tree<F16, 64>(a, mq, mk, mv, grid, s)
                  : launch_tree<F16, 128>(a, mq, mk, mv, grid, s);
}
