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
//   * A CTA's pieces run through two pipelines, each with its own scores S (two buffers, in
//     which the probabilities P take their place) and result O in tensor memory.  Where a unit has
//     two tiles, each has one of them and both take the same keys; a single tile they
//     share, one taking the even and one the odd steps, and join their results at the end.
//     warps 0-3, 4-7  softmax of pipeline 0 and 1, one thread per row: S -> registers,
//                     maximum, p = 2^(c s - c m), P (16 bits) -> tensor memory
//     warps 8, 11     load Q and K, and V, with TMA (no multicast), pages by the table;
//                     V past a sequence's end becomes zeros in shared memory: what lies
//                     in a page there has no effect
//     warps 9, 10     tcgen05.mma of pipeline 0 and 1: S = Q K^T, O += P V
//   * What CTAs hold of a unit that is cut is joined by a second kernel, in the order of
//     its keys; the order of all sums depends on the shapes, the lengths and the GPU only.
//     Short units are not cut: a few have a CTA each, of many the line is cut between them.
//   * Keys and values stand in one ring in the order of their use, and both MMA warps walk it tile
//     by tile: a barrier's parity tells one phase from the next only.  The keys are ahead of the
//     values by a step of a pipeline's own, so that its next scores are on their way during a softmax.
// Small trees (16 rows to a KV head) go to a kernel without tensor memory: tree_attention_few.cu.
//
// Measured in a graph (32 / 8 heads of 128, both kernels): 8 nodes over 64 x 512..640 fp16 44 us
// (165 MB, 3.7 TB/s: a unit's 9 steps stream at a copy's rate, its end and the next one's start do
// not; the join 4 us); 64 nodes over 16 x 2049..4095 bf16 70 us (shared memory: Q K^T reads 6 KB
// for 32 cycles of products, 1280 of a step's 1640 cycles; 38 MB of pieces of cut units); 27 nodes
// over 131071 + 85413 bf16 148 to 156 us from one GPU to another (888 MB, 5.7 to 6.0 TB/s); 16 nodes
// over 72 9.8 us, a chain of latencies.
//
// O is rescaled only when a row's maximum grew by more than 2^8 since the reference
// in use: probabilities stay below 2^8, O and l are sums of the same factor.
// Every wait is bounded: on a timeout the error word is set, the roles stop, and
// the CTA waits (bounded) for what it issued before it frees its tensor memory.
#include <algorithm>

#include "sm100_ptx.cuh"
#include "tree.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

constexpr int kM = 128;        // rows of a tile
constexpr int kN = 64;         // keys of a step
constexpr int kSoftWarps = 8, kKeyWarp = 8, kMmaWarp = 9, kValueWarp = 11;
constexpr int kThreads = 12 * 32;
// Registers a thread: 12 warps x 168 at launch, of which the softmax warps take kSoftRegs and
// the others keep kOtherRegs.
constexpr int kSoftRegs = 200, kOtherRegs = 104;
constexpr int kRegs = 2 * 128 * kSoftRegs + 128 * kOtherRegs;
constexpr int kMaxSeqs = 2048, kMaxNodes = 1024;
constexpr float kLazy = 8.f;   // log2 of what a row's maximum may grow before O is rescaled
// fp16 probabilities, up to 2^kLazy, take 2^7 on top: 2^15 fits, normal down to 2^-21.
template <typename T>
constexpr float prob_shift() { return T::kBf16 ? 0.f : 7.f; }
// Places of a unit's start, in steps: what it takes to begin and end one.  8 nodes over 1 x 600 keys
// 12.4 us with 2, 13.1 with 3, 14.4 with 5, 15.1 with 7; over 1 x 4000 16.6, 15.4, 16.0, 16.5; 64
// nodes over 16 x 2049..4095 72.2, 71.6, 72.0, 73.1.
constexpr int kStart = 3;
// Smallest share of a CTA in steps: 16 nodes over 1 x 72 11.1 us with 1, 10.3 with 2, 13.5 with 3.
constexpr int kMinShare = 2;
// Steps of a table up to which units have CTAs of their own, where the GPU has as many: nothing is
// joined then.  More where there are many units (own CTAs / even cut, us): 8 units, 16 nodes over 72
// 9.5 / 10.4, over 300 11.4 / 13.1, over 400 12.7 / 13.2, over 600 14.5 / 13.4, over 1000 18.8 / 13.4;
// 64 units, 8 nodes over 600 14.6 / 17.2, over 1000 18.6 / 18.9; 128 units, 64 nodes over 250..1000
// 29.6 / 34.8.
constexpr int64_t kWholeSteps = 6;
// And up to which the line is cut between units where there are more (8 nodes, between / anywhere):
// 64 x 160..200 26.9 / 31.6, 64 x 320..400 36.0 / 37.5, 64 x 8..200 25.2 / 27.3; but 64 x 512..640
// 44.4 / 44.4, 64 x 720..900 54.6 / 51.2, 20 x 512..640 25.0 / 23.2.
constexpr int kBetweenSteps = 8;

template <int HD>
struct Cfg {
  // 64 dims of a row are 128 bytes, 8 rows of them a swizzled atom of 1024 bytes.  A tile of Q has its
  // first 64 dims' atoms first, a tile of keys or values those of 8 keys together (kGroup bytes): a
  // box of any number of keys lies in one piece, one load.
  static constexpr int kHalves = HD / 64;
  static constexpr uint32_t kHalfQ = kM * 128, kGroup = 1024 * kHalves;
  static constexpr uint32_t kTileQ = kHalfQ * kHalves, kTileK = kN / 8 * kGroup;
  static constexpr int kStages = 8 * 2 / kHalves;  // K and V tiles in flight: 128 KB
  static constexpr uint32_t kRing = kStages * kTileK;
  // On its way out a softmax warp's result passes 32 rows x 64 bytes of shared memory.
  static constexpr uint32_t kOut = 32 * 64;
  static constexpr uint32_t smem(int seqs) {
    return 2 * kTileQ + kRing + kSoftWarps * kOut + 1024 + (seqs + 1) * 4;
  }
  // TMEM columns of pipeline 0, and how much further pipeline 1's are.  S has two buffers, and
  // P takes its step's S's place: the next step's S is computed while this one's softmax runs.
  static constexpr uint32_t kS = 0, kS1 = 2 * kN, kO = 4 * kN, kO1 = HD;
  static_assert(kO + 2 * HD <= 512, "TMEM columns");
  // Floats of a piece: O [kM / 16 warps of 32 rows][HD / 4][32 rows][4], then m and l per row.
  static constexpr int kPiece = 2 * kM * (HD + 2);
};

struct TreeArgs : TreeRows {
  int parts, tile_heads;        // a group's heads in tiles: parts x tile_heads
  int tokens;                   // nodes of a tile
  int blocks;                   // blocks of rows (two tiles) of a KV head's part
  int per_seq;                  // units of a sequence
  bool whole, between;          // a CTA has one unit; the line is cut between units: then none is cut
  int box, box_shift;           // rows of a K or V box, which lie in one page, and their log2
  int page_shift;               // log2 of a page's boxes, or -1
  int4* jobs;                   // [CTAs]: sequence, unit, CTAs and nodes of the cut unit that starts there
  float* part;                  // [CTAs][2] pieces: 0 of a unit that starts before, 1 of one that goes on
  uint64_t wait_ns;
};

// A whole warp's wait, with one result for all lanes.  After a first look the warp sleeps in
// hardware: with twelve warps to four schedulers those that poll slow down those that work.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  if (__all_sync(0xffffffffu, mbar_poll(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait_or(bar, parity, limit_ns, [] { set_device_error(kErrWaitTimeout); }));
}
// For a warp that runs it as a whole, with the same operands in every lane: issued by
// the lane with leader != 0.  Operands that differ between lanes make each load some 150
// cycles.
__device__ __forceinline__ void tma_load_4d_if(uint32_t leader, uint32_t dst, const CUtensorMap* map,
                                               uint32_t bar, int x, int y, int z, int w) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %7, 0;\n"
      " @q cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5, %6}], [%2];\n}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tma_load_5d_if(uint32_t leader, uint32_t dst, const CUtensorMap* map,
                                               uint32_t bar, int w, int v) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %5, 0;\n"
      " @q cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%6, %6, %6, %3, %4}], [%2];\n}\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(w), "r"(v), "r"(leader), "r"(0)
      : "memory");
}
__device__ __forceinline__ void mbar_expect_tx_if(uint32_t leader, uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
      " @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}\n" ::"r"(bar),
      "r"(bytes), "r"(leader)
      : "memory");
}
// fp32 accumulate, M = 128; b_rows: B is stored along N (V) instead of K.
template <typename T>
__device__ __forceinline__ uint32_t instr_desc(int n, bool b_rows) {
  const uint32_t ab = T::kBf16 ? ((1u << 7) | (1u << 10)) : 0u;
  return (1u << 4) | ab | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kM >> 4) << 24);
}
// A CTA's pieces in order: steps [s0, s1) of unit u of sequence b, which has n.  In the
// line a unit has kStart places before its steps: what it costs to begin and end one.
struct Piece {
  int b, u, s0, s1, n;
  int left, end;  // places from the unit's first step to the CTA's first and last (excluded)

  // The unit that place x lies in; left, end: the CTA's places.
  __device__ __forceinline__ void find(const TreeArgs& a, const int* prefix, int x, int lo, int hi) {
    int low = 0, y = a.kv.seqs;  // last b with prefix[b] * per_seq <= x
    while (y - low > 1) {
      const int mid = (low + y) >> 1;
      if (prefix[mid] * a.per_seq <= x) low = mid;
      else y = mid;
    }
    b = low;
    n = prefix[b + 1] - prefix[b] - kStart;
    const int r = x - prefix[b] * a.per_seq;
    u = r / (n + kStart);
    const int first = x - r + u * (n + kStart) + kStart;
    left = lo - first;
    end = hi - first;
  }
  // The place between units that is nearest to place x.
  static __device__ __forceinline__ int between(const TreeArgs& a, const int* prefix, int x, int total) {
    if (x >= total) return total;
    Piece p;
    p.find(a, prefix, x, x, x);
    const int places = p.n + kStart, in = p.left + kStart;
    return x - in + (2 * in >= places ? places : 0);
  }
  __device__ __forceinline__ bool cut() {  // false: the CTA has no step of the unit
    s0 = max(left, 0);
    s1 = min(n, end);
    return s0 < s1;
  }
  __device__ __forceinline__ bool start(const TreeArgs& a, const int* prefix, int lo, int hi) {
    if (lo >= hi) return false;
    find(a, prefix, lo, lo, hi);
    return cut() || next(a, prefix);
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, const int* prefix) {
    left -= n + kStart;
    end -= n + kStart;
    if (end <= 0) return false;
    if (++u == a.per_seq) {
      u = 0;
      do ++b;
      while (prefix[b + 1] == prefix[b]);
      n = prefix[b + 1] - prefix[b] - kStart;
    }
    return cut();
  }
};

// A piece as the first producer describes it to the other warps.
struct __align__(16) Item {
  int b, node0, head0, len;  // sequence, the unit's first node and head, cached positions
  int keys, s0, steps;       // positions with the nodes; first step, number of steps (0: no more items)
  int flags;                 // kTwo, kFirst, kLast, Q buffer << 3 (of a single tile), KV head << 8

  // Of a shared tile, pipeline t takes every second step from its t-th on.
  __device__ __forceinline__ int steps_of(int t) const { return flags & 1 ? steps : (steps + 1 - t) >> 1; }
};
constexpr int kTwo = 1;    // two tiles of rows, one to a pipeline; else the pipelines share one
constexpr int kFirst = 2;  // the unit starts with this piece
constexpr int kLast = 4;   // and ends with it
constexpr int kItems = 4;  // described ahead
constexpr int kReaders = 11;
// How many steps a piece's keys are ahead of its values: one of a pipeline's own, so that its next
// scores are on their way during a softmax.
__device__ __forceinline__ int lead_of(bool two) { return two ? 1 : 2; }

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

// By a softmax warp of pipeline t that has written a result which is not finite, once all of the
// CTA's pieces are done: looks at its rows of the whole units again and mends them.  It may take longer
// than a wait is allowed to, and nobody waits for the warp any more.
template <typename T, int HD>
__device__ __noinline__ void mend_units(const TreeArgs& a, const int* prefix, int t, int quad) {
  const int lane = threadIdx.x & 31;
  const uint32_t inf = T::kBf16 ? 0x7F80u : 0x7C00u;
  // The CTA's places, as the kernel finds them (one function for both costs it up to 1 %).
  const int total = prefix[a.kv.seqs] * a.per_seq;
  const int share = max((int)(((uint32_t)total + gridDim.x - 1) / gridDim.x), kMinShare + kStart);
  int lo = (int)min((int64_t)blockIdx.x * share, (int64_t)total), hi = (int)min((int64_t)lo + share, (int64_t)total);
  if (a.whole) {
    const int b = blockIdx.x / (uint32_t)a.per_seq, u = blockIdx.x - b * a.per_seq;
    lo = prefix[b] * a.per_seq + u * (prefix[b + 1] - prefix[b]);
    hi = lo + prefix[b + 1] - prefix[b];
  }
  if (a.between) {
    lo = Piece::between(a, prefix, lo, total);
    hi = Piece::between(a, prefix, hi, total);
  }
  __syncwarp();  // the lanes have written one another's rows
  Piece pc;
  for (bool more = pc.start(a, prefix, lo, hi); more; more = pc.next(a, prefix)) {
    if (pc.s0 > 0 || pc.s1 < pc.n) continue;  // joined, and mended there
    int len, keys;
    span(a, pc.b, len, keys);
    const int block = a.blocks == 1 ? 0 : pc.u % a.blocks;
    const bool two = a.nodes - block * 2 * a.tokens > a.tokens;
    const int from = two ? 0 : t * (HD / 2), to = two ? HD : from + HD / 2;
    const Row me = row_of(a, pc.u, two ? t : 0, quad * 32 + lane, keys - len);
    bool odd = false;
    if (me.node >= 0) {
      const uint4* o = reinterpret_cast<const uint4*>(
          a.out + (((int64_t)pc.b * a.nodes + me.node) * a.heads + me.head) * HD);
#pragma unroll 1
      for (int c = from / 8; c < to / 8; ++c) {
        const uint4 x = o[c];
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) odd |= (w[i] & inf) == inf || (w[i] >> 16 & inf) == inf;
      }
    }
    for (uint32_t again = __ballot_sync(0xffffffffu, odd); again; again &= again - 1) {
      const int r = __ffs(again) - 1;
      mend_row<T, HD>(a, pc.b, __shfl_sync(0xffffffffu, me.node, r), __shfl_sync(0xffffffffu, me.head, r),
                      len, keys, from, to);
    }
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
  __shared__ __align__(8) uint64_t s_qfull[2], s_qempty[2], s_full[NS], s_empty[NS], s_tail,
      s_sfull[2][2], s_pready[2][2], s_pvdone[2][2], s_drain[2], s_done[kSoftWarps],
      s_read[kSoftWarps], s_itfull[kItems], s_itempty[kItems];
  __shared__ Item s_item[kItems];
  __shared__ float2 s_ml[kSoftWarps][32];  // a shared tile's rows: maximum and sum of each pipeline
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[kThreads / 32];
  __shared__ volatile int s_abort;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (saddr(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_at = base, ring = base + 2 * C::kTileQ;
  // Prefix sums of the steps of a unit of each sequence.
  int* prefix = reinterpret_cast<int*>(smem_raw + (base - saddr(smem_raw)) + 2 * C::kTileQ + C::kRing +
                                       kSoftWarps * C::kOut);

  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(saddr(&s_qfull[t]), 1);
      mbar_init(saddr(&s_qempty[t]), 2);
      for (int i = 0; i < 2; ++i) {
        mbar_init(saddr(&s_sfull[t][i]), 1);
        mbar_init(saddr(&s_pready[t][i]), 4);
        mbar_init(saddr(&s_pvdone[t][i]), 1);
      }
      mbar_init(saddr(&s_drain[t]), 1);
    }
    for (int w = 0; w < kSoftWarps; ++w) {
      mbar_init(saddr(&s_done[w]), 1);
      mbar_init(saddr(&s_read[w]), 1);
    }
    mbar_init(saddr(&s_tail), 1);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(saddr(&s_itfull[i]), 1);
      mbar_init(saddr(&s_itempty[i]), kReaders);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(saddr(&s_full[i]), 1);
      mbar_init(saddr(&s_empty[i]), 2);
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
  for (int b0 = 0; b0 < a.kv.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    int steps = 0;
    if (b < a.kv.seqs) {
      int len, keys;
      if (!span(a, b, len, keys) && blockIdx.x == 0) set_device_error(kErrPage);
      steps = (keys + kN - 1) / kN;
    }
    const int places = steps > 0 ? steps + kStart : 0;
    int inc = places;
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
    if (b < a.kv.seqs) prefix[b] = before + inc - places;
    run += all;
    __syncthreads();
  }
  if (tid == 0) prefix[a.kv.seqs] = run;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int total = run * a.per_seq;
  const int share = max((int)(((uint32_t)total + gridDim.x - 1) / gridDim.x), kMinShare + kStart);
  int lo = (int)min((int64_t)blockIdx.x * share, (int64_t)total), hi = (int)min((int64_t)lo + share, (int64_t)total);
  if (a.whole) {  // the unit that the CTA has to itself
    const int b = blockIdx.x / (uint32_t)a.per_seq, u = blockIdx.x - b * a.per_seq;
    const int places = prefix[b + 1] - prefix[b];
    lo = prefix[b] * a.per_seq + u * places;
    hi = lo + places;
  }

  // The next item; false at the end or after a timeout (then ok is false).
  uint32_t n_it = 0;
  bool ok = true;
  auto next_item = [&](Item& it) {
    const uint32_t i = n_it % kItems;
    ok = warp_wait(saddr(&s_itfull[i]), n_it / kItems & 1, a.wait_ns);
    if (!ok) return false;
    it = s_item[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(saddr(&s_itempty[i]));
    ++n_it;
    return it.steps > 0;
  };
  // P V of a pipeline's step n, counted from the first.
  const int t = warp < kSoftWarps ? warp >> 2 : warp - kMmaWarp;  // the pipeline, of softmax and MMA warps
  auto product_done = [&](uint32_t n) {
    return warp_wait(saddr(&s_pvdone[t][n & 1]), n >> 1 & 1, a.wait_ns);
  };
  if (warp < kSoftWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // ---------------- softmax: one thread per row of pipeline t ----------------
    const int row = (warp & 3) * 32 + lane, pal = warp ^ 4;  // pal: the same rows' other warp
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + C::kS + t * C::kS1 + lane_base;
    const uint32_t o_at = tmem + C::kO + t * C::kO1 + lane_base;
    const uint32_t o_pal = tmem + C::kO + (1 - t) * C::kO1 + lane_base;
    const int row_node = row / a.tile_heads, row_head = row - row_node * a.tile_heads;
    uint32_t n_s = 0, n_pair = 0;  // steps and shared tiles so far
    bool mend = false;  // a row has met an infinity or NaN
    for (Item it; next_item(it);) {
      const bool two = it.flags & kTwo;
      const int second = two ? t : 0;
      Row me{it.node0 + second * a.tokens + row_node, it.head0 + row_head};
      if (row_node >= a.tokens || me.node >= it.keys - it.len) me.node = -1;
      const bool real = me.node >= 0;
      const bool idle = !__any_sync(0xffffffffu, real);  // no row of this warp is one
      const int mine = it.steps_of(t);
      uint64_t sees = 0;  // trees of up to 64 nodes: the row's mask
      if (real && a.words == 1) sees = a.visible[it.b * a.vis_seq + me.node * a.vis_node];
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < mine; ++i, ++n_s) {
        const int j0 = (it.s0 + (two ? i : 2 * i + t)) * kN;
        if (!(ok = warp_wait(saddr(&s_sfull[t][n_s & 1]), n_s >> 1 & 1, a.wait_ns))) break;
        tc_fence_after();
        if (!idle) {
          const uint32_t sp = s_at + (n_s & 1) * kN;
          uint32_t s[kN];
          tmem_ld32(sp, s);
          tmem_ld32(sp + 32, s + 32);
          tmem_wait_ld();
          if (j0 + kN > it.len) {
            const uint64_t mask = a.words == 1 ? seen_keys(sees, it.len, it.keys, j0)
                                  : real ? seen_keys(a, it.b, me.node, it.len, it.keys, j0) : 0;
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
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
          if (__any_sync(0xffffffffu, top > m + (m == -INFINITY ? 0.f : kLazy))) {
            const float nm = fmaxf(m, top);
            const float f = m == nm ? 1.f : exp2_approx(m - nm);
            m = nm;
            l *= f;
            if (i > 0) {
              if (!(ok = product_done(n_s - 1))) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                tmem_ld32(o_at + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
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
            const uint64_t e = exp2_mufu(x);
            sum[c / 2 & 1] = add2(sum[c / 2 & 1], e);
            p[c / 2] = T::pack(lo_of(e), hi_of(e));
          }
          tmem_st32(sp, p);
          tmem_wait_st();
          sum[0] = add2(sum[0], sum[1]);
          l += lo_of(sum[0]) + hi_of(sum[0]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_pready[t][n_s & 1]));
      }
      // The last two products; a barrier's next phase needs a P of the next piece.
      if (ok && mine > 1) ok = product_done(n_s - 2);
      if (ok && mine > 0) ok = product_done(n_s - 1);
      if (!ok) break;
      tc_fence_after();
      if (idle) continue;
      // A tile of one's own, or half the columns of a shared one: both results, joined by the
      // maxima that the warps tell each other.
      int from = 0, to = HD;
      float f = 1.f, f_pal = 0.f;
      const bool pal_has = !two && it.steps_of(1 - t) > 0;
      if (!two) {
        from = t * (HD / 2);
        to = from + HD / 2;
        s_ml[warp][lane] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_done[warp]));
        if (!(ok = warp_wait(saddr(&s_done[pal]), n_pair & 1, a.wait_ns))) break;
        tc_fence_after();
        const float2 other = s_ml[pal][lane];
        const float nm = fmaxf(m, other.x);
        f = m == nm ? 1.f : exp2_approx(m - nm);
        f_pal = other.x == nm ? 1.f : exp2_approx(other.x - nm);
        // The same order of the sum in both warps.
        l = t == 0 ? l * f + other.y * f_pal : other.y * f_pal + l * f;
        m = nm;
      }
      // Result columns go out 32 at a time: to the output, if the unit is whole, or to a piece (0:
      // of a unit that starts before, 1: of one that goes on).
      const bool whole = (it.flags & (kFirst | kLast)) == (kFirst | kLast);
      // A row without keys is zeros; one with keys has l above 0, unless every score is -inf
      // (0 / 0), and NaN where one is NaN or +inf: the row then is NaN.
      const bool none = whole && real && l == 0.f && blind(a, it.b, me.node, it.len, it.keys);
      const float inv = whole ? __fdividef(1.f, l) : 1.f;
      float* piece = a.part + ((int64_t)blockIdx.x * 2 + (it.flags & kFirst ? 1 : 0)) * C::kPiece;
      // A thread has a row; the 32 of a warp lie side by side in a piece, 4 columns after 4.  Stored
      // to the output that way every 16 bytes touch a line of their own, which is still faster for
      // the few rows of a shared tile.  Else 64 bytes of a row at a time cross shared memory, the
      // 16-byte pieces exchanged by the row's bits against bank conflicts, and leave as 8 rows a store.
      uint4* piece_o = reinterpret_cast<uint4*>(piece) + (second * 4 + (warp & 3)) * (HD / 4) * 32 + lane;
      const uint32_t stage = ring + C::kRing + warp * C::kOut;
      const int place = real ? me.node * a.heads * HD + me.head * HD : -1;  // in the sequence's output
      uint16_t* out = a.out + (int64_t)it.b * a.nodes * a.heads * HD;
      auto leave = [&](const uint32_t* w, auto where) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 +
                                                                        ((i ^ (lane >> 1 & 3)) << 4)),
                       "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3])
                       : "memory");
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 8 + (lane >> 2);
          uint4 x;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                       : "r"(stage + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4))
                       : "memory");
          uint4* dst = where(r);
          if (dst) *dst = x;
        }
      };
      float odd = 0.f;  // NaN once an element is not finite
      if (!two) {
        const uint64_t f2 = pair(f * inv, f * inv), f_pal2 = pair(f_pal * inv, f_pal * inv);
        uint64_t odd2 = 0;
#pragma unroll 1
        for (int c = from; c < to; c += 16) {
          uint32_t o[16] = {}, x[16] = {};
          if (mine > 0) tmem_ld16(o_at + c, o);
          if (pal_has) tmem_ld16(o_pal + c, x);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const uint64_t v = fma2(pair(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f_pal2,
                                    mul2(pair(__uint_as_float(o[e]), __uint_as_float(o[e + 1])), f2));
            odd2 = fma2(v, 0, odd2);
            o[e] = __float_as_uint(lo_of(v));
            o[e + 1] = __float_as_uint(hi_of(v));
          }
          if (none) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0;
          }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              piece_o[(c / 4 + i) * 32] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          } else if (real) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = T::pack(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
#pragma unroll
            for (int i = 0; i < 2; ++i)
              reinterpret_cast<uint4*>(out + place + c)[i] =
                  make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        odd = lo_of(odd2) + hi_of(odd2);
      } else {
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
          uint32_t o[32];
          tmem_ld32(o_at + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float v = __uint_as_float(o[e]);
            odd = fmaf(v, 0.f, odd);
            o[e] = __float_as_uint(none ? 0.f : v * inv);
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = T::pack(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
            leave(o, [&](int r) {
              const int at = __shfl_sync(0xffffffffu, place, r);
              return at < 0 ? nullptr : reinterpret_cast<uint4*>(out + at + c) + (lane & 3);
            });
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              piece_o[(c / 4 + i) * 32] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
      }
      if (!whole && from == 0) {
        piece[2 * kM * HD + second * kM + row] = m;
        piece[2 * kM * (HD + 1) + second * kM + row] = l;
      }
      tc_fence_before();
      if (!two) {  // neither result is overwritten before both warps have read it
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_read[warp]));
        if (!(ok = warp_wait(saddr(&s_read[pal]), n_pair++ & 1, a.wait_ns))) break;
        tc_fence_after();
      }
      mend |= whole && real && !none && odd != 0.f;
    }
    if (ok && __any_sync(0xffffffffu, mend)) mend_units<T, HD>(a, prefix, t, warp & 3);
    if (!ok) s_abort = 1;
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kKeyWarp || warp == kValueWarp) {
    // ---------------- TMA producers: Q and K, or V ----------------
    // Tiles of a piece stand in the ring in the order of their use: K(0) .. K(lead - 1), then
    // K(j + lead), V(j).
    const bool is_v = warp == kValueWarp;
    const CUtensorMap* map = is_v ? &map_v : &map_k;
    const uint32_t leader = elect_one();
    const int boxes = kN / a.box, page_boxes = a.kv.page_size / a.box;
    uint32_t g = 0, n_q0 = 0, n_q1 = 0, n_tail = 0, ones = 0;
    Piece pc;
    if (a.between) {
      const int x = Piece::between(a, prefix, lane & 1 ? hi : lo, total);
      lo = __shfl_sync(0xffffffffu, x, 0);
      hi = __shfl_sync(0xffffffffu, x, 1);
    }
    bool more = !is_v && pc.start(a, prefix, lo, hi);
    int len = 0, keys = 0, of = -1;  // of sequence `of`
    // The item after the one at hand, and its first 64 boxes' pages, on their way while this one's
    // loads are issued.
    Item nx;
    // Describes the next piece, or the end.
    auto publish = [&]() {
      const uint32_t i = n_it % kItems;
      ok = warp_wait(saddr(&s_itempty[i]), (n_it / kItems & 1) ^ 1, a.wait_ns);
      if (!ok) return;
      ++n_it;
      Item x{};
      if (more) {
        if (pc.b != of) span(a, of = pc.b, len, keys);
        const int kp = a.blocks == 1 ? pc.u : pc.u / a.blocks, block = pc.u - kp * a.blocks;
        const bool two = a.nodes - block * 2 * a.tokens > a.tokens;
        x = Item{pc.b, block * 2 * a.tokens, kp * a.tile_heads, len, keys, pc.s0,
                 pc.s1 - pc.s0,
                 (two ? kTwo : 0) | (pc.s0 == 0 ? kFirst : 0) | (pc.s1 == pc.n ? kLast : 0) |
                     (int)(ones & 1) << 3 | (a.parts == 1 ? kp : kp / a.parts) << 8};
        ones += !two;
      }
      nx = x;
      if (lane == 0) {
        s_item[i] = x;
        mbar_arrive(saddr(&s_itfull[i]));
      }
      __syncwarp();
      if (more) more = pc.next(a, prefix);
    };
    auto entry_of = [&](int box) { return a.page_shift >= 0 ? box >> a.page_shift : box / page_boxes; };
    auto look = [&](const Item& x, int box) {  // the table's entry for a box
      if (box * a.box >= x.keys) return 0;
      const int entry = entry_of(box);
      return entry < a.kv.max_pages ? a.kv.table[x.b * a.kv.table_stride + entry] : -1;
    };
    auto checked = [&](int page) {
      if (page >= 0 && page < a.kv.num_pages) return page;
      set_device_error(kErrPage);
      return 0;
    };
    int nx_page = 0, nx_next = 0;
    auto prepare = [&]() {
      if (is_v) next_item(nx);
      else publish();
      if (!ok || __shfl_sync(0xffffffffu, nx.steps, 0) == 0) return;
      const int first = nx.s0 * boxes / 32 * 32 + lane;
      nx_page = look(nx, first);
      nx_next = look(nx, first + 32);
    };
    prepare();
    while (ok && __shfl_sync(0xffffffffu, nx.steps, 0) > 0) {
      const Item it = nx;
      const int flags = __shfl_sync(0xffffffffu, it.flags, 0), seq = __shfl_sync(0xffffffffu, it.b, 0);
      const int s0 = __shfl_sync(0xffffffffu, it.s0, 0), all = __shfl_sync(0xffffffffu, it.steps, 0);
      const int end = __shfl_sync(0xffffffffu, it.keys, 0), kv_head = flags >> 8;
      const int lead = lead_of(flags & kTwo);
      // Pages and places in them (in groups of 8 rows) of 32 boxes of the sequence from w_base on,
      // one per lane, and the table's entries of the 32 after them.
      int w_base = s0 * boxes / 32 * 32;
      int w_page = checked(nx_page), w_next = nx_next;
      auto place_of = [&](int box) {
        return (kv_head * page_boxes + box - entry_of(box) * page_boxes) * (a.box / 8);
      };
      int w_at = place_of(w_base + lane);
      for (int t = 0; !is_v && t < (flags & kTwo ? 2 : 1) && ok; ++t) {
        const int slot = flags & kTwo ? t : flags >> 3 & 1;
        const uint32_t turn = slot ? n_q1++ : n_q0++;
        ok = warp_wait(saddr(&s_qempty[slot]), (turn & 1) ^ 1, a.wait_ns);
        if (!ok) break;
        const uint32_t bar = saddr(&s_qfull[slot]);
        mbar_expect_tx_if(leader, bar, a.tokens * a.tile_heads * 128 * C::kHalves);
        for (int hf = 0; hf < C::kHalves; ++hf)
          tma_load_4d_if(leader, q_at + slot * C::kTileQ + hf * C::kHalfQ, &map_q, bar, hf * 64,
                         __shfl_sync(0xffffffffu, it.head0, 0),
                         __shfl_sync(0xffffffffu, it.node0, 0) + t * a.tokens, seq);
      }
      if (!ok || __any_sync(0xffffffffu, s_abort)) break;
      for (int i = 0; i < all; ++i) {
        const uint32_t x = g + (is_v ? (i + lead < all ? 2 * i + lead + 1 : all + i) : i < lead ? i : 2 * i - lead);
        const uint32_t s = x % NS, dst = ring + s * C::kTileK;
        const int from = (s0 + i) * boxes - w_base;
        if (from >= 32) {
          w_base += 32;
          w_page = checked(w_next);
          w_at = place_of(w_base + lane);
          w_next = look(it, w_base + 32 + lane);
        }
        const int rows = end - (s0 + i) * kN, count = min(boxes, (rows + a.box - 1) >> a.box_shift);
        const bool tail = is_v && rows < kN;
        const uint32_t bar = tail ? saddr(&s_tail) : saddr(&s_full[s]);
        ok = warp_wait(saddr(&s_empty[s]), (x / NS & 1) ^ 1, a.wait_ns);
        if (!ok) break;
        mbar_expect_tx_if(leader, bar, count * a.box * 128 * C::kHalves);
        int page[kN / 16], at[kN / 16];
#pragma unroll
        for (int n = 0; n < kN / 16; ++n) {
          page[n] = __shfl_sync(0xffffffffu, w_page, from + n);
          at[n] = __shfl_sync(0xffffffffu, w_at, from + n);
        }
#pragma unroll
        for (int n = 0; n < kN / 16; ++n)
          if (n < count)
            tma_load_5d_if(leader, dst + n * a.box * 128 * C::kHalves, map, bar, at[n], page[n]);
        if (i == (is_v ? min(2, all - 1) : 0)) prepare();  // the item that V waits for is K's
        if (!ok) break;
        if (!tail) continue;
        ok = warp_wait(saddr(&s_tail), n_tail++ & 1, a.wait_ns);
        if (!ok) break;
        for (uint32_t z = rows * 128 + lane * 16; z < kN * 128; z += 512)
          for (int hf = 0; hf < C::kHalves; ++hf)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             dst + (z >> 10) * C::kGroup + hf * 1024 + (z & 1023)),
                         "r"(0)
                         : "memory");
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_full[s]));
      }
      g += 2 * all;
    }
    if (!ok) s_abort = 1;
    // After a timeout copies may be in flight: the CTA stays until they have landed.
    if (s_abort) {
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 1000000) __nanosleep(1000);
    }
    if (is_v) {
      auto have_of = [&](int b) {
        int len, keys;
        span(a, b, len, keys);
        return keys - len;
      };
      Piece last;
      if (lane == 0) {  // what is to be joined
        int4 job = make_int4(0, 0, 0, 0);
        if (lo < hi) {
          last.find(a, prefix, hi - 1, lo, hi);
          // Its first step is this CTA's, its last another's.
          if (last.left <= 0 && last.end > 0 && last.end < last.n)
            job = make_int4(last.b, last.u, (hi - last.end + last.n - 1) / share - blockIdx.x + 1, have_of(last.b));
        }
        a.jobs[blockIdx.x] = job;
      }
      // Rows of nodes that are not there: zeros.
      for (int b = blockIdx.x; b < a.kv.seqs; b += gridDim.x) {
        const int row = a.heads * HD / 8;
        uint4* o = reinterpret_cast<uint4*>(a.out) + (int64_t)b * a.nodes * row;
        for (int i = have_of(b) * row + lane; i < a.nodes * row; i += 32) o[i] = make_uint4(0, 0, 0, 0);
      }
    }
  } else {
    // ---------------- MMA issuers: one warp per pipeline ----------------
    // The whole warp walks the loop and one elected lane issues: addresses and
    // descriptors are then uniform over the warp and stay in uniform registers.
    const uint32_t d_qk = instr_desc<T>(kN, false), d_pv = instr_desc<T>(HD, true);
    const uint32_t leader = elect_one();
    const uint64_t desc_q = smem_desc(q_at), desc_k = smem_desc(ring, C::kGroup);
    const uint64_t desc_v = smem_desc_mn(ring, 1024, C::kGroup);
    const uint32_t s_col = tmem + C::kS + t * C::kS1;
    const uint32_t o_col = tmem + C::kO + t * C::kO1;
    uint32_t ring_slot = 0, ring_turn = 0;  // of the ring's next tile, and the parity of its barrier
    uint32_t n_q0 = 0, n_q1 = 0;            // uses of the Q buffers
    uint32_t n_qk = 0, n_pv = 0;
    // A slot, like a Q buffer, counts two releases: one of each pipeline.
    for (Item it; ok && next_item(it);) {
      const int flags = __shfl_sync(0xffffffffu, it.flags, 0);
      const int all = __shfl_sync(0xffffffffu, it.steps, 0);
      const bool two = flags & kTwo;
      const int lead = lead_of(two), mine = two ? all : (all + 1 - t) >> 1, slot = two ? t : flags >> 3 & 1;
      const uint32_t q_turn = slot ? n_q1 : n_q0;
      n_q0 += two || slot == 0;
      n_q1 += two || slot == 1;
      ok = warp_wait(saddr(&s_qfull[slot]), q_turn & 1, a.wait_ns);
      if (ok && mine == 0 && lane == 0) mbar_arrive(saddr(&s_qempty[slot]));
      const uint64_t qd = desc_q + slot * (C::kTileQ >> 4);
      // The piece's tiles in the ring's order (see the producers).  A warp waits for all of
      // them and releases those that the other pipeline alone uses: a barrier's parity tells one
      // phase from the next only, so a warp that skipped tiles could take an older phase of a
      // slot for the one it wants.
      int j_k = 0, j_v = 0, qk_left = mine;
      bool first = true;
      for (int r = 0; r < 2 * all && ok; ++r) {
        const bool is_k = j_k < all && (r <= lead || !(r - lead & 1));
        const int j = is_k ? j_k++ : j_v++;
        const uint32_t at = ring_slot;
        ok = warp_wait(saddr(&s_full[at]), ring_turn, a.wait_ns);
        if (++ring_slot == NS) {
          ring_slot = 0;
          ring_turn ^= 1;
        }
        if (!ok) break;
        if (!two && (j & 1) != t) {
          if (lane == 0) mbar_arrive(saddr(&s_empty[at]));
          continue;
        }
        if (is_k) {  // Q K^T, into the buffer whose P the last product but one has read
          if (n_qk >= 2) ok = product_done(n_qk - 2);
          if (!ok) break;
          tc_fence_after();
          const uint64_t kd = desc_k + at * (C::kTileK >> 4);
          const uint32_t sc = s_col + (n_qk & 1) * kN;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            tc_mma_if(leader, sc, qd + ((kk / 4 * C::kHalfQ + kk % 4 * 32) >> 4),
                      kd + ((kk / 4 * 1024 + kk % 4 * 32) >> 4), d_qk, kk != 0);
          tc_commit_if(leader, saddr(&s_sfull[t][n_qk & 1]));
          if (--qk_left == 0) {
            tc_commit_if(leader, saddr(&s_qempty[slot]));
            if (two) tc_commit_if(leader, saddr(&s_qempty[slot]));
          }
          ++n_qk;
        } else {
          ok = warp_wait(saddr(&s_pready[t][n_pv & 1]), n_pv >> 1 & 1, a.wait_ns);
          if (!ok) break;
          tc_fence_after();
          const uint64_t vd = desc_v + at * (C::kTileK >> 4);
          const uint32_t pc = s_col + (n_pv & 1) * kN;
          tc_mma_ta_if(leader, o_col, pc, vd, d_pv, first ? 0 : 1);
#pragma unroll
          for (int kk = 1; kk < kN / 16; ++kk)
            tc_mma_ta_if(leader, o_col, pc + kk * 8, vd + (kk * 2 * C::kGroup >> 4), d_pv, 1);
          tc_commit_if(leader, saddr(&s_pvdone[t][n_pv & 1]));
          first = false;
          ++n_pv;
        }
        tc_commit_if(leader, saddr(&s_empty[at]));
      }
    }
    if (!ok) s_abort = 1;
    // What was issued is over before the CTA ends, after a timeout too.
    tc_commit_if(leader, saddr(&s_drain[t]));
    warp_wait(saddr(&s_drain[t]), 0, a.wait_ns);
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u)
                 : "memory");
  }
}

// The cut units' results, in the order of the keys: a warp takes 16 columns of 32 rows, a row to a
// lane, of the unit that is cut at the end of the main kernel's CTA blockIdx.x.  AHEAD pieces are on
// their way at once.
constexpr int kJoinThreads = 128, kJoinCols = 16;
template <typename T, int HD, int AHEAD>
__device__ __forceinline__ void join_rows(const TreeArgs& a, int4 job) {
  constexpr int kPiece = Cfg<HD>::kPiece, kSets = HD / kJoinCols, kVec = kJoinCols / 4;
  const int item = blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int quad = item / kSets, c0 = item % kSets * kJoinCols;  // rows 32 quad ..
  const int b = job.x, n = job.z, r = quad * 32 + lane;
  const Row me = row_of(a, job.y, r / kM, r % kM, job.w);
  const bool real = me.node >= 0;
  if (!__any_sync(0xffffffffu, real)) return;
  // Piece 0 is CTA c's second, the others the first of the CTAs after it.
  const float* first = a.part + (int64_t)blockIdx.x * 2 * kPiece;
  float m = -INFINITY, l = 0.f, acc[kJoinCols] = {};
  for (int k0 = 0; k0 < n && real; k0 += AHEAD) {
    float mk[AHEAD], lk[AHEAD];
    float4 ok[AHEAD][kVec];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      mk[k] = -INFINITY;
      lk[k] = 0.f;
#pragma unroll
      for (int i = 0; i < kVec; ++i) ok[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + k >= n) continue;
      const float* src = first + (int64_t)(k0 + k == 0 ? 1 : 2 * (k0 + k)) * kPiece;
      mk[k] = src[2 * kM * HD + r];
      lk[k] = src[2 * kM * (HD + 1) + r];
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        ok[k][i] = reinterpret_cast<const float4*>(src)[(quad * (HD / 4) + c0 / 4 + i) * 32 + lane];
    }
    float nm = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) nm = fmaxf(nm, mk[k]);
    const float f = m == nm ? 1.f : exp2_approx(m - nm);
    m = nm;
    l *= f;
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c) acc[c] *= f;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float fk = mk[k] == nm ? 1.f : exp2_approx(mk[k] - nm);
      l = fmaf(fk, lk[k], l);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        acc[4 * i] = fmaf(fk, ok[k][i].x, acc[4 * i]);
        acc[4 * i + 1] = fmaf(fk, ok[k][i].y, acc[4 * i + 1]);
        acc[4 * i + 2] = fmaf(fk, ok[k][i].z, acc[4 * i + 2]);
        acc[4 * i + 3] = fmaf(fk, ok[k][i].w, acc[4 * i + 3]);
      }
    }
  }
  bool none = false;
  float odd = 0.f;
  if (real) {
    int len = 0, keys = 0;
    if (l == 0.f) {
      span(a, b, len, keys);
      none = blind(a, b, me.node, len, keys);
    }
    const float inv = __fdividef(1.f, l);
    uint32_t o[kJoinCols / 2];
#pragma unroll
    for (int c = 0; c < kJoinCols; c += 2) {
      odd = fmaf(acc[c], 0.f, fmaf(acc[c + 1], 0.f, odd));
      o[c / 2] = none ? 0u : T::pack(acc[c] * inv, acc[c + 1] * inv);
    }
    uint4* dst = reinterpret_cast<uint4*>(a.out +
                                          (((int64_t)b * a.nodes + me.node) * a.heads + me.head) * HD + c0);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  }
  for (uint32_t again = __ballot_sync(0xffffffffu, odd != 0.f && !none); again; again &= again - 1) {
    const int at = __ffs(again) - 1;
    int len, keys;
    span(a, b, len, keys);
    mend_row<T, HD>(a, b, __shfl_sync(0xffffffffu, me.node, at), __shfl_sync(0xffffffffu, me.head, at),
                    len, keys, c0, c0 + kJoinCols);
  }
}
template <typename T, int HD>
__global__ void __launch_bounds__(kJoinThreads, 4) k_tree_join(const __grid_constant__ TreeArgs a) {
  pdl_trigger();
  pdl_wait();
  const int4 job = a.jobs[blockIdx.x];
  if (job.z == 0) return;
  if (job.z == 2) join_rows<T, HD, 2>(a, job);
  else join_rows<T, HD, 4>(a, job);
}

// N dimensions of which the innermost box is 64 elements, 128-byte swizzle.
template <int N>
bool make_map(CUtensorMap* map, const uint16_t* x, bool bf16, const cuuint64_t (&dims)[N],
              const int64_t (&stride)[N - 1], const cuuint32_t (&box)[N]) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t strides[N - 1];
  cuuint32_t ones[N];
  for (int i = 0; i < N; ++i) ones[i] = 1;
  for (int i = 0; i < N - 1; ++i) strides[i] = (cuuint64_t)stride[i] * 2;
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, N,
            const_cast<uint16_t*>(x), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
bool tree_attr() {
  // The warps' register shares must not exceed what the block is launched with: the last to
  // ask would wait for good.
  cudaFuncAttributes at;
  return cudaFuncGetAttributes(&at, k_tree_attention<T, HD>) == cudaSuccess &&
         at.numRegs * kThreads >= kRegs &&
         cudaFuncSetAttribute(k_tree_attention<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
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
  if (a.whole || a.between) return MOE_OK;
  if (launch_pdl(k_tree_join<T, HD>, dim3(grid, 2 * kM / 32 * (HD / kJoinCols) / (kJoinThreads / 32)), dim3(kJoinThreads), 0, s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

constexpr int64_t kJobsAt = 4096;  // behind the counters of the calls that share a workspace

}  // namespace
}  // namespace moe

extern "C" size_t moe_tree_attention_workspace_size(int64_t head_dim) {
  using namespace moe;
  if (head_dim != 64 && head_dim != 128) return 0;
  return kJobsAt + (size_t)sm_count() * 16 +
         (size_t)sm_count() * 2 * 4 * (head_dim == 64 ? Cfg<64>::kPiece : Cfg<128>::kPiece);
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
  // Places of boxes are looked up some thousand positions past a table's end, in 32 bits.
  if (c.kv.page_size % 16 || c.kv.seqs > kMaxSeqs || c.nodes > kMaxNodes || c.kv.num_pages > INT32_MAX ||
      c.kv.max_pages * c.kv.page_size > 1 << 30)
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
  a.scale_log2 = scale * 1.4426950408889634f;
  const size_t need = moe_tree_attention_workspace_size(hd);
  if (!c.workspace || c.workspace_bytes < (int64_t)need) return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  // Rows may be computed again from their queries after results have been written.
  const int64_t row = 2 * c.heads * hd, rows = 2 * (c.nodes - 1) * c.q_node_stride + row;
  if (overlap(c.out, c.kv.seqs * c.nodes * row, c.q, 2 * (c.kv.seqs - 1) * c.q_seq_stride + rows))
    for (int64_t b = 0; b < c.kv.seqs; ++b)
      if (overlap(c.out, c.kv.seqs * c.nodes * row, c.q + b * c.q_seq_stride, rows))
        return MOE_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  const bool bf16 = c.kv.dtype == MOE_DTYPE_BF16;
  if (tree_is_few(a)) return tree_attention_few(a, static_cast<int>(hd), bf16, s);
  // A tile's rows are the heads of a group for neighbouring nodes; a group above 128
  // heads is cut.
  a.parts = (a.group + kM - 1) / kM;
  while (a.group % a.parts) ++a.parts;
  a.tile_heads = a.group / a.parts;
  a.tokens = kM / a.tile_heads;
  a.blocks = (a.nodes + 2 * a.tokens - 1) / (2 * a.tokens);
  const int64_t per_seq = (int64_t)a.kv.kv_heads * a.parts * a.blocks;
  const int64_t steps = ceil_div(c.kv.max_pages * c.kv.page_size, kN) + kStart;
  if (per_seq > INT32_MAX || c.kv.seqs * per_seq > (INT32_MAX - 4096) / steps)  // the line's places: 32 bits
    return MOE_ERR_UNSUPPORTED;
  a.per_seq = static_cast<int>(per_seq);
  a.box_shift = 4;
  while ((1 << a.box_shift) < kN && a.kv.page_size % (2 << a.box_shift) == 0) ++a.box_shift;
  a.box = 1 << a.box_shift;
  a.page_shift = -1;
  for (int i = 0; i < 17; ++i)  // pages have 2^20 rows at most
    if (a.kv.page_size == a.box << i) a.page_shift = i;
  a.jobs = reinterpret_cast<int4*>(static_cast<char*>(c.workspace) + kJobsAt);
  a.part = reinterpret_cast<float*>(a.jobs + sm_count());
  a.wait_ns = wait_limit_ns();
  CUtensorMap mq, mk, mv;
  const cuuint64_t q_dims[4] = {(cuuint64_t)hd, (cuuint64_t)c.heads, (cuuint64_t)c.nodes,
                                (cuuint64_t)c.kv.seqs};
  const int64_t q_strides[3] = {hd, c.q_node_stride, c.kv.seqs > 1 ? c.q_seq_stride : c.q_node_stride * c.nodes};
  const cuuint32_t q_box[4] = {64, (cuuint32_t)a.tile_heads, (cuuint32_t)a.tokens, 1};
  // Keys and values as (64 dims, 8 rows, the dims' halves, 8 rows each of all KV heads, pages).
  const bool none = c.kv.max_pages == 0;  // no keys at all: the maps describe q, unread
  const cuuint64_t kv_dims[5] = {64, 8, (cuuint64_t)hd / 64,
                                 none ? 1 : (cuuint64_t)(c.kv.kv_heads * c.kv.page_size / 8),
                                 none ? 1 : (cuuint64_t)c.kv.num_pages};
  const cuuint32_t kv_box[5] = {64, 8, (cuuint32_t)hd / 64, none ? 1 : (cuuint32_t)a.box / 8, 1};
  auto kv_map = [&](CUtensorMap* m, const uint16_t* x, int64_t page_stride) {
    const int64_t whole = c.kv.kv_heads * c.kv.page_size * hd;
    return make_map(m, none ? c.q : x, bf16, kv_dims,
                    {hd, 64, 8 * hd, c.kv.num_pages > 1 && !none ? page_stride : whole}, kv_box);
  };
  if (!make_map(&mq, c.q, bf16, q_dims, q_strides, q_box) ||
      !kv_map(&mk, c.kv.k_pages, c.kv.k_page_stride) || !kv_map(&mv, c.kv.v_pages, c.kv.v_page_stride))
    return MOE_ERR_CUDA;
  const int64_t line = c.kv.seqs * per_seq * steps, most = ceil_div(line, kMinShare + kStart);
  const int64_t units = c.kv.seqs * per_seq, sms = sm_count();
  a.whole = units <= sms && steps - kStart <= std::max(kWholeSteps, units / 6);
  a.between = !a.whole && steps - kStart <= kBetweenSteps;
  const int grid = static_cast<int>(a.whole ? units : most < 1 ? 1 : most < sms ? most : sms);
  if (bf16)
    return hd == 64 ? launch_tree<BF16, 64>(a, mq, mk, mv, grid, s)
                    : launch_tree<BF16, 128>(a, mq, mk, mv, grid, s);
  return hd == 64 ? launch_tree<F16, 64>(a, mq, mk, mv, grid, s)
                  : launch_tree<F16, 128>(a, mq, mk, mv, grid, s);
}
