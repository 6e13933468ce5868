// Sampling one token per row of logits: temperature, top-k, top-p, min-p, from
// random numbers the caller gives.  No counterpart in the reference (greedy
// decoding only, engine/engine.py:579-663).
//
// For a row x of V logits (NaN counts as -inf), m its maximum:
//   d_i = 0 where x_i == m, else (x_i - m) / temperature
//   w_i = trunc(2^40 exp(d_i)), exp in fp32, w as a 64-bit integer
// Tokens are ordered by falling x, equal ones by rising index.
//   top-k keeps the first k; W = sum of their w
//   top-p keeps of those the shortest prefix with sum >= ceil(p W)
//   min-p keeps of those exp(d_i) >= min_p
// W' = sum of the w kept, r = floor(u W'); the token is the first kept index,
// in index order, whose inclusive sum of w exceeds r, its probability w / W'.
// Temperature 0, or k = 1: the maximum of lowest index, probability 1.
//
// Sums of integers do not depend on their order, so the token does not either:
// the same logits and numbers give the same token however a row is split.  40
// bits below the maximum leave every weight that has a chance to be drawn
// fp32's precision, and 2^18 of them fit 64 bits with room to spare.
//
// Many rows, or short ones, take a CTA each (sample_rows.cuh).  Here a row is
// spread over a cluster of CTAs whose threads hold it in registers, as integers of
// the same order ("keys").  Such a call is a chain of reductions and bound by their
// latency: in a graph 8 to 18 us for one row of 32000 fp16 logits at top-p 0.95, by
// whether few logits hold it (64 KB: a plain copy would take 0.01), 22 for one of
// 131072 fp32.
//   * A first pass adds each weight to the sums of 7 thresholds (21
//     instructions a logit), 0.5 to 16 below the maximum in units of the
//     temperature, where a language model's boundaries usually lie.  If then at
//     most 256 logits are above the threshold that already holds enough, they go
//     to one CTA of the cluster, which orders them and applies every filter by
//     comparing each with each (more would cost it longer than another pass); the
//     others are done.
//   * Else no sort either: the k-th token and the top-p boundary are found by
//     search over the keys, 8 ways a pass.  The logits still between the bounds
//     are gathered in shared memory before each pass, so that it works on full
//     warps of them, and once at most 256 are left every CTA takes a copy and
//     decides by itself.
//   * Exponentials are not kept: the first pass needs every logit's, what
//     follows only those of the few between the bounds or kept.  That leaves 64
//     registers a thread and two CTAs to an SM, one's barriers under the other's
//     arithmetic (16 logits a thread do not quite fit them: some 250 bytes of a thread
//     are spilled).
//   * Between passes the CTAs exchange sums, which is most of a call: each
//     stores its 8 into every CTA's shared memory with st.async, whose bytes
//     complete an mbarrier there (a cluster barrier behind plain stores took 2000
//     cycles, this a third: the one row 13.3 -> 12.0 us).  Waits are bounded:
//     on a timeout the error word is set and the CTA leaves, as then do the others
//     (Exchange::leave).
#include <cooperative_groups.h>

#include "paged.cuh"
#include "sample_rows.cuh"
#include "sm100_ptx.cuh"

namespace moe {
namespace {

namespace cg = cooperative_groups;

MOE_DEFINE_ERROR_WORD()

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;            // 8 is the portable size; 16 only where a row needs it
constexpr int kMaxPer = 32;                // logits a thread holds at most
constexpr int kList = 256;                 // logits that a search finishes with directly
constexpr int kMaxSyncs = 2;               // cluster barriers: one a search, or one for the few
constexpr int kMaxVocab = kMaxCluster * kThreads * kMaxPer;

__device__ __forceinline__ uint32_t map_rank(uint32_t addr, int rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}

// Sums over the cluster, 8 values at a time: lane j of every warp ends up with
// the sum of value j % 8.  slot(r, j): what CTA r contributed to the last one;
// warp_sum[w][j]: what warp w of this CTA did.
//
// Two sets of slots and barriers are used in turn.  A CTA sends its sums of
// exchange n + 2 (the set of n) after it has those of n + 1 from every CTA, and
// each of them sent these after all its warps had read n.
struct Exchange {
  int rank, size, warp, lane;
  uint64_t wait_ns;
  uint64_t (*warp_sum)[8];
  uint64_t (*slots)[kMaxCluster][8];
  uint32_t bar;       // two mbarriers of one arrival (this CTA's, with the bytes to come)
  volatile int* s_dead;
  uint32_t count = 0;
  bool dead = false;  // a wait of this CTA ran out: it gives nothing any more

  __device__ __forceinline__ int turn() const { return count & 1; }
  __device__ __forceinline__ uint64_t slot(int r, int j) const { return slots[turn() ^ 1][r][j]; }
  // Warp 0: value lane % 8 of this CTA to every CTA (just value 0 if `one`).
  __device__ __forceinline__ void give(uint64_t mine, bool one) {
    const uint32_t here = bar + 8 * turn(), at = saddr(&slots[turn()][rank][lane & 7]);
    if (lane == 0) mbar_expect_tx(here, size * (one ? 8 : 64));
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kMaxCluster / 4; ++i) {
      const int r = (lane >> 3) + 4 * i;
      if (r < size && (!one || (lane & 7) == 0))
        asm volatile(
            "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                map_rank(at, r)),
            "l"(mine), "r"(map_rank(here, r))
            : "memory");
    }
  }
  // Warp 0 waits for the bytes and the others for warp 0, so that a timeout is one
  // for the whole CTA.
  __device__ __forceinline__ void wait() {
    if (warp == 0 && !mbar_poll_or(bar + 8 * turn(), count >> 1 & 1, wait_ns,
                                   [] { set_device_error(kErrWaitTimeout); }))
      *s_dead = 1;
    __syncthreads();
    dead = *s_dead;
    ++count;
  }
  // After a timeout.  The other CTAs may have sums for this one on their way, of
  // the exchange that ran out or the next, so its shared memory has to last: it goes
  // along with their cluster barriers, of which a launch has kMaxSyncs at most after
  // the first exchange.  The one after those is passed when every other CTA has ended
  // or is in here too; their last stores are then given ample time to land.
  __device__ __forceinline__ void leave() const {
    for (int i = 0; i <= kMaxSyncs; ++i) cg::this_cluster().sync();
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 20000) __nanosleep(1000);
  }
  template <int N>
  __device__ __forceinline__ uint64_t sum(const uint64_t (&v)[N]) {
    uint64_t mine = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {  // 27 bits and the rest: 32 of them fit 32 bits
      const uint32_t lo = __reduce_add_sync(kAll, (uint32_t)v[j] & 0x7FFFFFFu);
      const uint32_t hi = __reduce_add_sync(kAll, (uint32_t)(v[j] >> 27));
      if ((lane & 7) == j) mine = lo + ((uint64_t)hi << 27);
    }
    if (lane < 8) warp_sum[warp][lane] = mine;
    return sum_of();
  }
  // The same by halves: a lane hands the values that the other half of its group
  // keeps over, 8 -> 4 -> 2 -> 1, so that lanes 4j .. 4j + 3 end up with value j.
  __device__ __forceinline__ uint64_t sum(const Limbs (&v)[8]) {
    Limbs a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = v[j];
#pragma unroll
    for (int half = 4; half; half >>= 1) {
      const bool up = lane & 4 * half;
#pragma unroll
      for (int j = 0; j < half; ++j) {
        const Limbs keep = up ? a[j + half] : a[j], give = up ? a[j] : a[j + half];
        a[j].hi = keep.hi + __shfl_xor_sync(kAll, give.hi, 4 * half);
        a[j].lo = keep.lo + __shfl_xor_sync(kAll, give.lo, 4 * half);
      }
    }
#pragma unroll
    for (int o = 2; o; o >>= 1) {
      a[0].hi += __shfl_xor_sync(kAll, a[0].hi, o);
      a[0].lo += __shfl_xor_sync(kAll, a[0].lo, o);
    }
    if ((lane & 3) == 0) warp_sum[warp][lane >> 2] = a[0].lo + ((uint64_t)a[0].hi << 20);
    return sum_of();
  }
  __device__ __forceinline__ uint64_t sum_of() {  // of the warps' sums in warp_sum
    __syncthreads();
    if (warp == 0) {
      uint64_t s = 0;
#pragma unroll
      for (int w = 0; w < kWarps; w += 4) s += warp_sum[w + (lane >> 3)][lane & 7];
      s += __shfl_xor_sync(kAll, s, 8);
      s += __shfl_xor_sync(kAll, s, 16);
      give(s, false);
    }
    wait();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < kMaxCluster / 4; ++i) {
      const int r = (lane >> 3) + 4 * i;
      if (r < size) s += slot(r, lane & 7);
    }
    s += __shfl_xor_sync(kAll, s, 8);
    s += __shfl_xor_sync(kAll, s, 16);
    return s;
  }
  __device__ __forceinline__ uint32_t max(uint32_t v) {  // of all threads, in every thread
    v = __reduce_max_sync(kAll, v);
    if (lane == 0) warp_sum[warp][0] = v;
    __syncthreads();
    if (warp == 0)
      give(__reduce_max_sync(kAll, (uint32_t)warp_sum[lane & (kWarps - 1)][0]), true);
    wait();
    return __reduce_max_sync(kAll, lane < size ? (uint32_t)slot(lane & (kMaxCluster - 1), 0) : 0u);
  }
};

template <typename T, int PER>
__global__ void __launch_bounds__(kThreads, PER <= 16 ? 2 : 1) k_sample(const SampleArgs a) {
  using L = Logit<T>;
  constexpr int kVec = L::kVec, kIters = PER / kVec;
  __shared__ uint64_t s_warp[kWarps][8], s_slots[2][kMaxCluster][8];
  extern __shared__ uint32_t s_dyn[];  // two lists of kThreads * PER keys
  __shared__ uint32_t s_all[kList], s_index[kList];
  __shared__ uint64_t s_weight[kList], s_above;
  __shared__ uint32_t s_count[2], s_few, s_key;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ __align__(8) uint64_t s_bar[2];
  __shared__ int s_dead;
  cg::cluster_group cluster = cg::this_cluster();
  const int64_t row = blockIdx.x / a.cluster;
  Exchange ex{static_cast<int>(blockIdx.x % a.cluster), a.cluster, warp, lane, a.wait_ns, s_warp,
              s_slots, saddr(s_bar), &s_dead};
  if (threadIdx.x == 0) {
    s_dead = 0;
    mbar_init(ex.bar, 1);
    mbar_init(ex.bar + 8, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  cluster.barrier_arrive();  // waited for before the first store to another CTA
  pdl_trigger();
  pdl_wait();

  // ---- the row: element v of step i of a lane has index first + i * 32 * kVec + v ----
  uint32_t key[PER];
  const int first = ((ex.rank * kWarps + warp) * kIters * 32 + lane) * kVec;
  const typename L::Raw* x = static_cast<const typename L::Raw*>(a.logits) + row * a.stride;
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    const int at = first + i * 32 * kVec;
    if (wide && at + kVec <= a.vocab) {
      const uint4 v = *reinterpret_cast<const uint4*>(x + at);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (kVec == 8) key[i * kVec + j] = L::key((uint16_t)(w[j / 2] >> (16 * (j & 1))));
        else key[i * kVec + j] = L::key(__uint_as_float(w[j]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) key[i * kVec + j] = at + j < a.vocab ? L::key(x[at + j]) : 0u;
    }
  }
  const float temperature = a.temperature[row], u = a.uniforms[row], p = a.top_p[row];
  const float min_p = fminf(a.min_p[row], 1.f);  // above 1 the maxima stay
  const int k = a.top_k[row];

  // ---- the maximum ----
  uint32_t top = 0;
#pragma unroll
  for (int c = 0; c < PER; ++c) top = max(top, key[c]);
  cluster.barrier_wait();
  top = ex.max(top);
  if (ex.dead) return ex.leave();
  if (!(temperature > 0.f) || k == 1) {  // its lowest index
    uint32_t index = 0xFFFFFFFFu;
#pragma unroll
    for (int c = PER - 1; c >= 0; --c)
      if (key[c] == top) index = first + c / kVec * 32 * kVec + c % kVec;
    index = ~ex.max(~index);
    if (ex.dead) return ex.leave();
    if (ex.rank == 0 && threadIdx.x == 0) {
      a.tokens[row] = index;
      a.probs[row] = 1.f;
    }
    return;
  }
  const float m = L::value(top);
  const Softmax soft(m, temperature);
  auto exp_of = [&](uint32_t key) {  // key 0 is a NaN; m may be infinite
    return key == top ? 1.f : soft.exp(L::value(key));
  };
  if (threadIdx.x == 0) s_count[0] = s_few = 0;

  // Sums of the weights (or counts) of the keys that are >= the threshold t of
  // lane 0 .. 7, as lane j's result: of all logits, and of a list's, where lane
  // 0's is the length of all CTAs' lists.
  auto add = [&](Limbs (&sum)[8], const uint32_t (&th)[8], bool count, uint32_t kk) {
    Limbs w{0, 1};
    if (!count) w = limbs(exp_of(kk));
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (kk >= th[j]) {
        sum[j].hi += w.hi;
        sum[j].lo += w.lo;
      }
  };
  auto pass = [&](bool count, uint32_t t) {
    uint32_t th[8];
    Limbs sum[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) th[j] = __shfl_sync(kAll, t, j);
#pragma unroll
    for (int c = 0; c < PER; ++c) add(sum, th, count, key[c]);
    return ex.sum(sum);
  };
  auto pass_list = [&](bool count, const uint32_t* list, uint32_t n, uint32_t t) {
    uint32_t th[8];
    Limbs sum[8] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) th[j] = __shfl_sync(kAll, t, j);
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) add(sum, th, count, list[i]);
    sum[0] = Limbs{0, threadIdx.x == 0 ? n : 0u};
    return ex.sum(sum);
  };
  // The largest key whose sum over it and all above is >= need, and the sum
  // above it.  t, s: thresholds of a first pass (rising with the lane, lane 0
  // not among them) and their sums.  lo's sum is known to be enough, hi's not.
  struct Bound {
    uint32_t key;
    uint64_t above;
  };
  auto search = [&](bool count, uint64_t need, uint32_t lo, uint32_t hi, uint32_t t, uint64_t s) {
    uint64_t above = 0;
    uint32_t held_n = ~0u;  // keys in the last list
    for (int turn = 0;; turn ^= 1) {
      const uint32_t enough = __ballot_sync(kAll, lane >= 1 && lane < 8 && s >= need) | 1u;
      const int j = 31 - __clz(enough);  // sums fall as thresholds rise
      const uint32_t t_lo = __shfl_sync(kAll, t, j), t_hi = __shfl_sync(kAll, t, (j + 1) & 7);
      const uint64_t s_hi = shfl64(s, (j + 1) & 7);
      if (j > 0 && t_lo > lo) lo = t_lo;
      if (j < 7 && t_hi < hi) {
        hi = t_hi;
        above = s_hi;
      }
      if (hi - lo <= 1) {
        // A second search begins with list 0, empty: between this and its first
        // entry lies an exchange (the sums of its first thresholds).
        if (threadIdx.x == 0) s_count[0] = 0;
        return Bound{lo, above};
      }
      // The logits between the bounds, from the registers or the last list.
      uint32_t *list = s_dyn + turn * kThreads * PER, *counter = &s_count[turn];
      if (held_n == ~0u) {
        uint32_t slots = 0;
#pragma unroll
        for (int c = 0; c < PER; ++c) slots |= (key[c] - lo < hi - lo ? 1u : 0u) << c;
        uint32_t at = slots ? atomicAdd(counter, __popc(slots)) : 0u;
#pragma unroll
        for (int c = 0; c < PER; ++c)
          if (slots >> c & 1) list[at++] = key[c];
      } else {
        const uint32_t* from = s_dyn + (turn ^ 1) * kThreads * PER;
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < held_n; i += kThreads) {
          const uint32_t kk = from[i];
          if (kk - lo < hi - lo) list[atomicAdd(counter, 1)] = kk;
        }
      }
      if (threadIdx.x == 0) s_count[turn ^ 1] = 0;
      __syncthreads();
      held_n = *counter;
      const uint32_t step = (hi - lo + 7) / 8;
      const uint64_t next = (uint64_t)lo + (uint64_t)step * (lane & 7);
      t = next < hi ? (uint32_t)next : hi;
      s = pass_list(count, list, held_n, t);
      const uint64_t n = shfl64(s, 0);
      s += above;
      if (ex.dead) return Bound{lo, above};
      if (n > kList) continue;
      cluster.sync();  // the lists of the other CTAs
      if (warp < ex.size) {  // warp r copies CTA r's
        int from = 0, held = 0;
        for (int r = 0; r <= warp; ++r) {
          from += held;
          held = (int)ex.slot(r, 0);
        }
        const uint32_t* its = cluster.map_shared_rank(list, warp);
        for (int i = lane; i < held; i += 32) {
          const uint32_t kk = its[i];
          s_all[from + i] = kk;
          s_weight[from + i] = count ? 1ull : weight(exp_of(kk));
        }
      }
      if (threadIdx.x == 0) s_key = 0;
      __syncthreads();
      uint64_t over = 0, equal = 0;  // weights above and at the thread's key
      uint32_t own = 0;
      bool ok = false;
      if (threadIdx.x < n) {
        own = s_all[threadIdx.x];
        for (int i = 0; i < (int)n; ++i) {
          const uint32_t kk = s_all[i];
          const uint64_t w = s_weight[i];
          over += kk > own ? w : 0ull;
          equal += kk == own ? w : 0ull;
        }
        ok = above + over + equal >= need;
      }
      const uint32_t found_key = __reduce_max_sync(kAll, ok ? own : 0u);
      if (lane == 0 && found_key) atomicMax(&s_key, found_key);
      if (threadIdx.x == 0) s_count[0] = 0;  // as above
      __syncthreads();
      if (threadIdx.x < n && own == s_key) s_above = above + over;  // the same value from each
      __syncthreads();
      return Bound{s_key, s_above};
    }
  };
  // First thresholds: lane 7 the nearest to the maximum.
  const float reach[8] = {0.f, 16.f, 11.f, 8.f, 5.5f, 3.5f, 1.75f, 0.5f};
  float mine = 0.f;
#pragma unroll
  for (int j = 1; j < 8; ++j)
    if ((lane & 7) == j) mine = reach[j];
  uint32_t guess = L::key_near(m - mine * temperature);
  if (guess > top) guess = top;

  uint32_t cut = 0;    // keys above it are kept
  uint64_t ties = 0;   // and so many of those equal to it, by index
  const bool by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
  if (by_k || by_p) {
    uint64_t s = pass(by_k, (lane & 7) == 0 ? 1u : guess);
    if (ex.dead) return ex.leave();
    const uint64_t need = by_k ? (uint64_t)k : need_of(p, shfl64(s, 0));
    // ---- few enough at or above the threshold that holds enough: one CTA takes them ----
    const uint32_t enough = __ballot_sync(kAll, lane >= 1 && lane < 8 && s >= need) | 1u;
    const int j = 31 - __clz(enough);
    const uint32_t floor_key = j == 0 ? 1u : __shfl_sync(kAll, guess, j);
    const int owner = static_cast<int>(row % a.cluster);
    uint32_t slots = 0;
#pragma unroll
    for (int c = 0; c < PER; ++c) slots |= (key[c] >= floor_key ? 1u : 0u) << c;
    const uint64_t found[1] = {(uint64_t)__popc(slots)};
    const uint64_t total_n = shfl64(ex.sum(found), 0);
    if (ex.dead) return ex.leave();
    if (total_n <= kList) {
      uint32_t base = 0;  // of this CTA's places
      for (int r = 0; r < ex.rank; ++r) base += (uint32_t)ex.slot(r, 0);
      if (slots) {
        uint32_t at = base + atomicAdd(&s_few, __popc(slots));
        uint32_t* keys = cluster.map_shared_rank(s_all, owner);
        uint32_t* indices = cluster.map_shared_rank(s_index, owner);
#pragma unroll
        for (int c = 0; c < PER; ++c)
          if (slots >> c & 1) {
            keys[at] = key[c];
            indices[at] = first + c / kVec * 32 * kVec + c % kVec;
            ++at;
          }
      }
      cluster.sync();
      if (ex.rank == owner)
        finish_few<kThreads, kList>(a, row, (int)total_n, s_all, s_index, s_weight, by_k ? k : 0, p,
                                    min_p, by_k ? 0ull : need, u, exp_of, &s_warp[0][0]);
      return;
    }
    // ---- top-k: keys above the cut, and the first `ties` of those equal to it ----
    if (by_k) {
      const Bound b = search(true, k, 1, top + 1, guess, s);
      if (ex.dead) return ex.leave();
      cut = b.key;
      ties = k - b.above;
    }
    // ---- top-p ----
    if (by_p) {
      if (by_k) s = pass(false, (lane & 7) == 0 ? cut + 1 : guess);
      if (ex.dead) return ex.leave();
      const uint64_t total = shfl64(s, 0) + ties * (cut ? weight(exp_of(cut)) : 0ull);
      const uint64_t want = need_of(p, total);
      const Bound b = search(false, want, cut ? cut : 1u, top + 1, guess, s);
      if (ex.dead) return ex.leave();
      const uint64_t w = weight(exp_of(b.key));
      const uint64_t n = (want - b.above + w - 1) / w;
      ties = b.key == cut && n > ties ? ties : n;
      cut = b.key;
    }
  }
  // ---- what is kept, per warp and CTA ----
  auto keeps = [&](uint32_t kk) {  // the weight of a key above the cut, if it is kept
    const float e = exp_of(kk);
    return e >= min_p ? weight(e) : 0ull;
  };
  uint64_t sums[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < PER; ++c) {
    if (key[c] > cut) sums[0] += keeps(key[c]);
    if (key[c] == cut) ++sums[1];
  }
  ex.sum(sums);
  if (ex.dead) return ex.leave();
  const uint64_t w_cut = cut ? keeps(cut) : 0ull;
  auto place = [&](uint64_t w, uint64_t equal, uint64_t ahead) {
    return place_pieces(w, equal, ahead, ties, w_cut);
  };
  const bool is_cta = lane < a.cluster;
  const Piece ctas = place(is_cta ? ex.slot(lane, 0) : 0ull, is_cta ? ex.slot(lane, 1) : 0ull, 0);
  const uint64_t total = ctas.all, r = draw_of(u, total);
  const uint64_t cta_before = shfl64(ctas.before, ex.rank), cta_own = shfl64(ctas.own, ex.rank);
  if (r < cta_before || r >= cta_before + cta_own) return;
  // ---- the CTA that holds the token: its warp, step, lane, element ----
  const bool is_warp = lane < kWarps;
  const Piece warps = place(is_warp ? s_warp[lane][0] : 0ull, is_warp ? s_warp[lane][1] : 0ull,
                            shfl64(ctas.ties_before, ex.rank));
  uint64_t run = cta_before + shfl64(warps.before, warp);
  uint64_t ties_before = shfl64(warps.ties_before, warp);
  const uint64_t warp_own = shfl64(warps.own, warp);
  if (r < run || r >= run + warp_own) return;
#pragma unroll
  for (int i = 0; i < kIters; ++i) {
    uint64_t w[kVec], own = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const uint32_t kk = key[i * kVec + j];
      w[j] = kk > cut ? keeps(kk) : 0ull;
      own += w[j];
      equal += kk == cut;
    }
    const Piece lanes = place(own, equal, ties_before);
    uint64_t at = run + lanes.before, seen = lanes.ties_before;
    if (r >= at && r < at + lanes.own) {
      bool found = false;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if (key[i * kVec + j] == cut) {
          w[j] = seen < ties ? w_cut : 0ull;
          ++seen;
        }
        if (!found && r < at + w[j]) {
          found = true;
          a.tokens[row] = first + i * 32 * kVec + j;
          a.probs[row] = (float)(__ull2double_rn(w[j]) / __ull2double_rn(total));
        }
        at += w[j];
      }
    }
    run += lanes.all;
    if (r < run) return;
    ties_before = shfl64(lanes.ties_before + equal, 31);
  }
}

template <typename T, int PER>
bool sample_attr() {
  return cudaFuncSetAttribute(k_sample<T, PER>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) ==
             cudaSuccess &&
         cudaFuncSetAttribute(k_sample<T, PER>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              2 * kThreads * PER * 4) == cudaSuccess;
}

template <typename T, int PER>
int launch_sample(const SampleArgs& a, int64_t rows, cudaStream_t s) {
  if (!once_per_device(reinterpret_cast<const void*>(&sample_attr<T, PER>), &sample_attr<T, PER>))
    return MOE_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * a.cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 2 * kThreads * PER * 4;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, k_sample<T, PER>, a) != cudaSuccess) return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

// One CTA a row where rows are many or short.  Measured with mixed parameters, fp16,
// in a graph (cluster / one CTA, us): 1 x 16000 10.8 / 12.8, 2 x 16000 13.5 / 12.7,
// 16 x 16000 25.9 / 19.4; 1 x 32000 12.4 / 20.4, 8 x 32000 22.1 / 27.2, 16 x 32000
// 26.2 / 28.4, 24 x 32000 29.3 / 28.5, 40 x 32000 32.6 / 29.3; 16 x 65536 35.2 / 42.9,
// 32 x 65536 44.3 / 42.8; 32 x 131072 58.9 / 74.4, 40 x 131072 68.6 / 74.4, 48 x 131072
// 79.9 / 75.4; 24 x 200000 90.8 / 108, 40 x 200000 140 / 110.  Between 11 and 21 rows of
// 32000, 22 and 30 of 65536 and 36 and 44 of 131072 the cluster is up to a fifth
// faster than the one CTA chosen here: the rule is from before one warp waited for an
// exchange.
// In a cluster 8 logits a thread, and so more CTAs, as far as 8 CTAs go; then 16
// (a cluster of up to 16 CTAs); 32 and one CTA to an SM for the longest rows.
template <typename T>
int launch_rows(SampleArgs& a, int64_t rows, cudaStream_t s) {
  if (a.vocab <= 16384 || rows >= 36 || rows * 3000 >= a.vocab) return launch_sample_rows<T>(a, rows, s);
  const int per = a.vocab <= 8 * kThreads * 8 ? 8 : a.vocab <= kMaxCluster * kThreads * 16 ? 16 : 32;
  a.cluster = a.vocab <= 8 * kThreads * per ? 8 : kMaxCluster;
  if (per == 8) return launch_sample<T, 8>(a, rows, s);
  if (per == 16) return launch_sample<T, 16>(a, rows, s);
  return launch_sample<T, 32>(a, rows, s);
}

}  // namespace
}  // namespace moe

extern "C" int moe_sample_tokens(const moe_sample_tokens_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_sample_tokens_args_t& c = *args;
  if (c.rows < 0 || c.vocab < 1 || (c.rows > 1 && c.stride != 0 && c.stride < c.vocab))
    return MOE_ERR_INVALID_ARG;
  if (c.dtype != MOE_DTYPE_F16 && c.dtype != MOE_DTYPE_BF16 && c.dtype != MOE_DTYPE_F32)
    return MOE_ERR_UNSUPPORTED;
  if (c.vocab > kMaxVocab) return MOE_ERR_UNSUPPORTED;
  if (c.rows == 0) return MOE_OK;
  if (!c.logits || !c.uniforms || !c.temperature || !c.top_k || !c.top_p || !c.min_p ||
      !c.tokens || !c.probs)
    return MOE_ERR_INVALID_ARG;
  SampleArgs a{c.logits, c.stride, (int)c.vocab, 1,        c.uniforms, c.temperature,
               c.top_p,  c.min_p,  c.top_k,      c.tokens, c.probs,    wait_limit_ns()};
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (c.dtype == MOE_DTYPE_F16) return launch_rows<F16>(a, c.rows, s);
  if (c.dtype == MOE_DTYPE_BF16) return launch_rows<BF16>(a, c.rows, s);
  return launch_rows<float>(a, c.rows, s);
}
