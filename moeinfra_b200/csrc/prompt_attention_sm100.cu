// Causal (or full) attention over packed prompts of different lengths, with
// grouped heads, on the 5th-generation tensor cores.
//
//   o[t, h] = sum_j softmax_j(scale q[t,h] . k_j) v_j
//
// over the keys j of t's sequence, j <= t + (len_k - len_q) if causal: the
// queries are the last len_q of len_k positions (len_k < len_q leaves the
// first rows without keys: zeros).
//
// One pass over the keys with the softmax's running maximum m and sum l.  A
// persistent CTA per SM walks items of 256 rows, the longest first.  The rows
// are the queries of neighbouring tokens of one sequence for P heads of one KV
// head (P the largest power of two that divides the group, up to 16): with 4
// heads 64 tokens, so that a short prompt or a sequence's end leaves few rows
// empty and the causal edge cuts closer to it than 256 tokens would.  An item
// is two tiles of 128 rows, so that one tile's softmax overlaps the other's
// products:
//   warps 0-3, 4-7  softmax of tile 0 and 1, one thread per row:
//                   S (tensor memory) -> registers, maximum, p = 2^(c s - c m),
//                   P (16 bits) -> tensor memory; at the end O / l
//   warp 8          lane 0 loads Q, K and V tiles with TMA (no multicast)
//   warps 9, 10     tcgen05.mma of tile 0 and 1: S = Q K^T (both from shared memory),
//                   O += P V (P from tensor memory, V as stored)
//   warp 11         looks the items up, some ahead of their use
//
// What bounds a step: 64 cycles of tensor core per 128 x 128 x 16 product
// (measured, both kinds), 16 exponentials a cycle, and the latency of the
// chain S -> softmax -> P -> products (about 400 cycles from issue to a
// waiting warp).  The chain is cut by giving P columns of its own: S is in
// registers after the first ~150 cycles of a softmax, and the next Q K^T is
// issued then, not after P V.  Tensor memory has 512 columns for two tiles'
// S, P and O: with head_dim 128 a step takes 80 keys (2 x (80 + 40 + 128)),
// with head_dim 64 96 keys (the softmax's registers hold no more).
//
// Measured in a graph of ten calls, 32 / 8 heads of 128, causal: one prompt of 8192,
// either type, 500 to 515 us (1.07 to 1.10 PFLOP/s, 77 to 79 % of what the library's best
// product sustains: the clock falls to 1.5-1.75 GHz under the power limit), 64 prompts of
// 129..512 120 us (412 MB and 61 GFLOP: an item has 3 to 7 steps, and as much again to
// start and to drain; 142 us call after call, at the lower clock), one of 2048 36 us,
// one of 40 7.4 us.  Heads of 64: 2 x 4096 bf16 203 us, fp16 231 (119 us of exponentials
// alone), 64 prompts of 129..512 bf16 101.
//
// O is rescaled only when a row's maximum grew by more than 2^8 since the
// reference in use (m is then that reference): probabilities stay below 2^8,
// O and l are sums of the same factor, and the quotient is exact either way.
//
// Barriers: q_full / q_empty, full / empty of the K and V ring, and per tile
// s_full (S computed), s_free (S read), p_ready (P stored, O rescaled), pv_done
// (P read, O updated).
// Every wait is bounded, as in the grouped GEMM: on a timeout the error word
// is set, the roles stop, and the CTA waits (bounded) for what it issued
// before it frees its tensor memory.
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

constexpr int kM = 128;         // rows of a tile
constexpr int kSoftWarps = 8, kTmaWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 12 * 32;  // three warpgroups: registers are moved between them
// Registers a thread: 12 warps x 168 at launch, of which the softmax warps
// (a row of 80 or 96 scores each) take kSoftRegs and the others keep kOtherRegs.
constexpr int kSoftRegs = 200, kOtherRegs = 104;
constexpr int kRegs = 2 * 128 * kSoftRegs + 128 * kOtherRegs;
constexpr float kLazy = 8.f;    // log2 of what a row's maximum may grow before O is rescaled
// P is rounded to 16 bits with m's reference up to 2^kLazy low: fp16 takes 2^7
// on top (2^15 fits, normal down to 2^-21 of the reference); bf16 needs none.
template <typename T>
constexpr float prob_shift() { return T::kBf16 ? 0.f : 7.f; }

template <int HD>
struct Cfg {
  static constexpr int kN = HD == 128 ? 80 : 96;              // keys of a step
  // A tile's 64 dims: rows of 128 bytes, in swizzled groups of 8 (1024 bytes).
  static constexpr uint32_t kHalfQ = kM * 128, kHalfK = kN * 128;
  static constexpr uint32_t kTileQ = kHalfQ * (HD / 64), kTileK = kHalfK * (HD / 64);
  static constexpr int kStages = HD == 128 ? 6 : 11;           // K and V tiles in flight
  // On its way out a softmax warp's O passes 32 rows x 64 dims of shared memory.
  static constexpr uint32_t kOut = 32 * 128;
  static constexpr uint32_t kSmem = 2 * kTileQ + kStages * kTileK + kSoftWarps * kOut + 1024;
  // TMEM columns of tile 0, and how much further tile 1's are.
  static constexpr uint32_t kS = 0, kS1 = kN, kP = 2 * kN, kP1 = (kN / 2 + 15) / 16 * 16;
  static constexpr uint32_t kO = 512 - 2 * HD, kO1 = HD;
  static_assert(kP + 2 * kP1 <= kO, "TMEM columns");
  static_assert(kSmem + 1024 <= 227 * 1024, "shared memory");
};

struct PromptArgs {
  const int32_t *cu_q, *cu_k;
  int64_t rows_q, rows_k;       // rows of q, and of k and v
  int seqs, heads, group;       // group: query heads per KV head
  int pack;                     // log2 of the heads that share a tile
  int max_q, max_k;
  int blocks;                   // ceil(max_q / tokens of an item)
  bool causal;
  float scale_log2;
  const uint16_t *q, *k, *v;    // for redo_rows alone; strides in elements
  int64_t q_stride, q_head, k_stride, k_head, v_stride, v_head;
  uint16_t* out;                // [rows_q, heads, HD]
  uint32_t* counts;             // items claimed, CTAs done: zero between calls
  uint64_t wait_ns;
};

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  return mbar_wait_or(bar, parity, limit_ns, [] { set_device_error(kErrWaitTimeout); });
}
// A whole warp's wait, with one result for all lanes.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  return mbar_poll_or(bar, parity, limit_ns, [] { set_device_error(kErrWaitTimeout); });
}

// fp32 accumulate, M = 128; b_rows: B is stored along N (V) instead of K.
template <typename T>
__device__ __forceinline__ uint32_t instr_desc(int n, bool b_rows) {
  const uint32_t ab = T::kBf16 ? ((1u << 7) | (1u << 10)) : 0u;
  return (1u << 4) | ab | ((b_rows ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kM >> 4) << 24);
}

// Two fp32 values in one 64-bit register pair: Blackwell's packed arithmetic
// takes one issue slot for both.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ uint64_t exp2_mufu(uint64_t x) {
  return pair(exp2_approx(lo_of(x)), exp2_approx(hi_of(x)));
}
// 2^x of a pair in ordinary arithmetic: x = n + f with n = round(x) (adding
// 1.5 * 2^23 leaves n in the low bits of the sum) and |f| <= 1/2, 2^f by its
// minimax polynomial, n added to the exponent.  Coefficients: Remez exchange
// on the relative error over [-1/2, 1/2]; degree 3 is off by at most 7.5e-5 (a
// bf16 probability rounds by 2e-3), degree 4 by 2.6e-6 (fp16: 4.9e-4).
// 2^n is a factor of its own, its exponent's bits from n + 127: arguments of -127
// and below (a masked score, -inf) give 0, NaN and +inf give NaN.
template <typename T>
__device__ __forceinline__ uint64_t exp2_fma(uint64_t x) {
  constexpr float kBig = 12582912.f;
  x = pair(max_nan(lo_of(x), -127.f), max_nan(hi_of(x), -127.f));
  const uint64_t r = add2(x, pair(kBig, kBig));
  const uint64_t n = add2(r, pair(-kBig, -kBig));
  const uint64_t f = fma2(n, pair(-1.f, -1.f), x);
  uint64_t p;
  if constexpr (T::kBf16) {
    p = fma2(pair(0.0551716691f, 0.0551716691f), f, pair(0.242611122f, 0.242611122f));
    p = fma2(p, f, pair(0.693260985f, 0.693260985f));
    p = fma2(p, f, pair(0.999928074f, 0.999928074f));
  } else {
    p = fma2(pair(0.00957010201f, 0.00957010201f), f, pair(0.0559178603f, 0.0559178603f));
    p = fma2(p, f, pair(0.240247448f, 0.240247448f));
    p = fma2(p, f, pair(0.693121815f, 0.693121815f));
    p = fma2(p, f, pair(0.999999261f, 0.999999261f));
  }
  const uint32_t lo = ((uint32_t)r << 23) + 0x3F800000u;
  const uint32_t hi = ((uint32_t)(r >> 32) << 23) + 0x3F800000u;
  return mul2(p, pair(__uint_as_float(lo), __uint_as_float(hi)));
}
// Of 8 pairs, those that go through exp2_fma.  With heads of 128 the tensor cores
// (and the power limit) bound a step and it only costs: 1 x 8192 causal fp16, at the
// full clock, 450 us with none, 454 with 1, 461 with 2, 495 with 4.  With heads of 64 a
// step has twice the exponentials per product: 2 x 4096 fp16 215, 207, 210, 241 us.
template <int HD>
constexpr int kFmaOf8 = HD == 128 ? 0 : 1;

// kN consecutive columns of the thread's own lane.
template <int N>
__device__ __forceinline__ void load_cols(uint32_t at, uint32_t* v) {
#pragma unroll
  for (int c = 0; c < N / 32 * 32; c += 32) tmem_ld32(at + c, v + c);
  if constexpr (N % 32 == 16) tmem_ld16(at + N / 32 * 32, v + N / 32 * 32);
}
template <int N>
__device__ __forceinline__ void store_cols(uint32_t at, const uint32_t* v) {
#pragma unroll
  for (int c = 0; c < N / 32 * 32; c += 32) tmem_st32(at + c, v + c);
  if constexpr (N % 32 == 8) tmem_st8(at + N / 32 * 32, v + N / 32 * 32);
  if constexpr (N % 32 == 16) tmem_st16(at + N / 32 * 32, v + N / 32 * 32);
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

// kRedo rows of one KV head by the formula, by one warp: 32 keys a step, one to a
// lane, then their values, HD / 32 dims to a lane.  q, out: the rows' queries and
// places; k, v: the first key and value; seen: how many of them each row sees (0: no
// row).  A warp's 32 rows over 8192 keys take 13 ms, over 131072 0.2 s, latency of
// loads mostly: the other warps' waits end after 2 s.
constexpr int kRedo = 4;
template <typename T, int HD>
__device__ __forceinline__ void redo_rows(const uint16_t* const (&q)[kRedo], const uint16_t* k,
                                          int64_t k_stride, const uint16_t* v, int64_t v_stride,
                                          const int (&seen)[kRedo], float scale_log2,
                                          uint16_t* const (&out)[kRedo]) {
  constexpr int kWords = HD / 64;
  const int lane = threadIdx.x & 31;
  float m[kRedo], l[kRedo];
  float2 acc[kRedo][kWords] = {};
  int most = 0;
#pragma unroll
  for (int r = 0; r < kRedo; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
    most = max(most, seen[r]);
  }
#pragma unroll 1
  for (int j0 = 0; j0 < most; j0 += 32) {
    const int j = j0 + lane;
    float s[kRedo] = {};
    const uint16_t* row = k + min(j, most - 1) * k_stride;
#pragma unroll 4
    for (int d = 0; d < HD; d += 8) {
      const uint4 ks = *reinterpret_cast<const uint4*>(row + d);
      const uint32_t kw[4] = {ks.x, ks.y, ks.z, ks.w};
#pragma unroll
      for (int r = 0; r < kRedo; ++r) {
        const uint4 qs = *reinterpret_cast<const uint4*>(q[r] + d);
        const uint32_t qw[4] = {qs.x, qs.y, qs.z, qs.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 x = T::unpack(qw[i]), y = T::unpack(kw[i]);
          s[r] = fmaf(x.x, y.x, fmaf(x.y, y.y, s[r]));
        }
      }
    }
    bool nan = true;
#pragma unroll
    for (int r = 0; r < kRedo; ++r) {
      s[r] = j < seen[r] ? s[r] * scale_log2 : -INFINITY;
      float top = s[r];
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float nm = fmaxf(m[r], top), f = m[r] == nm ? 1.f : exp2_approx(m[r] - nm);
      m[r] = nm;
      s[r] = exp2_approx(s[r] - (nm == -INFINITY ? 0.f : nm));
      l[r] = l[r] * f + warp_sum(s[r]);
      nan &= l[r] != l[r] || seen[r] == 0;
#pragma unroll
      for (int w = 0; w < kWords; ++w) acc[r][w] = make_float2(acc[r][w].x * f, acc[r][w].y * f);
    }
    if (nan) break;  // and they stay so
    const int n = min(32, most - j0);
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
      float2 x[kWords];
#pragma unroll
      for (int w = 0; w < kWords; ++w)
        x[w] = T::unpack(
            *reinterpret_cast<const uint32_t*>(v + (j0 + i) * v_stride + w * 64 + lane * 2));
#pragma unroll
      for (int r = 0; r < kRedo; ++r) {
        const float p = __shfl_sync(0xffffffffu, s[r], i);
        if (j0 + i >= seen[r]) continue;
#pragma unroll
        for (int w = 0; w < kWords; ++w)
          acc[r][w] = make_float2(fmaf(p, x[w].x, acc[r][w].x), fmaf(p, x[w].y, acc[r][w].y));
      }
    }
  }
#pragma unroll
  for (int r = 0; r < kRedo; ++r) {
    if (seen[r] == 0) continue;
    const float inv = 1.f / l[r];
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      *reinterpret_cast<uint32_t*>(out[r] + w * 64 + lane * 2) =
          T::pack(acc[r][w].x * inv, acc[r][w].y * inv);
  }
}

struct __align__(16) Item {
  int h, q0;            // first head (-1: no more items), first token in the sequence
  int len_q, len_k;
  int row_q, row_k;     // the sequence's first rows
  int steps0, steps1;   // key steps of tile 0 and 1
};
constexpr int kItems = 1;                   // items looked up ahead
constexpr int kReaders = kSoftWarps + 3;    // warps that read each of them

// A sequence's first rows and lengths; false, with the error bit set, if its offsets
// do not describe rows of q and k or it is longer than the call said.
__device__ __forceinline__ bool get_sequence(const PromptArgs& a, uint32_t b, Item& it) {
  const int q_lo = a.cu_q[b], q_hi = a.cu_q[b + 1], k_lo = a.cu_k[b], k_hi = a.cu_k[b + 1];
  it.len_q = q_hi - q_lo;
  it.len_k = k_hi - k_lo;
  it.row_q = q_lo;
  it.row_k = k_lo;
  if (q_lo < 0 || q_hi < q_lo || q_hi > a.rows_q || k_lo < 0 || k_hi < k_lo || k_hi > a.rows_k ||
      it.len_q > a.max_q || it.len_k > a.max_k) {
    set_device_error(kErrPage);
    return false;
  }
  return true;
}

// Block x of the launch (all heads of 256 >> pack tokens of a sequence, the last
// tokens first); false where the sequence has no such block, or counts as empty.
template <int HD>
__device__ __forceinline__ bool get_block(const PromptArgs& a, uint32_t x, Item& it) {
  const uint32_t blk = x / a.seqs, b = x - blk * a.seqs;
  const int tokens = kM >> a.pack;
  it.q0 = (a.blocks - 1 - (int)blk) * 2 * tokens;
  if (!get_sequence(a, b, it) || it.q0 >= it.len_q) return false;
  constexpr int kN = Cfg<HD>::kN;
  auto steps = [&](int first) {
    int keys = it.len_k;
    if (a.causal) keys = min(keys, min(first + tokens, it.len_q) + it.len_k - it.len_q);
    return first < it.len_q && keys > 0 ? (keys + kN - 1) / kN : 0;
  };
  it.steps0 = steps(it.q0);
  it.steps1 = steps(it.q0 + tokens);
  return true;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    k_prompt_attention(const PromptArgs a, const __grid_constant__ CUtensorMap map_q,
                       const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v,
                       const __grid_constant__ CUtensorMap map_o) {
  using C = Cfg<HD>;
  constexpr int NS = C::kStages, kN = C::kN;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t s_qfull, s_qempty, s_full[NS], s_empty[NS], s_sfull[2],
      s_sfree[2], s_pready[2], s_pvdone[2], s_tail, s_drain[2],
      s_itfull[kItems], s_itempty[kItems];
  __shared__ Item s_item[kItems];
  __shared__ uint32_t s_tmem;
  __shared__ int2 s_keys[kSoftWarps];  // first row and number of the keys a softmax warp is at
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (saddr(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_at = base, ring = base + 2 * C::kTileQ;

  if (threadIdx.x == 0) {
    mbar_init(saddr(&s_qfull), 1);
    mbar_init(saddr(&s_qempty), 2);
    for (int i = 0; i < NS; ++i) {
      mbar_init(saddr(&s_full[i]), 1);
      mbar_init(saddr(&s_empty[i]), 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(saddr(&s_sfull[t]), 1);
      mbar_init(saddr(&s_sfree[t]), 4);
      mbar_init(saddr(&s_pready[t]), 4);
      mbar_init(saddr(&s_pvdone[t]), 1);
      mbar_init(saddr(&s_drain[t]), 1);
    }
    mbar_init(saddr(&s_tail), 1);
    for (int i = 0; i < kItems; ++i) {
      mbar_init(saddr(&s_itfull[i]), 1);
      mbar_init(saddr(&s_itempty[i]), kReaders);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // The items of this CTA in order, from the look-up warp; the same for every
  // reading warp.  False at the end or after a timeout.
  Item it;
  uint32_t n_it = 0;
  auto next_item = [&]() {
    const uint32_t i = n_it % kItems;
    if (!warp_wait(saddr(&s_itfull[i]), n_it / kItems & 1, a.wait_ns)) {
      s_abort = 1;
      return false;
    }
    it = s_item[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(saddr(&s_itempty[i]));
    ++n_it;
    return it.h >= 0 && !__any_sync(0xffffffffu, s_abort);
  };

  if (warp < kSoftWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // ---------------- softmax: one thread per row of tile t ----------------
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + C::kS + t * C::kS1 + lane_base;
    const uint32_t p_at = tmem + C::kP + t * C::kP1 + lane_base;
    const uint32_t o_at = tmem + C::kO + t * C::kO1 + lane_base;
    const uint32_t stage = base + 2 * C::kTileQ + NS * C::kTileK + warp * C::kOut;
    uint32_t n_s = 0, n_pv = 0;  // phases of s_full and pv_done
    while (next_item()) {
      const int first = it.q0 + t * (kM >> a.pack), q = first + (row >> a.pack);  // the row's token
      if (first >= it.len_q) continue;
      const int steps = t ? it.steps1 : it.steps0;
      if (lane == 0) s_keys[warp] = make_int2(it.row_k, it.len_k);
      // Keys this row sees.
      const int seen = a.causal ? min(it.len_k, q + 1 + it.len_k - it.len_q) : it.len_k;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < steps; ++j) {
        if (!warp_wait(saddr(&s_sfull[t]), n_s++ & 1, a.wait_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[kN];
        load_cols<kN>(s_at, s);
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_sfree[t]));
        const int vis = seen - j * kN;
        if (__any_sync(0xffffffffu, vis < kN)) {
#pragma unroll
          for (int c = 0; c < kN; ++c)
            if (c >= vis) s[c] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < kN; c += 2)
          mx[c / 2 & 3] = max3(mx[c / 2 & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
        // P's columns and O are free once the previous product is done.
        if (j > 0) {
          if (!warp_wait(saddr(&s_pvdone[t]), n_pv++ & 1, a.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, top > m + (m == -INFINITY ? 0.f : kLazy))) {
          const float nm = fmaxf(m, top);
          const float f = m == nm ? 1.f : exp2_approx(m - nm);
          m = nm;
          l *= f;
          if (j > 0) {
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
          const uint64_t e = c / 2 % 8 < kFmaOf8<HD> ? exp2_fma<T>(x) : exp2_mufu(x);
          sum[c / 2 & 1] = add2(sum[c / 2 & 1], e);
          p[c / 2] = T::pack(lo_of(e), hi_of(e));
        }
        store_cols<kN / 2>(p_at, p);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(saddr(&s_pready[t]));
        sum[0] = add2(sum[0], sum[1]);
        l += lo_of(sum[0]) + hi_of(sum[0]);
      }
      if (ok && steps > 0) ok = warp_wait(saddr(&s_pvdone[t]), n_pv++ & 1, a.wait_ns);
      if (!ok) {
        s_abort = 1;
        break;
      }
      tc_fence_after();
      // A row without keys is zeros.  With keys l is above 0, unless every score is
      // -inf (0 / 0), and NaN where one is NaN or +inf: the row then is NaN.
      const bool blind = steps == 0 || seen <= 0;
      const float inv = __fdividef(1.f, l);
      // A thread holds a row; written out that way every 16 bytes would touch a
      // line of its own.  64 dims at a time the warp's 32 rows cross shared
      // memory (in the swizzle that the TMA store undoes); where the sequence
      // ends among them the lanes write whole 128-byte lines themselves.
      const int lane_row = (warp & 3) * 32, heads_mask = (1 << a.pack) - 1;
      const int warp_token = first + (lane_row >> a.pack);
      const bool whole = warp_token + (32 >> a.pack) <= it.len_q;
      const uint64_t inv2 = pair(inv, inv);
      uint64_t odd[2] = {0, 0};  // sums of products of O: not finite once an element is not
#pragma unroll 1
      for (int c = 0; c < HD; c += 64) {
        uint32_t w[32];
#pragma unroll
        for (int hf = 0; hf < 64; hf += 32) {
          uint32_t o[32];
          if (steps > 0) {
            tmem_ld32(o_at + c + hf, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const uint64_t x = pair(__uint_as_float(o[2 * i]), __uint_as_float(o[2 * i + 1]));
            const uint64_t y = pair(__uint_as_float(o[2 * i + 2]), __uint_as_float(o[2 * i + 3]));
            odd[i / 2 & 1] = fma2(x, y, odd[i / 2 & 1]);
            const uint64_t xs = mul2(x, inv2), ys = mul2(y, inv2);
            w[hf / 2 + i] = blind ? 0u : T::pack(lo_of(xs), hi_of(xs));
            w[hf / 2 + i + 1] = blind ? 0u : T::pack(lo_of(ys), hi_of(ys));
          }
        }
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the last store read it
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 +
                                                                        ((i ^ (lane & 7)) << 4)),
                       "r"(w[4 * i]), "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3])
                       : "memory");
        if (whole) {
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&map_o, stage, c, it.h + (lane_row & heads_mask), it.row_q + warp_token);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
          continue;
        }
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
          const int r = i * 4 + (lane >> 3), col8 = lane & 7;
          const int token = first + ((lane_row + r) >> a.pack), head = it.h + (r & heads_mask);
          uint4 w;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                       : "r"(stage + r * 128 + ((col8 ^ (r & 7)) << 4))
                       : "memory");
          if (token < it.len_q)
            *reinterpret_cast<uint4*>(a.out + ((int64_t)(it.row_q + token) * a.heads + head) * HD +
                                      c + col8 * 8) = w;
        }
      }
      // A probability of 0 does not silence an infinity or NaN among the values of
      // a key that this row does not see and others of the tile do.  Rows that may
      // have met one are computed again without the tile.  Looking costs 1 % (64
      // prompts of 129..512: 119.6 -> 120.7 us in a graph; heads of 64 99 -> 101).
      const uint64_t both = add2(odd[0], odd[1]);
      const bool finite = fabsf(lo_of(both)) + fabsf(hi_of(both)) < INFINITY;
      uint32_t again = __ballot_sync(0xffffffffu, !finite && !blind && q < it.len_q);
      if (again) {
        __syncwarp();
        const int2 keys = s_keys[warp];  // kept out of the registers until here
        const int loaded = min(steps * kN, keys.y), kv_head = it.h / a.group;
        const uint16_t* v = a.v + keys.x * a.v_stride + kv_head * a.v_head;
        again &= __ballot_sync(0xffffffffu, seen < loaded);
        const int from = __reduce_min_sync(0xffffffffu, again >> lane & 1 ? seen : loaded);
        uint32_t met = 0;
        for (int i = lane; i < (loaded - from) * (HD / 2); i += 32)  // at most a tile and a step
          met = trace_odd<T>(*reinterpret_cast<const uint32_t*>(
                                 v + (from + i / (HD / 2)) * a.v_stride + i % (HD / 2) * 2), met);
        if (!__any_sync(0xffffffffu, met)) again = 0;
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the rows are written once more
        __syncwarp();
        while (again) {
          const uint16_t* qs[kRedo];
          uint16_t* outs[kRedo];
          int sees[kRedo];
#pragma unroll
          for (int i = 0; i < kRedo; ++i) {  // past the last: the first row, seeing nothing
            const int r = again ? __ffs(again) - 1 : 0;
            const int64_t at = it.row_q + first + ((lane_row + r) >> a.pack);
            const int head = it.h + (r & heads_mask);
            qs[i] = a.q + at * a.q_stride + head * a.q_head;
            outs[i] = a.out + (at * a.heads + head) * HD;
            sees[i] = __shfl_sync(0xffffffffu, again ? seen : 0, r);
            again &= again - 1;
          }
          redo_rows<T, HD>(qs, a.k + keys.x * a.k_stride + kv_head * a.k_head, a.k_stride, v,
                           a.v_stride, sees, a.scale_log2, outs);
        }
      }
      tc_fence_before();
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  } else {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == kTmaWarp) {
    // ---------------- TMA producer ----------------
    // Q, K(0), then K(j + 1), V(j): the order of use.
    uint32_t g = 0, n_q = 0, n_tail = 0;
    bool ok = true;
    int kv_head = 0;
    auto load = [&](bool is_v, int j) {
      const int s = g % NS;
      ok = ok && warp_wait(saddr(&s_empty[s]), ((g / NS) & 1) ^ 1, a.wait_ns);
      if (!ok) return;
      ++g;
      const uint32_t dst = ring + s * C::kTileK, full = saddr(&s_full[s]);
      // Rows past the sequence's last key belong to the next one: scores of
      // such keys are dropped, but a probability of 0 does not silence an
      // infinity or NaN among their values.  Those rows become zeros before
      // the tile is handed on.
      const int rows = it.len_k - j * kN;
      const bool tail = is_v && rows < kN;
      if (lane == 0) {
        const uint32_t bar = tail ? saddr(&s_tail) : full;
        mbar_expect_tx(bar, C::kTileK);
        for (int hf = 0; hf < HD / 64; ++hf)
          tma_load_3d(dst + hf * C::kHalfK, is_v ? &map_v : &map_k, bar, hf * 64, kv_head,
                      it.row_k + j * kN);
      }
      if (!tail) return;
      ok = warp_wait(saddr(&s_tail), n_tail++ & 1, a.wait_ns);
      if (!ok) return;
      for (int hf = 0; hf < HD / 64; ++hf)
        for (uint32_t z = rows * 128 + lane * 16; z < C::kHalfK; z += 512)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + hf * C::kHalfK + z),
                       "r"(0)
                       : "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    };
    while (ok && next_item()) {
      const int steps = max(it.steps0, it.steps1);
      if (steps == 0) continue;
      kv_head = it.h / a.group;
      ok = warp_wait(saddr(&s_qempty), (n_q++ & 1) ^ 1, a.wait_ns);
      if (!ok) break;
      if (lane == 0) {
        const uint32_t bar = saddr(&s_qfull);
        mbar_expect_tx(bar, ((it.steps0 > 0) + (it.steps1 > 0)) * C::kTileQ);
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if ((t ? it.steps1 : it.steps0) > 0)
            for (int hf = 0; hf < HD / 64; ++hf)
              tma_load_3d(q_at + t * C::kTileQ + hf * C::kHalfQ, &map_q, bar, hf * 64, it.h,
                          it.row_q + it.q0 + t * (kM >> a.pack));
      }
      load(false, 0);
      for (int j = 0; j < steps; ++j) {
        if (j + 1 < steps) load(false, j + 1);
        load(true, j);
      }
    }
    if (!ok) s_abort = 1;
    // Copies issued into stages never consumed (timeout): let them land.
    if (s_abort && lane == 0) {
      for (uint32_t j = g > (uint32_t)NS ? g - NS : 0; j < g; ++j)
        mbar_wait(saddr(&s_full[j % NS]), (j / NS) & 1, a.wait_ns);
      if (n_q > 0) mbar_wait(saddr(&s_qfull), (n_q - 1) & 1, a.wait_ns);
    }
  } else if (warp == kMmaWarp || warp == kMmaWarp + 1) {
    // ---------------- MMA issuers: one warp per tile ----------------
    // The whole warp walks the loop and one elected lane issues: addresses and
    // descriptors are then uniform over the warp and stay in uniform registers
    // (with one lane in the branch each instruction took ~150 cycles to issue).
    // A warp of its own per tile: between two products there are ~100
    // instructions of waits and bookkeeping, which share issue slots with the
    // softmax warps, and one tile's waits do not hold up the other's products.
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
    auto product_qk = [&](uint32_t k) {  // S, once the last one is read
      if (n_qk > 0) ok = ok && warp_wait(saddr(&s_sfree[t]), (n_qk - 1) & 1, a.wait_ns);
      if (!ok) return;
      ++n_qk;
      tc_fence_after();
      const uint64_t kd = desc_k + k * (C::kTileK >> 4);
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
        tc_mma_if(leader, s_col, desc_q + ((kk / 4 * C::kHalfQ + kk % 4 * 32) >> 4),
                  kd + ((kk / 4 * C::kHalfK + kk % 4 * 32) >> 4), d_qk, kk != 0);
      tc_commit_if(leader, saddr(&s_sfull[t]));
    };
    auto product_pv = [&](uint32_t v, bool first) {
      ok = ok && warp_wait(saddr(&s_pready[t]), n_pv & 1, a.wait_ns);
      if (!ok) return;
      ++n_pv;
      tc_fence_after();
      const uint64_t vd = desc_v + v * (C::kTileK >> 4);
      const uint32_t add = first ? 0 : 1;
      tc_mma_ta_if(leader, o_col, p_col, vd, d_pv, add);
#pragma unroll
      for (int kk = 1; kk < kN / 16; ++kk)
        tc_mma_ta_if(leader, o_col, p_col + kk * 8, vd + (kk * 2048 >> 4), d_pv, 1);
      tc_commit_if(leader, saddr(&s_pvdone[t]));
    };
    // A slot is released by both warps, after the last product that reads it.
    while (ok && next_item()) {
      const int mine = __shfl_sync(0xffffffffu, t ? it.steps1 : it.steps0, 0);
      const int both = __shfl_sync(0xffffffffu, max(it.steps0, it.steps1), 0);
      if (both == 0) continue;
      ok = warp_wait(saddr(&s_qfull), n_q++ & 1, a.wait_ns);
      for (int j = -1; j < both; ++j) {  // Q K^T of step j + 1, P V of step j
        if (j + 1 < both) {
          const uint32_t k = next();
          if (ok && j + 1 < mine) product_qk(k);
          if (!ok) break;
          tc_commit_if(leader, saddr(&s_empty[k]));
          if (j + 2 == both) tc_commit_if(leader, saddr(&s_qempty));
        }
        if (j < 0) continue;
        const uint32_t v = next();
        if (ok && j < mine) product_pv(v, j == 0);
        if (!ok) break;
        tc_commit_if(leader, saddr(&s_empty[v]));
      }
    }
    if (!ok) s_abort = 1;
    // After a timeout, wait (bounded) for the MMAs already issued.
    if (__any_sync(0xffffffffu, s_abort)) {
      tc_commit_if(leader, saddr(&s_drain[t]));
      warp_wait(saddr(&s_drain[t]), 0, a.wait_ns);
    }
  } else {
    // ---------------- look-up of the items ----------------
    // Items are the head groups of each block that has rows, in order.  A CTA
    // starts with the item of its own number and claims further ones from a
    // counter as it goes: lengths and clocks differ too much for a fixed share
    // (64 prompts of 129 to 512 tokens: 138 us, 103 of them at the median CTA).
    // To find an item's block, every CTA walks the blocks, 32 at a time, and
    // counts those with rows.  After some without any it looks for the next that has
    // (the stated maximum may be far above the lengths, or one sequence above the
    // others: 1000 prompts of 1..64, 16 heads of 64, stated as up to 131072, took 60 ms
    // and take 0.09; 64 prompts of 129..512 1.08 and 0.12).
    const uint32_t groups = a.heads >> a.pack, blocks = (uint32_t)a.blocks * a.seqs;
    constexpr int kEmpty = 4;  // looks without a block before the next is searched for
    uint32_t n = 0, n_q = 0, at = 0, before = 0, live = 0;
    int empty = 0;
    bool ok = true, mine = false;
    auto look = [&]() {  // the next 32 blocks
      mine = at + lane < blocks && get_block<HD>(a, at + lane, it);
      live = __ballot_sync(0xffffffffu, mine);
      at += 32;
    };
    auto skip = [&]() {  // from block `at` to the next that has rows
      const uint32_t tokens = 2 * kM >> a.pack;
      uint32_t next = blocks;
      for (uint32_t b = lane; b < (uint32_t)a.seqs; b += 32) {
        Item one;
        if (!get_sequence(a, b, one)) continue;
        const uint32_t first = a.blocks - ((uint32_t)one.len_q + tokens - 1) / tokens;
        const uint32_t blk = max(first, at > b ? (at - b + a.seqs - 1) / a.seqs : 0u);
        if (blk < (uint32_t)a.blocks) next = min(next, blk * a.seqs + b);
      }
      at = __reduce_min_sync(0xffffffffu, next);
    };
    auto push = [&](uint32_t from) {  // lane `from` hands its item on
      ok = ok && warp_wait(saddr(&s_itempty[n % kItems]), (n / kItems & 1) ^ 1, a.wait_ns);
      if (!ok) return;
      if (lane == (int)from) {
        s_item[n % kItems] = it;
        mbar_arrive(saddr(&s_itfull[n % kItems]));
      }
      ++n;
    };
    uint32_t y = blockIdx.x;
    look();
    while (ok && !__any_sync(0xffffffffu, s_abort)) {
      const uint32_t block = y / groups;
      while (block >= before + __popc(live) && at < blocks) {
        before += __popc(live);
        empty = live ? 0 : empty + 1;
        if (empty == kEmpty) {
          skip();
          empty = 0;
        }
        look();
      }
      if (block >= before + __popc(live)) break;
      it.h = (y - block * groups) << a.pack;
      const uint32_t from = __ffs(__ballot_sync(
          0xffffffffu, mine && __popc(live & ((1u << lane) - 1)) == block - before)) - 1;
      push(from);
      const int steps = __shfl_sync(0xffffffffu, max(it.steps0, it.steps1), from);
      // In the last rounds an item is claimed late, once the one at hand has
      // issued its last Q K^T: a claim made early binds it to a busy CTA (one
      // prompt of 2048: 47 us early, 39 late).
      if (steps > 0) ++n_q;
      if (steps > 0 && y + 2 * gridDim.x > blocks * groups)
        ok = ok && warp_wait(saddr(&s_qempty), (n_q - 1) & 1, a.wait_ns);
      if (lane == 0) y = gridDim.x + atomicAdd(a.counts, 1);
      y = __shfl_sync(0xffffffffu, y, 0);
    }
    // The last CTA to get here sets the counters back: nobody claims any more.
    if (lane == 0) {
      __threadfence();
      if (atomicAdd(a.counts + 1, 1) == gridDim.x - 1) a.counts[0] = a.counts[1] = 0;
    }
    it.h = -1;
    it.steps0 = it.steps1 = 0;
    push(0);
    if (!ok) s_abort = 1;
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

// [rows, heads, HD] with any row and head strides (multiples of 16 bytes):
// boxes of box_rows rows x box_heads heads x 64 dims, 128-byte swizzle.
bool make_map(CUtensorMap* map, const uint16_t* x, int64_t rows, int heads, int hd, int64_t row_stride,
              int64_t head_stride, bool bf16, int box_rows, int box_heads) {
  auto fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)row_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
  const cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<uint16_t*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int HD>
bool prompt_attr() {
  // The warps' register shares must not exceed what the block is launched
  // with: the last to ask would wait for good.
  cudaFuncAttributes at;
  return cudaFuncGetAttributes(&at, k_prompt_attention<T, HD>) == cudaSuccess &&
         at.numRegs * kThreads >= kRegs &&
         cudaFuncSetAttribute(k_prompt_attention<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Cfg<HD>::kSmem) == cudaSuccess;
}

template <typename T, int HD>
int launch_prompt(const PromptArgs& a, const CUtensorMap& q, const CUtensorMap& k,
                  const CUtensorMap& v, const CUtensorMap& o, cudaStream_t s) {
  if (!once_per_device(reinterpret_cast<const void*>(&prompt_attr<T, HD>), &prompt_attr<T, HD>))
    return MOE_ERR_CUDA;
  const int64_t items = (int64_t)a.blocks * a.seqs * (a.heads >> a.pack);
  const int grid = static_cast<int>(items < sm_count() ? items : sm_count());
  if (launch_pdl(k_prompt_attention<T, HD>, dim3(grid), dim3(kThreads), Cfg<HD>::kSmem, s, a, q, k,
                 v, o) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

bool bad_strides(int64_t row, int64_t head, int64_t heads, int64_t hd) {
  return row < hd || (heads > 1 && head < hd);
}

}  // namespace
}  // namespace moe

extern "C" size_t moe_prompt_attention_workspace_size(void) { return 16; }

extern "C" int moe_prompt_attention(const moe_prompt_attention_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_prompt_attention_args_t& c = *args;
  const float scale = static_cast<float>(c.scale);
  // Rows, and so offsets and coordinates of a tile past the end, are 32-bit.
  constexpr int64_t kMostRows = INT32_MAX - 256;
  if (c.q_rows < 0 || c.k_rows < 0 || c.q_rows > kMostRows || c.k_rows > kMostRows || c.seqs < 0 ||
      c.max_q < 0 || c.max_k < 0 || c.max_q > INT32_MAX || c.max_k > INT32_MAX || c.heads < 1 ||
      c.heads > 4096 || c.kv_heads < 1 || c.heads % c.kv_heads || !(scale > 0.f && scale < INFINITY))
    return MOE_ERR_INVALID_ARG;
  if (c.dtype != MOE_DTYPE_F16 && c.dtype != MOE_DTYPE_BF16) return MOE_ERR_UNSUPPORTED;
  if (c.head_dim != 64 && c.head_dim != 128) return MOE_ERR_UNSUPPORTED;
  const int hd = static_cast<int>(c.head_dim), heads = static_cast<int>(c.heads);
  const int kv_heads = static_cast<int>(c.kv_heads);
  if (bad_strides(c.q_stride, c.q_head_stride, heads, hd) ||
      bad_strides(c.k_stride, c.k_head_stride, kv_heads, hd) ||
      bad_strides(c.v_stride, c.v_head_stride, kv_heads, hd))
    return MOE_ERR_INVALID_ARG;
  if (c.q_rows == 0 || c.seqs == 0 || c.max_q == 0) return MOE_OK;
  if (c.seqs > INT32_MAX / heads || ceil_div(c.max_q, 16) > INT32_MAX / (c.seqs * heads))
    return MOE_ERR_UNSUPPORTED;
  if (!c.q || !c.cu_q || !c.cu_k || !c.out || (c.k_rows > 0 && (!c.k || !c.v)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(c.q) || !aligned16(c.k) || !aligned16(c.v) || !aligned16(c.out) ||
      ((c.q_stride | c.q_head_stride | c.k_stride | c.k_head_stride | c.v_stride | c.v_head_stride) & 7))
    return MOE_ERR_ALIGNMENT;
  if (!c.workspace || c.workspace_bytes < (int64_t)moe_prompt_attention_workspace_size())
    return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  const bool bf16 = c.dtype == MOE_DTYPE_BF16;
  // Heads that share a tile's rows: see the kernel.
  int pack = 0;
  while (pack < 4 && heads / kv_heads % (2 << pack) == 0) ++pack;
  const int keys = hd == 64 ? Cfg<64>::kN : Cfg<128>::kN;
  // Without any key no K or V tile is loaded: the maps then describe q.
  const bool none = c.k_rows == 0;
  const uint16_t *k = none ? c.q : c.k, *v = none ? c.q : c.v;
  const int64_t k_rows = none ? c.q_rows : c.k_rows;
  const int map_heads = none ? heads : kv_heads;
  CUtensorMap mq, mk, mv, mo;  // mo: a warp's rows of the output, 32 / P tokens x P heads
  if (!make_map(&mq, c.q, c.q_rows, heads, hd, c.q_stride, c.q_head_stride, bf16, kM >> pack,
                1 << pack) ||
      !make_map(&mk, k, k_rows, map_heads, hd, none ? c.q_stride : c.k_stride,
                none ? c.q_head_stride : c.k_head_stride, bf16, keys, 1) ||
      !make_map(&mv, v, k_rows, map_heads, hd, none ? c.q_stride : c.v_stride,
                none ? c.q_head_stride : c.v_head_stride, bf16, keys, 1) ||
      !make_map(&mo, c.out, c.q_rows, heads, hd, (int64_t)heads * hd, hd, bf16, 32 >> pack,
                1 << pack))
    return MOE_ERR_CUDA;
  PromptArgs a{};
  a.cu_q = c.cu_q;
  a.cu_k = c.cu_k;
  a.rows_q = c.q_rows;
  a.rows_k = c.k_rows;
  a.seqs = static_cast<int>(c.seqs);
  a.heads = heads;
  a.group = heads / kv_heads;
  a.max_q = static_cast<int>(c.max_q);
  a.max_k = static_cast<int>(c.max_k);
  a.pack = pack;
  a.blocks = static_cast<int>(ceil_div(c.max_q, 2 * kM >> pack));
  a.causal = c.causal != 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.q = c.q;
  a.k = c.k;
  a.v = c.v;
  a.q_stride = c.q_stride;
  a.q_head = c.q_head_stride;
  a.k_stride = c.k_stride;
  a.k_head = c.k_head_stride;
  a.v_stride = c.v_stride;
  a.v_head = c.v_head_stride;
  a.out = c.out;
  a.counts = static_cast<uint32_t*>(c.workspace);
  a.wait_ns = wait_limit_ns();
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (bf16)
    return hd == 64 ? launch_prompt<BF16, 64>(a, mq, mk, mv, mo, s)
                    : launch_prompt<BF16, 128>(a, mq, mk, mv, mo, s);
  return hd == 64 ? launch_prompt<F16, 64>(a, mq, mk, mv, mo, s)
                  : launch_prompt<F16, 128>(a, mq, mk, mv, mo, s);
}
