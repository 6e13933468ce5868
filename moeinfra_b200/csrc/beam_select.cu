// Beam search's choice: the best continuations over beams and vocabulary.
//
// For beam k of a group with logits x and running score s_k, token t scores
//   v[k,t] = s_k + ((x_t - m) - ln sum_u exp(x_u - m)),   m = max_u x_u
// and the `count` largest of the group's beams x vocabulary are returned, larger
// scores first, then lower beams, in a beam larger logits, then lower tokens.  In a
// beam v follows x, so the order in it needs no sum: one pass over the logits
// finds each row's maximum, sum and `count` largest, and the group's are chosen
// among those.
//
// Bound by memory: every logit is read once.  A row is cut into `splits` CTAs
// where there are few rows.  A thread takes groups of 4 vectors of 16 bytes, the next
// group's loads in flight:
//   * it keeps a running maximum and the sum of exponentials below it (a group's
//     terms in fp32, their sums in fp64, so that beams' scores can be compared nearly to
//     the last bit of their rounding);
//   * logits above a threshold go to a list in shared memory, and `count` logits
//     are known to reach the threshold.  A CTA's first chunk (a group a thread) sets it from
//     the threads' own maxima, of which the warps' largest few are taken.  Then come stretches
//     without a barrier, each kGrow times as long as all before it: each puts in some kGrow x
//     `count` logits, and one comparison a group skips the others.  Vectors that have one are set
//     aside whole and looked at by all threads at the stretch's end, where the threshold rises.
//   * A stretch that puts in more than the list holds (rising logits) is looked at
//     again chunk by chunk, each with a threshold of its own, and a chunk that still has too
//     many (equal logits) is searched round by round.
// The last CTA of a group joins the lists of its rows.
// Measured in a graph: 32 groups of 8 rows of 131072 fp32, 16 of each 38.7 us (134 MB, 3.5 TB/s; 56 %
// of the issue slots, and the barriers at a stretch's end), 64 of each 51; 16 x 4 rows of 32000 fp16
// 13.8 us, 1 x 4 10.7, chains of latencies (first chunk, up to three stretches, the join's 4 us).
#include <algorithm>

#include "sample.cuh"

namespace moe {
namespace {

constexpr int kMostBeams = 64, kMostCount = 64;
constexpr int kBeamThreads = 256, kBeamWarps = kBeamThreads / 32;
constexpr int kVecs = 4;            // 16-byte vectors of a thread in a group
constexpr int kList = 1024;         // entries of the list
constexpr int kFound = 512;         // vectors that may have some for it
constexpr int kRank = 384;          // entries that are put in order by counting
constexpr int kCounted = 64;        // and those of which that is the quicker way to the largest
                                    // (16 x 4 rows of 32000, 8 of them 13.6 us, 15.7 with 32; 64 of
                                    // 32 x 8 rows of 131072 56.5, 62.8 with 128, 75.3 with 384)
// A stretch is so many times as long as all before it: it puts in kGrow x `count` logits.  32 x 8 rows
// of 131072 fp32, 16 and 64 of them: 40.6 and 56.5 us with 1, 38.3 and 52.0 with 3, 38.6 and 52.2 with 5.
constexpr int kGrow = 3;
constexpr int kGroups = 1000;       // counters of a launch (the workspace's first 4096 bytes)
constexpr float kLog2e = 1.4426950408889634f;

struct BeamArgs {
  const void* logits;
  int64_t stride;
  int vocab, beams, count, splits;
  const float* scores;              // [groups, beams]
  float* out_scores;                // [groups, count]
  int32_t* out_parents;
  int64_t* out_tokens;
  uint32_t* done;                   // [groups]: CTAs done, zero between calls
  double2* sums;                    // [rows, splits]: sum, maximum
  uint64_t* keys;                   // [rows, splits, count]: 0: none
};

template <typename T>
struct Vec {
  static constexpr int kN = 8;
  static constexpr uint32_t kNone = T::kBf16 ? 0xFF80u : 0xFC00u;  // -inf
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[kN]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = T::unpack(w[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // NaN: the other
    uint32_t d;
    if constexpr (T::kBf16) asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  static __device__ __forceinline__ float top(const uint4& r) {  // NaN where all are
    const float2 x = T::unpack(max2(max2(r.x, r.y), max2(r.z, r.w)));
    return fmaxf(x.x, x.y);
  }
  // Elements outside [lo, hi) become -inf.
  static __device__ __forceinline__ void cut(uint4& r, int64_t lo, int64_t hi) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < lo || i >= hi)
        w[i / 2] = i & 1 ? (w[i / 2] & 0xFFFFu) | kNone << 16 : (w[i / 2] & 0xFFFF0000u) | kNone;
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[kN]) {
    f[0] = __uint_as_float(r.x);
    f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z);
    f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ float top(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                 fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ void cut(uint4& r, int64_t lo, int64_t hi) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < lo || i >= hi) w[i] = 0xFF800000u;
    r = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A logit and its token as one key: larger logits are larger, of equal ones lower
// tokens.  0 stands for none; -inf and NaN never become keys.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return (uint64_t)Logit<float>::key(x) << 32 | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  return Logit<float>::value((uint32_t)(key >> 32));
}

struct Pick {  // a continuation's place in the group's order
  uint64_t hi, lo;  // score and beam; logit and token
  __device__ __forceinline__ bool above(const Pick& o) const {
    return hi != o.hi ? hi > o.hi : lo > o.lo;
  }
};
__device__ __forceinline__ Pick warp_best(Pick p) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Pick q{__shfl_xor_sync(kAll, p.hi, o), __shfl_xor_sync(kAll, p.lo, o)};
    if (q.above(p)) p = q;
  }
  return p;
}
// The block's largest, in every thread.
__device__ __forceinline__ Pick block_best(Pick p, Pick* s_warp) {
  p = warp_best(p);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x / 32] = p;
  __syncthreads();
  p = warp_best(s_warp[threadIdx.x % kBeamWarps]);
  __syncthreads();
  return p;
}
// out(i, number of j < n with above(j, i)) for each i < n, as many threads to an i as there are.
template <typename A, typename O>
__device__ __forceinline__ void rank_all(int n, A above, O out) {
  int per = 32;
  while (per > 1 && per * n > kBeamThreads) per >>= 1;
  const int tid = threadIdx.x, part = tid & (per - 1);
  for (int i0 = 0; i0 < n; i0 += kBeamThreads / per) {
    const int i = i0 + tid / per;
    int count = 0;
    if (i < n)
      for (int j = part; j < n; j += per) count += above(j, i);
    for (int o = per >> 1; o; o >>= 1) count += __shfl_xor_sync(kAll, count, o);
    if (i < n && part == 0) out(i, count);
  }
}
// A key that at least `count` of the threads' keys reach, or 0: the smallest of the warps'
// ceil(count / warps)-th largest, of those warps that have 16 keys.  Keys 0 do not count.
__device__ __forceinline__ uint32_t reached_by(uint32_t key, int count, uint32_t* s_warp) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (lane == 0) s_warp[warp] = 0;
  const bool full = __popc(__ballot_sync(kAll, key != 0)) >= 16;
  const int warps = __syncthreads_count(full) / 32;
  if (warps == 0) return 0;
  const int each = (count + warps - 1) / warps;
  if (full) {
    uint32_t top = 0;
    for (int i = 0; i < min(each, 16); ++i) {
      top = __reduce_max_sync(kAll, key);
      const uint32_t who = __ballot_sync(kAll, key == top);
      if (lane == __ffs(who) - 1) key = 0;
    }
    if (lane == 0) s_warp[warp] = top;
  }
  __syncthreads();
  uint32_t low = 0xFFFFFFFFu;  // warps that are not full have left 0
  for (int w = 0; w < kBeamWarps; ++w) low = min(low, s_warp[w] - 1u);
  __syncthreads();
  return each > 16 ? 0 : low + 1;
}

// The sum of exponentials of a vector below m: ordinary arithmetic where all goes well.
template <typename T>
__device__ __forceinline__ float exp_sum(const uint4& r, float m) {
  constexpr int kN = Vec<T>::kN;
  float f[kN];
  Vec<T>::unpack(r, f);
  uint64_t e[kN / 2];
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) {
    const uint64_t d = mul2(add2(pair(f[2 * i], f[2 * i + 1]), pair(-m, -m)), pair(kLog2e, kLog2e));
    e[i] = pair(exp2_approx(lo_of(d)), exp2_approx(hi_of(d)));
  }
#pragma unroll
  for (int w = kN / 4; w; w /= 2)
#pragma unroll
    for (int i = 0; i < w; ++i) e[i] = add2(e[i], e[i + w]);
  return lo_of(e[0]) + hi_of(e[0]);
}
// The same where a logit is NaN (counts as -inf) or m is +inf (its equals count 1).
template <typename T>
__device__ __noinline__ float exp_sum_odd(uint4 r, float m) {
  float f[Vec<T>::kN], sum = 0.f;
  Vec<T>::unpack(r, f);
  for (int i = 0; i < Vec<T>::kN; ++i)
    sum += f[i] == m ? 1.f : f[i] < m && m < INFINITY ? exp2_approx((f[i] - m) * kLog2e) : 0.f;
  return sum;
}

template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 4) k_beam_select(const BeamArgs a) {
  constexpr int kN = Vec<T>::kN;
  constexpr int kChunk = kBeamThreads * kVecs;  // vectors
  __shared__ __align__(16) uint64_t s_list[kList];
  __shared__ uint4 s_found[kFound];
  __shared__ int s_found_at[kFound];
  __shared__ Pick s_best[kBeamWarps];
  __shared__ uint64_t s_top[kMostCount];
  __shared__ uint32_t s_warp[kBeamWarps];
  __shared__ double s_sum[kBeamWarps];
  __shared__ float s_max[kBeamWarps], s_rowmax[kMostBeams], s_rowsum[kMostBeams], s_score[kMostBeams];
  __shared__ int s_count, s_founds, s_last;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, M = a.count;
  const int row = blockIdx.x / (uint32_t)a.splits, split = blockIdx.x - row * a.splits;
  using Raw = typename Logit<T>::Raw;
  const Raw* x0 = static_cast<const Raw*>(a.logits) + row * a.stride;
  // Vectors start at 16-byte boundaries: `skew` elements of the first are not the row's.
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(Raw));
  const uint4* vecs = reinterpret_cast<const uint4*>(x0 - skew);
  const int total = (skew + a.vocab + kN - 1) / kN, share = (total + a.splits - 1) / a.splits;
  const int lo = split * share, hi = min(total, lo + share);
  if (tid == 0) s_count = s_founds = 0;
  pdl_trigger();
  pdl_wait();

  uint4 r[kVecs], next[kVecs];
  int next_at = -1;  // the group that `next` holds
  auto fetch = [&](int c) {
    next_at = c;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int v = c + u * kBeamThreads + tid;
      next[u] = make_uint4(0, 0, 0, 0);
      if (v < hi) next[u] = __ldcs(vecs + v);
    }
  };
  float top[kVecs], gtop;
  // The group at c to r, the next one's loads on their way; its maxima.
  auto take = [&](int c) {
    if (next_at != c) fetch(c);
#pragma unroll
    for (int u = 0; u < kVecs; ++u) r[u] = next[u];
    if (c + kChunk < hi) fetch(c + kChunk);
    if (c + kChunk > hi || (c == 0 && skew) || c + kChunk >= total) {  // not all are the row's
#pragma unroll
      for (int u = 0; u < kVecs; ++u) {
        const int64_t v = c + u * kBeamThreads + tid, at = v * kN - skew;
        Vec<T>::cut(r[u], v < hi ? -at : kN, a.vocab - at);
      }
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) top[u] = Vec<T>::top(r[u]);
    gtop = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), -INFINITY);
  };
  float m = -INFINITY, thr = -INFINITY;
  double sum = 0;
  auto absorb = [&]() {
    if (gtop > m) {
      sum = m == -INFINITY ? 0 : sum * exp2_approx((m - gtop) * kLog2e);
      m = gtop;
    }
    if (gtop == -INFINITY) return;
    float e = 0.f;
#pragma unroll
    for (int u = 0; u < kVecs; ++u) e += exp_sum<T>(r[u], m);
    if (!(e < INFINITY)) {  // a NaN among them
      e = 0.f;
#pragma unroll
      for (int u = 0; u < kVecs; ++u) e += exp_sum_odd<T>(r[u], m);
    }
    sum += e;
  };
  // Vectors with a logit above thr (level: that reaches it) are set aside as they are: the loop
  // stays short, and the threads share their elements out at the stretch's end.
  bool some = false;  // this thread has, in this stretch
  auto find = [&](int c, bool level) {
    some = true;
#pragma unroll
    for (int u = 0; u < kVecs; ++u)
      if (level ? top[u] >= thr : top[u] > thr) {
        const int at = atomicAdd(&s_founds, 1);
        if (at < kFound) {
          s_found[at] = r[u];
          s_found_at[at] = c + u * kBeamThreads + tid;
        }
      }
  };
  int had = 0;  // entries of the list
  // A logit that exactly M of the list's n reach, by bisection, becomes the threshold and they the
  // list; false where equal logits leave none.
  auto narrow = [&](int n) {
    constexpr int kEach = kList / kBeamThreads;
    uint64_t k[kEach];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = tid + i * kBeamThreads;
      k[i] = at < n ? s_list[at] : 0;
      top = max(top, (uint32_t)(k[i] >> 32));
    }
    top = __reduce_max_sync(kAll, top);
    if (lane == 0) s_warp[warp] = top;
    if (tid == 0) s_count = 0;
    __syncthreads();
    for (int w = 0; w < kBeamWarps; ++w) top = max(top, s_warp[w]);
    uint32_t low = Logit<float>::key(thr), high = top;  // more than M reach low; fewer, high + 1
    bool exact = false;
    while (low < high && !exact) {
      const uint32_t mid = high - (high - low) / 2;  // above low
      int reach = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (i * kBeamThreads < n) reach += __syncthreads_count((uint32_t)(k[i] >> 32) >= mid);
      exact = reach == M;
      if (reach >= M) low = mid;
      else high = mid - 1;
    }
    if (exact) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if ((uint32_t)(k[i] >> 32) >= low) s_list[atomicAdd(&s_count, 1)] = k[i];
      thr = Logit<float>::value(low);
      had = M;
    } else if (tid == 0) {
      s_count = n;
    }
    __syncthreads();
    return exact;
  };
  // The list holds every logit so far that is above thr, and of those that reach it as
  // many as `count` needs.
  int summed = lo, one_by_one = lo + kChunk;
  for (int pos = lo; pos < hi;) {
    const bool chunk = pos < one_by_one;
    some = false;
    const int end = min(pos + (chunk ? kChunk : max(kChunk, kGrow * ((pos - lo) / kChunk * kChunk))), hi);
    for (int c = pos; c < end; c += kChunk) {
      take(c);
      if (c >= summed) absorb();
      if (!chunk && gtop > thr) find(c, false);
    }
    summed = max(summed, end);
    bool level = false;
    if (chunk) {
      const int busy = __syncthreads_count(gtop > thr);
      if (busy > 0 && (thr == -INFINITY || busy > 2 * M + 32)) {
        const uint32_t k = reached_by(gtop == -INFINITY ? 0 : Logit<float>::key(gtop), M, s_warp);
        const float t = k ? Logit<float>::value(k) : -INFINITY;
        if (t > thr) {
          thr = t;
          level = true;
        }
      }
      if (level ? gtop >= thr : gtop > thr) find(pos, level);
    }
    if (!__syncthreads_or(some)) {
      pos = end;
      continue;
    }
    const int found = s_founds;
    if (found <= kFound)
      for (int i = tid; i < found * kN; i += kBeamThreads) {
        const int e = i % kN;
        const float f = Logit<T>::of(reinterpret_cast<const Raw*>(s_found + i / kN)[e]);
        if (level ? f >= thr : f > thr) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kList) s_list[at] = key_of(f, (uint32_t)(s_found_at[i / kN] * kN - skew + e));
        }
      }
    __syncthreads();
    const int n = found <= kFound ? s_count : kList + 1, kept = found <= kFound ? min(n, kList) : had;
    if (tid == 0) s_founds = 0;
    __syncthreads();
    if (n > kList && !chunk) {  // once more, chunk by chunk
      if (tid == 0) s_count = had;
      one_by_one = end;
      continue;
    }
    pos = end;
    had = n;
    if (n <= M) continue;
    // The `count` best so far become the list, the last of them the threshold: by counting
    // what is above each, or round by round of a long list, and of the chunk where it overflowed.
    if (n > kCounted && n <= kList && narrow(n)) continue;
    if (n <= kRank) {
      rank_all(n, [&](int j, int i) { return s_list[j] > s_list[i]; },
               [&](int i, int above) {
                 if (above < M) s_top[above] = s_list[i];
               });
    } else {
      uint64_t last = ~0ull;
      for (int found = 0; found < M; ++found) {
        uint64_t best = 0;
        for (int i = tid; i < kept; i += kBeamThreads)
          if (s_list[i] < last && s_list[i] > best) best = s_list[i];
        if (n > kList && gtop >= thr) {  // the chunk's logits are read again
          const int c = end - 1 - (end - 1 - lo) % kChunk;
#pragma unroll 1
          for (int v = c + tid; v < end; v += kBeamThreads)
#pragma unroll 1
            for (int i = 0; i < kN; ++i) {
              const int token = v * kN - skew + i;
              if ((uint32_t)token >= (uint32_t)a.vocab) continue;
              const float f = Logit<T>::of(x0[token]);
              const uint64_t k = f >= thr && f > -INFINITY ? key_of(f, token) : 0;
              if (k < last && k > best) best = k;
            }
        }
        last = block_best(Pick{best, 0}, s_best).hi;
        if (tid == 0) s_top[found] = last;
      }
    }
    __syncthreads();
    if (tid < M) s_list[tid] = s_top[tid];
    if (tid == 0) s_count = M;
    had = M;
    thr = logit_of(s_top[M - 1]);
    __syncthreads();
  }

  // This part's maximum and sum, and its list.
  {
    float top = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
    top = s_max[lane % kBeamWarps];
#pragma unroll
    for (int o = 4; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    sum = m == -INFINITY || (m != top && top == INFINITY) ? 0 : m == top ? sum : sum * expf(m - top);
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    const int n = s_count, part = row * a.splits + split;
    uint64_t* keys = a.keys + (int64_t)part * M;
    for (int i = tid; i < n; i += kBeamThreads) keys[i] = s_list[i];  // at most M, in any order
    for (int i = n + tid; i < M; i += kBeamThreads) keys[i] = 0;
    __syncthreads();
    if (tid == 0) {
      double all = 0;
      for (int w = 0; w < kBeamWarps; ++w) all += s_sum[w];
      a.sums[part] = make_double2(all, top);
    }
  }
  // The last CTA of the group goes on.
  const int group = row / a.beams, parts = a.beams * a.splits;
  __threadfence();
  __syncthreads();
  if (tid == 0) s_last = atomicAdd(a.done + group, 1) == parts - 1;
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  if (tid == 0) a.done[group] = 0;
  const double2* sums = a.sums + (int64_t)group * parts;
  // A thread's first key is on its way while the sums are joined.  Each warp looks at one of
  // every 8, so that none has a poor row's alone, nor all parts' last (their keys may be in order).
  const uint64_t* keys = a.keys + (int64_t)group * parts * M;
  const int all = parts * M, per_beam = a.splits * M, at0 = lane * kBeamWarps + (warp + lane) % kBeamWarps;
  const uint64_t key0 = at0 < all ? __ldcg(keys + at0) : 0;
  const float* scores = a.scores + (int64_t)group * a.beams;
  for (int k = warp; k < a.beams; k += kBeamWarps) {  // a row's parts: at most 64
    const double2 none = make_double2(0, -INFINITY);
    const double2 p = lane < a.splits ? __ldcg(sums + k * a.splits + lane) : none;
    const double2 q = lane + 32 < a.splits ? __ldcg(sums + k * a.splits + lane + 32) : none;
    float top = fmaxf((float)p.y, (float)q.y);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    auto part = [&](const double2& x) {
      return (float)x.y == top ? x.x : x.x == 0 ? 0 : x.x * expf((float)x.y - top);
    };
    double all = part(p) + part(q);
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(kAll, all, o);
    if (lane == 0) {
      s_rowmax[k] = top;
      s_rowsum[k] = (float)log(all);
      s_score[k] = scores[k];
    }
  }
  if (tid == 0) s_count = 0;
  __syncthreads();
  auto score_of = [&](float x, int beam) {
    const float top = s_rowmax[beam], d = x == top ? 0.f : x - top;
    return __fadd_rn(s_score[beam], __fsub_rn(d, s_rowsum[beam]));
  };
  auto pick = [&](int i) {
    const uint64_t k = i == at0 ? key0 : __ldcg(keys + i);
    if (k == 0) return Pick{0, 0};
    const int beam = i / per_beam;
    const float v = score_of(logit_of(k), beam);
    if (!(v > -INFINITY)) return Pick{0, 0};
    return Pick{(uint64_t)Logit<float>::key(v) << 32 | (0xFFFFFFFFu - beam), k};
  };
  // Scores below `limit` are not among the best.
  const Pick mine = at0 < all ? pick(at0) : Pick{0, 0};
  uint32_t best = static_cast<uint32_t>(mine.hi >> 32);
  for (int i = at0 + kBeamThreads; i < all; i += kBeamThreads) best = max(best, (uint32_t)(pick(i).hi >> 32));
  const uint32_t limit = reached_by(best, M, s_warp);
  Pick* list = reinterpret_cast<Pick*>(s_list);
  for (int i = at0; i < all; i += kBeamThreads) {
    const Pick p = i == at0 ? mine : pick(i);
    if (p.hi == 0 || (uint32_t)(p.hi >> 32) < limit) continue;
    const int at = atomicAdd(&s_count, 1);
    if (at < kRank) list[at] = p;
  }
  __syncthreads();
  const int n = s_count;
  auto put_out = [&](int at, const Pick& p) {
    const int beam = static_cast<int>(0xFFFFFFFFu - (uint32_t)p.hi);
    const int64_t o = (int64_t)group * M + at;
    a.out_scores[o] = p.hi ? score_of(logit_of(p.lo), beam) : -INFINITY;
    a.out_parents[o] = p.hi ? beam : 0;
    a.out_tokens[o] = p.hi ? 0xFFFFFFFFu - (uint32_t)p.lo : 0;
  };
  if (n <= kRank) {
    rank_all(n, [&](int j, int i) { return list[j].above(list[i]); },
             [&](int i, int above) {
               if (above < M) put_out(above, list[i]);
             });
    for (int i = n + tid; i < M; i += kBeamThreads) put_out(i, Pick{0, 0});
    return;
  }
  Pick last{~0ull, ~0ull};
  for (int at = 0; at < M; ++at) {
    Pick best{0, 0};
    for (int i = tid; i < all && last.hi; i += kBeamThreads) {
      const Pick p = pick(i);
      if (last.above(p) && p.above(best)) best = p;
    }
    last = block_best(best, s_best);
    if (tid == 0) put_out(at, last);
  }
}

// CTAs of a row: as many as the GPU takes at once, four to an SM; where rows are fewer than the SMs
// one to an SM, each with a vector a thread at least, and more only if each still has four chunks
// (16 x 8 rows of 37025 fp32 19.9 us, 21.1 with one to an SM; 16 x 8 of 131072 fp16 23.2 / 26.7, 16 x 4
// of them 17.4 / 20.3; with one chunk each 16 x 4 of 32000 16.0 / 13.7).
int splits_of(int64_t rows, int64_t vocab, int64_t vec) {
  if (rows < 1) rows = 1;
  const int64_t sms = sm_count(), most = ceil_div(vocab, vec * kBeamThreads), full = 4 * sms / rows;
  const int64_t long_ones = std::min(full, vocab / (vec * kBeamThreads * kVecs * 4));
  const int64_t want = rows > sms ? full : std::max(sms / rows, long_ones), s = std::min(want, most);
  return static_cast<int>(s < 1 ? 1 : s > 64 ? 64 : s);
}

template <typename T>
int launch_beams(BeamArgs a, int64_t groups, cudaStream_t s) {
  using Raw = typename Logit<T>::Raw;
  for (int64_t g = 0; g < groups; g += kGroups) {
    const int64_t n = groups - g < kGroups ? groups - g : kGroups, parts = (int64_t)a.beams * a.splits;
    BeamArgs b = a;
    b.logits = static_cast<const Raw*>(a.logits) + g * a.beams * a.stride;
    b.scores += g * a.beams;
    b.out_scores += g * a.count;
    b.out_parents += g * a.count;
    b.out_tokens += g * a.count;
    b.sums += g * parts;
    b.keys += g * parts * a.count;
    if (launch_pdl(k_beam_select<T>, dim3(static_cast<unsigned>(n * parts)), dim3(kBeamThreads), 0, s,
                   b) != cudaSuccess)
      return MOE_ERR_CUDA;
    MOE_CHECK_LAUNCH();
  }
  return MOE_OK;
}

constexpr int64_t kSumsAt = 4096;  // behind the counters that every call leaves zero

}  // namespace
}  // namespace moe

extern "C" size_t moe_beam_select_workspace_size(int64_t groups, int64_t beams, int64_t vocab,
                                                 int64_t count, int64_t dtype) {
  using namespace moe;
  if (groups < 0 || beams < 1 || beams > kMostBeams || count < 1 || count > kMostCount || vocab < 1 ||
      groups > INT32_MAX / beams)
    return 0;
  // Rows times splits go up and down with the rows (148 rows of 131072 fp16 have 4 each, 149 have 3)
  // and never above 4 CTAs to an SM unless each row has one: a workspace made for the largest batch
  // has to serve the smaller ones.
  const int64_t most = std::max(groups * beams, (int64_t)4 * sm_count());
  return kSumsAt + most * (16 + 8 * count);
}

extern "C" int moe_beam_select(const moe_beam_select_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_beam_select_args_t& c = *args;
  if (c.groups < 0 || c.beams < 1 || c.vocab < 1 || c.count < 1 || c.stride < 0 ||
      (c.stride > 0 && c.stride < c.vocab && c.groups * c.beams > 1))
    return MOE_ERR_INVALID_ARG;
  if (c.beams > kMostBeams || c.count > kMostCount || c.vocab > (1 << 20) ||
      c.groups > INT32_MAX / (kMostBeams * 64) ||
      (c.dtype != MOE_DTYPE_F16 && c.dtype != MOE_DTYPE_BF16 && c.dtype != MOE_DTYPE_F32))
    return MOE_ERR_UNSUPPORTED;
  if (c.groups == 0) return MOE_OK;
  if (!c.logits || !c.scores || !c.out_scores || !c.out_parents || !c.out_tokens)
    return MOE_ERR_INVALID_ARG;
  const int64_t size = c.dtype == MOE_DTYPE_F32 ? 4 : 2, rows = c.groups * c.beams;
  // A group's scores are read by the CTA that writes its new ones, at the same place or none of theirs.
  if (overlap(c.scores, 4 * rows, c.out_scores, 4 * c.groups * c.count) &&
      (c.scores != c.out_scores || c.beams != c.count))
    return MOE_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(c.logits) % size) return MOE_ERR_ALIGNMENT;
  if (!c.workspace || c.workspace_bytes < (int64_t)moe_beam_select_workspace_size(
                                              c.groups, c.beams, c.vocab, c.count, c.dtype))
    return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  BeamArgs a{};
  a.logits = c.logits;
  a.stride = c.stride;
  a.vocab = static_cast<int>(c.vocab);
  a.beams = static_cast<int>(c.beams);
  a.count = static_cast<int>(c.count);
  a.splits = splits_of(rows, c.vocab, 16 / size);
  a.scores = c.scores;
  a.out_scores = c.out_scores;
  a.out_parents = c.out_parents;
  a.out_tokens = c.out_tokens;
  a.done = static_cast<uint32_t*>(c.workspace);
  char* ws = static_cast<char*>(c.workspace) + kSumsAt;
  a.sums = reinterpret_cast<double2*>(ws);
  a.keys = reinterpret_cast<uint64_t*>(ws + rows * a.splits * 16);
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (c.dtype == MOE_DTYPE_F32) return launch_beams<float>(a, c.groups, s);
  return c.dtype == MOE_DTYPE_BF16 ? launch_beams<BF16>(a, c.groups, s)
                                   : launch_beams<F16>(a, c.groups, s);
}
