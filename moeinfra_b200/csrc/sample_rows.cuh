// The sampler for many rows, or short ones: one CTA a row (formulas in
// sample_tokens.cu).
//
// The row is read from memory once, for its maximum, and then from the caches:
//   * Weights (or counts, for top-k) are added up in 1024 bins of 1/32 in units of
//     the temperature, which hold every weight above 0.  A scan of the bins finds
//     the one with the boundary.
//   * The logits above that bin and those in it are gathered, at most 2048 of
//     each, and the weights of those above that found no place added up instead (of
//     all of them at once where the bins' sums tell that there are too many).
//     Up to 256 are compared with each other and drawn from at once.  Of more, the
//     bin's are cut to one value by histograms over their bits, 10 bits a round.
//   * The draw is one more histogram, over the indices of the logits kept; or, if
//     they do not fit, sums of contiguous parts of the row, and of parts of the part.
// Sums are exact integers: the order in which atomics add them does not matter.
//
// Bound by instruction issue.  256 x 131072 fp32 of mixed parameters: 127 us, 134
// MB, which a plain copy's rate would read in 21 (greedy rows alone: 35); 256 CTAs are
// 1.73 waves, so 40 SMs have nothing to do in the second.  What
// costs: the exponential of a correctly rounded quotient and its 40 bits, in each
// of two passes (13 and 15 cycles an SM for 32 logits, at two thirds of the issue
// slots).  64 x 32000 fp16: 30 us, as long as the slowest row's CTA, 8 of them its
// histogram, 8 the second pass.  1024 threads and one CTA to an SM; with 512 and two, 64 x 32000
// took 4 us longer and 256 x 131072 32.  Bins in two copies, for fewer conflicts:
// no faster.  Four pieces on their way in the first pass, not one: 26 us less.
#pragma once

#include "sample.cuh"

namespace moe {
namespace {

constexpr int kRowThreads = 1024, kRowWarps = kRowThreads / 32;
constexpr int kBinBits = 10, kBins = 1 << kBinBits;
static_assert(kBins == kRowThreads && kRowWarps == 32);
constexpr float kBinsPerUnit = 32.f;  // 1024 bins reach 32 units down, weights above 0 27.8
constexpr float kLeast = 1.f / (1ull << 40);  // of weight 1; its bin is below 890
constexpr int kFew = 256;             // candidates that are compared with each other directly
constexpr int kHeld = 2048;           // logits of a list

// Everything at or below `cut` but the first `ties` logits equal to it is left out.
struct Cut {
  float x = NAN;  // NaN: nothing is
  uint64_t ties = 0, equal = 0;
};

template <typename T>
__global__ void __launch_bounds__(kRowThreads, 1) k_sample_rows(const SampleArgs a) {
  using L = Logit<T>;
  constexpr int kVec = L::kVec, kStep = 32 * kVec;
  __shared__ uint32_t s_lo[kBins], s_hi[kBins];  // the bins' 64-bit sums
  __shared__ float s_x[2][kHeld];                // logits above the boundary's bin, in it
  __shared__ int s_at[2][kHeld];
  __shared__ uint64_t s_part[2][kRowWarps];
  struct Pick {
    uint64_t before, own, total;
    int bin, about;
  };
  __shared__ Pick s_pick;
  __shared__ uint64_t s_sum[kRowWarps];  // what the warps' parts of the row keep for sure
  __shared__ uint64_t s_few[kFew];
  __shared__ uint32_t s_key[2];
  __shared__ int s_n[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  pdl_trigger();
  pdl_wait();
  const typename L::Raw* x = static_cast<const typename L::Raw*>(a.logits) + row * a.stride;
  const bool wide = (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
  const float temperature = a.temperature[row], u = a.uniforms[row], p = a.top_p[row];
  const float min_p = fminf(a.min_p[row], 1.f);  // above 1 the maxima stay
  const int k = a.top_k[row];

  // f(logits, index of the first) for every lane's piece of [from, to), from a
  // multiple of kVec; past `to` the logits are NaN, and where the row has a NaN,
  // -inf.  One piece is on its way while the last is worked on.
  auto load = [&](int at, int to) {
    uint4 v = {};
    if (wide && at + kVec <= to) v = *reinterpret_cast<const uint4*>(x + at);
    return v;
  };
  float only = NAN;  // the maximum, if it or the temperature leave others no weight
  auto unpack = [&](const uint4& v, int at, int to, float (&out)[kVec]) {
    if (wide && at + kVec <= to) {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (kVec == 8) out[j] = L::of((uint16_t)(w[j / 2] >> (16 * (j & 1))));
        else out[j] = __uint_as_float(w[j]);
        out[j] = fmaxf(out[j], -INFINITY);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) out[j] = at + j < to ? fmaxf(L::of(x[at + j]), -INFINITY) : NAN;
    }
    if (only == only) {  // as if it were 0 and all others -inf: the same weights
#pragma unroll
      for (int j = 0; j < kVec; ++j) out[j] = out[j] == only ? 0.f : out[j] - INFINITY;
    }
  };
  auto each = [&](int from, int to, auto f) {
    int at = from + lane * kVec;
    uint4 now = load(at, to);
#pragma unroll 1
    for (int step = from; step < to; step += kStep, at += kStep) {
      const uint4 next = load(at + kStep, to);
      float v[kVec];
      unpack(now, at, to, v);
      f(v, at);
      now = next;
    }
  };
  const int part = (a.vocab + kRowWarps * kStep - 1) / (kRowWarps * kStep) * kStep;  // a warp's
  const int from = min(warp * part, a.vocab), to = min(from + part, a.vocab);

  // ---- the maximum and its lowest index ----
  s_lo[threadIdx.x] = s_hi[threadIdx.x] = 0;
  if (threadIdx.x < 2) s_n[threadIdx.x] = 0;
  float m = -INFINITY;
  int where = INT_MAX;
  auto see = [&](const float (&v)[kVec], int at) {
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kVec; ++j) most = fmaxf(most, v[j]);
    if (most > m || where == INT_MAX) {
      m = fmaxf(most, -INFINITY);
      where = at;
    }
  };
#pragma unroll 1
  for (int at = from + lane * kVec; at - lane * kVec < to; at += 4 * kStep) {
    uint4 raw[4];  // four pieces on their way: memory's latency
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = load(at + i * kStep, to);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[kVec];
      unpack(raw[i], at + i * kStep, to, v);
      see(v, at + i * kStep);
    }
  }
  {
    const uint32_t own = Logit<float>::key(m);
    const uint32_t top = __reduce_max_sync(kAll, own);
    const uint32_t first = __reduce_min_sync(kAll, own == top ? (uint32_t)where : 0xFFFFFFFFu);
    if (lane == 0) {
      s_part[0][warp] = top;
      s_part[1][warp] = first;
    }
    __syncthreads();
    const uint32_t wtop = (uint32_t)s_part[0][lane];
    const uint32_t all = __reduce_max_sync(kAll, wtop);
    where = (int)__reduce_min_sync(
        kAll, wtop == all ? (uint32_t)s_part[1][lane] : 0xFFFFFFFFu);
    m = Logit<float>::value(all);
  }
  if (!(temperature > 0.f) || k == 1) {
    if (threadIdx.x == 0) {
      while (where + 1 < a.vocab && !(fmaxf(L::of(x[where]), -INFINITY) == m)) ++where;  // in the piece
      a.tokens[row] = where;
      a.probs[row] = 1.f;
    }
    return;
  }
  const bool alone = fabsf(m) == INFINITY || __frcp_rn(temperature) == INFINITY;
  if (alone) {
    only = m;
    m = 0.f;
  }
  const Softmax soft(m, alone ? 1.f : temperature);
  // Bin 0 is the maximum's; the quotient falls with the logit, so bins do not
  // overlap.  Added to 2^23, a number leaves its whole part in the sum's low bits.
  auto bin_at = [&](float q) { return __float_as_uint(fmaf(-q, kBinsPerUnit, 8388608.f)) - 0x4B000000u; };
  auto bin_of = [&](float v) {
    const float q = soft.quotient(v);
    return q >= -32.f ? (int)min(bin_at(q), kBins - 1u) : kBins - 1;
  };
  // The lowest key whose bin is at most `bin`, by one warp, 5 bits at a time from
  // what the division undone gives, a bin's width and two keys to either side.
  auto key_from = [&](int bin) {
    const uint32_t least = L::key_near(-INFINITY), most = L::key_near(m);
    if (bin < 0) return most + 1;
    auto near = [&](int b) {
      return L::key_near(fmaf(-soft.divisor, b * (1.f / kBinsPerUnit), m));
    };
    uint32_t lo = least, hi = most;  // hi's bin is low enough
    if (bin < kBins - 1 && soft.inverse != 0.f) {
      lo = max(near(bin + 2), least + 2) - 2;
      hi = min(near(bin - 1) + 2, most);
    }
    while (lo < hi) {
      const uint32_t step = (hi - lo) / 32 + 1, key = min(lo + step * (uint32_t)lane, hi);
      const uint32_t in = __ballot_sync(kAll, bin_of(L::value(key)) <= bin);
      const int j = in ? __ffs(in) - 1 : 32;  // the first that is
      const uint32_t next = j < 32 ? min(lo + step * (uint32_t)j, hi) : hi;
      lo = j == 0 ? next : min(lo + step * (uint32_t)(j - 1), hi - 1) + 1;
      hi = next;
    }
    return hi;
  };
  auto add = [&](int bin, uint64_t w) {
    const uint32_t low = (uint32_t)w, carry = atomicAdd(&s_lo[bin], low) + low < low;
    const uint32_t high = (uint32_t)(w >> 32) + carry;
    if (high) atomicAdd(&s_hi[bin], high);
  };
  // The weights of a piece's logits above `cut` (NaN: of all) that min-p keeps.  An
  // overflowed quotient has the exponential NaN, which nothing keeps.
  auto add_up = [&](Limbs& sum, const float (&v)[kVec], float cut) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const float e = expf(soft.quotient(v[j]));
      const Limbs w = limbs_biased(e >= min_p && !(v[j] <= cut) ? e : 0.f);
      sum.hi += w.hi;
      sum.lo += w.lo;
    }
    sum.hi -= kVec * kLimbBias;
    sum.lo -= kVec * kLimbBias;
  };
  // The first bin with which the sum reaches `need` (0: what top-p asks of the
  // total), then known to every thread; leaves the bins empty.
  // `weights`: the bins hold weights of the first kind, and about counts the logits
  // before the bin, to a few percent: each weighs what its bin's middle does.
  auto pick = [&](uint64_t& need, bool weights) {
    __syncthreads();
    const uint64_t own = (uint64_t)s_hi[threadIdx.x] << 32 | s_lo[threadIdx.x];
    s_lo[threadIdx.x] = s_hi[threadIdx.x] = 0;
    const uint64_t of_warp = warp_sum64(own);
    uint32_t count = 0;
    if (weights) {
      count = __float2uint_rn(__ull2float_rn(own) * kLeast *
                              __expf((int)threadIdx.x * (1.f / kBinsPerUnit)));
      const uint32_t all = __reduce_add_sync(kAll, min(count, 1u << 20));
      if (lane == 0) s_part[1][warp] = all;
    }
    if (lane == 0) s_part[0][warp] = of_warp;
    __syncthreads();
    const uint64_t of_lane = s_part[0][lane];
    const uint64_t total = warp_sum64(of_lane), ahead = warp_sum64(lane < warp ? of_lane : 0ull);
    if (need == 0) need = need_of(p, total);
    if (ahead < need && need <= ahead + of_warp) {  // the bin is this warp's
      uint64_t run = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(kAll, run, o);
        if (lane >= o) run += v;
      }
      const uint64_t before = ahead + run - own;
      const bool here = before < need && need <= before + own;
      int about = 0;
      if (weights) {
        const int at = __ffs(__ballot_sync(kAll, here)) - 1;
        about = (int)__reduce_add_sync(kAll, (lane < at ? min(count, 1u << 20) : 0u) +
                                                 (lane < warp ? (uint32_t)s_part[1][lane] : 0u));
      }
      if (here) s_pick = Pick{before, own, total, (int)threadIdx.x, about};
    }
    __syncthreads();
    return s_pick;
  };

  Cut cut;
  bool summed = false;  // s_sum and the lists have what may be kept
  bool skip = false;    // the first list is not used
  bool held = false;    // all that may be kept is in the two lists
  auto held_each = [&](int list, auto f) {
    const int n = list == 0 && skip ? 0 : min(s_n[list], kHeld);
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += kRowThreads) f(s_x[list][i], s_at[list][i]);
  };
#pragma unroll 1
  for (int step = 0; step < 2; ++step) {  // top-k, then top-p
    const bool count = step == 0;
    if (count ? !(k > 0 && k < a.vocab) : !(p < 1.f)) continue;
    // The tokens that are still in at the last cut are added as one.
    auto share = [&](float v) {
      return count ? (uint64_t)1 : v <= cut.x ? (uint64_t)0 : weight(soft.exp(v));
    };
    const uint64_t at_cut = cut.ties ? cut.ties * weight(soft.exp(cut.x)) : 0ull;
    uint64_t need = count ? (uint64_t)k : 0ull, above = 0, own = 0;
    uint32_t lo, hi;  // keys between which the boundary is
    bool row_left = false;
    if (held) {
      lo = L::key_near(cut.x);
      hi = L::key_near(m);
    } else {
      if (count) {
        each(from, to, [&](const float (&v)[kVec], int) {
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (v[j] == v[j]) atomicAdd(&s_lo[bin_of(v[j])], 1u);
        });
      } else {
        each(from, to, [&](const float (&v)[kVec], int) {
#pragma unroll
          for (int j0 = 0; j0 < kVec; j0 += 4) {
            // Four at a time: an atomic's result (for the carry) takes a while.
            uint32_t low[4], old[4] = {}, bin[4];
            float e[4], most = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float x = v[j0 + j], q = soft.quotient(x);
              e[j] = expf(q);  // NaN where the quotient overflowed
              const Limbs w = limbs(e[j]);
              low[j] = (w.hi << 20) + w.lo;
              bin[j] = bin_at(q);
              if (e[j] >= kLeast && !(x <= cut.x)) {
                old[j] = atomicAdd(&s_lo[bin[j]], low[j]);
                most = fmaxf(most, e[j]);
              } else {
                low[j] = 0;
                e[j] = 0.f;
              }
            }
            bool carry = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) carry |= old[j] + low[j] < low[j];
            if (carry || most >= 1.f / 256) {  // else the weights are below 2^32
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const uint32_t high = (limbs(e[j]).hi >> 12) + (old[j] + low[j] < low[j]);
                if (high) atomicAdd(&s_hi[bin[j]], high);
              }
            }
          }
        });
        if (threadIdx.x == 0 && at_cut) add(bin_of(cut.x), at_cut);
      }
      if (threadIdx.x == 0) s_n[0] = s_n[1] = 0;
      const Pick found = pick(need, !count);
      above = found.before;
      own = found.own;
      // Too many above the bin for the first list: it stays empty.
      skip = (count ? (int)above : found.about) > kHeld + kHeld / 4;
      if (skip && threadIdx.x == 0) s_n[0] = kHeld + 1;
      if (warp < 2) s_key[warp] = key_from(found.bin - warp);
      __syncthreads();
      lo = s_key[0];
      hi = s_key[1];
      // ---- gather; and if no other filter follows, add up what is above the bin and
      // has no place ----
      const bool last = !count || !(p < 1.f);
      const float x_lo = fmaxf(L::value(lo), count ? -INFINITY : cut.x);
      const float x_hi = L::value(hi - 1);
      Limbs sum{0, 0};
      each(from, to, [&](const float (&v)[kVec], int at) {
        float most = v[0];
#pragma unroll
        for (int j = 1; j < kVec; ++j) most = fmaxf(most, v[j]);
        if (!__any_sync(kAll, most >= x_lo)) return;
        uint32_t in[2] = {0, 0};
        // The other warps add to the count, so lanes may read it differently: a lane
        // goes by its own reading, and no vote depends on it.
        const bool full = *(volatile int*)&s_n[0] > kHeld;
        if (full && last) {
          add_up(sum, v, x_hi);
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) in[0] |= (v[j] > x_hi ? 1u : 0u) << j;
        }
#pragma unroll
        for (int j = 0; j < kVec; ++j) in[1] |= (v[j] >= x_lo && v[j] <= x_hi ? 1u : 0u) << j;
        uint32_t out = in[0];  // above the bin, but without a place
#pragma unroll
        for (int l = 0; l < 2; ++l) {
          if (!in[l] || *(volatile int*)&s_n[l] > kHeld) continue;
          int slot = atomicAdd(&s_n[l], __popc(in[l]));
#pragma unroll
          for (int j = 0; j < kVec; ++j)
            if (in[l] >> j & 1) {
              if (slot < kHeld) {
                s_x[l][slot] = v[j];
                s_at[l][slot] = at + j;
                if (l == 0) out &= ~(1u << j);
              }
              ++slot;
            }
        }
        if (last && __any_sync(kAll, out)) {  // the list has just become full
#pragma unroll
          for (int j = 0; j < kVec; ++j) {
            const float e = soft.exp(v[j]);
            const Limbs w = limbs((out >> j & 1) && e >= min_p ? e : 0.f);
            sum.hi += w.hi;
            sum.lo += w.lo;
          }
        }
      });
      const uint64_t all = warp_sum64(sum.value());
      if (lane == 0) s_sum[warp] = all;
      hi -= 1;
      __syncthreads();
      held = s_n[0] <= kHeld && s_n[1] <= kHeld;
      row_left = s_n[1] > kHeld;
      summed = !row_left;
      const int n0 = s_n[0], n1 = s_n[1];
      __syncthreads();  // the counts begin anew in a second search
      if (n0 + n1 <= kFew) {
        if ((int)threadIdx.x < n1) {
          s_x[0][n0 + threadIdx.x] = s_x[1][threadIdx.x];
          s_at[0][n0 + threadIdx.x] = s_at[1][threadIdx.x];
        }
        __syncthreads();
        finish_few<kRowThreads, kFew>(
            a, row, n0 + n1, s_x[0], s_at[0], s_few, k > 0 && k < a.vocab ? k : 0, p, min_p,
            count ? 0ull : need, u,
            [&](float v) { return soft.exp(v); }, &s_part[0][0]);
        return;
      }
    }
    // ---- to one key ----
#pragma unroll 1
    while (lo < hi) {
      const int bits = 32 - __clz(hi - lo), shift = bits > kBinBits ? bits - kBinBits : 0;
      auto put = [&](float v) {
        const uint32_t key = L::key_near(v);
        if (v == v && key - lo <= hi - lo) {
          const uint64_t w = share(v);
          if (w) add((int)((hi - key) >> shift), w);
        }
      };
      if (row_left) {
        each(from, to, [&](const float (&v)[kVec], int) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) put(v[j]);
        });
      } else {
        // A first search's boundary lies in the second list, a second's in either.
        if (held) held_each(0, [&](float v, int) { put(v); });
        held_each(1, [&](float v, int) { put(v); });
      }
      if (threadIdx.x == 0 && at_cut) {
        const uint32_t key = L::key_near(cut.x);
        if (key - lo <= hi - lo) add((int)((hi - key) >> shift), at_cut);
      }
      uint64_t rest = need ? need - above : 0ull;
      const Pick found = pick(rest, false);
      if (!need) need = rest;
      above += found.before;
      own = found.own;
      hi -= (uint32_t)found.bin << shift;
      lo = max(lo, hi - min(hi, (1u << shift) - 1));
    }
    if (!need) need = need_of(p, at_cut);  // the cut is at the maximum
    const float v = L::value(lo);
    if (count) {
      cut = Cut{v, k - above, own};
    } else {
      const uint64_t w = weight(soft.exp(v)), n = (need - above + w - 1) / w;
      cut = v == cut.x ? Cut{v, min(n, cut.ties), cut.equal} : Cut{v, n, own / w};
    }
  }

  // ---- the draw ----
  auto keeps = [&](float v) {  // the weight of a logit at or above the cut
    const float e = soft.exp(v);
    return e >= min_p ? weight(e) : 0ull;
  };
  if (held) {
    const int bits = 32 - __clz(a.vocab - 1), shift = bits > kBinBits ? bits - kBinBits : 0;
    const int mask = (1 << shift) - 1;
    // Of the logits equal to the cut the first by index: up to `last`.
    int last = INT_MAX;
    if (cut.ties < cut.equal) {
      auto equal = [&](auto f) {
        for (int l = 0; l < 2; ++l)
          held_each(l, [&](float v, int at) {
            if (v == cut.x) f(at);
          });
      };
      equal([&](int at) { atomicAdd(&s_lo[at >> shift], 1u); });
      uint64_t need = cut.ties;
      const Pick found = pick(need, false);
      equal([&](int at) {
        if (at >> shift == found.bin) s_lo[at & mask] = 1;
      });
      __syncthreads();
      int rest = (int)(cut.ties - found.before);
      for (last = found.bin << shift; (rest -= s_lo[last & mask]) > 0 && (last & mask) < mask; ++last) {}
      __syncthreads();
      if ((int)threadIdx.x <= mask) s_lo[threadIdx.x] = 0;
      __syncthreads();
    }
    auto kept = [&](auto f) {
#pragma unroll 1
      for (int l = 0; l < 2; ++l)
        held_each(l, [&](float v, int at) {
          if (v < cut.x || (v == cut.x && at > last)) return;
          const uint64_t w = keeps(v);
          if (w) f(w, at);
        });
    };
    kept([&](uint64_t w, int at) { add(at >> shift, w); });
    __syncthreads();
    uint64_t total = 0;
    {
      const uint64_t sum = warp_sum64((uint64_t)s_hi[threadIdx.x] << 32 | s_lo[threadIdx.x]);
      if (lane == 0) s_part[1][warp] = sum;
      __syncthreads();
      total = warp_sum64(s_part[1][lane]);
    }
    const uint64_t r = draw_of(u, total);
    uint64_t need = r + 1;
    const Pick found = pick(need, false);
    kept([&](uint64_t w, int at) {
      if (at >> shift == found.bin) {
        s_lo[at & mask] = (uint32_t)w;
        s_hi[at & mask] = (uint32_t)(w >> 32);
      }
    });
    __syncthreads();
    if (warp) return;
    uint64_t run = found.before;
#pragma unroll 1
    for (int i = 0; i <= mask; i += 32) {
      const uint64_t w = i + lane <= mask ? (uint64_t)s_hi[i + lane] << 32 | s_lo[i + lane] : 0ull;
      uint64_t sum = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(kAll, sum, o);
        if (lane >= o) sum += v;
      }
      if (r >= run + sum - w && r < run + sum) {
        a.tokens[row] = (found.bin << shift) + i + lane;
        a.probs[row] = (float)(__ull2double_rn(w) / __ull2double_rn(total));
      }
      run += shfl64(sum, 31);
    }
    return;
  }
  const uint64_t w_cut = cut.ties ? keeps(cut.x) : 0ull;
  uint64_t run = 0, ahead = 0, total = 0, r = 0;
  int begin = 0, end = a.vocab;
#pragma unroll 1
  do {  // the part, of one for each warp, that holds the token
    const int size = (end - begin + kRowWarps * kStep - 1) / (kRowWarps * kStep) * kStep;
    const int lo = min(begin + warp * size, end), hi = min(lo + size, end);
    uint64_t sum = 0;
    uint32_t equal = 0;
    __syncthreads();
    if (summed) {  // then just the lists' are missing
      for (int l = 0; l < 2; ++l)
        held_each(l, [&](float v, int at) {
          if (v > cut.x) {
            const uint64_t w = keeps(v);
            if (w) add(at / size, w);
          }
          if (v == cut.x) atomicAdd(&s_lo[kRowWarps + at / size], 1u);
        });
      __syncthreads();
      sum = s_sum[warp] + ((uint64_t)s_hi[warp] << 32) + s_lo[warp];
      equal = s_lo[kRowWarps + warp];
      summed = false;
    } else {
      Limbs own{0, 0};  // of at most 2^9 logits
      each(lo, hi, [&](const float (&v)[kVec], int) {
        add_up(own, v, cut.x);
        if (cut.ties) {
#pragma unroll
          for (int j = 0; j < kVec; ++j) equal += v[j] == cut.x;
        }
      });
      sum = warp_sum64(own.value());
      equal = __reduce_add_sync(kAll, equal);
    }
    if (lane == 0) {
      s_part[0][warp] = sum;
      s_part[1][warp] = equal;
    }
    __syncthreads();
    const Piece parts =
        place_pieces(s_part[0][lane],
                     s_part[1][lane], ahead, cut.ties, w_cut);
    if (begin == 0 && end == a.vocab) {
      total = parts.all;
      r = draw_of(u, total);
    }
    const uint64_t at = run + parts.before;
    const int j = __ffs(__ballot_sync(kAll, r >= at && r < at + parts.own)) - 1;
    if (j < 0) return;
    run = shfl64(at, j);
    ahead = shfl64(parts.ties_before, j);
    begin += j * size;
    end = min(begin + size, end);
  } while (end - begin > 4 * kStep);
  if (warp) return;
#pragma unroll 1
  for (int at = begin; at < end; at += kStep) {
    const int first = at + lane * kVec;
    float v[kVec];
    unpack(load(first, end), first, end, v);
    uint64_t w[kVec], own = 0, equal = 0;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      w[j] = !(v[j] <= cut.x) ? keeps(v[j]) : 0ull;
      own += w[j];
      equal += v[j] == cut.x;
    }
    const Piece lanes = place_pieces(own, equal, ahead, cut.ties, w_cut);
    uint64_t before = run + lanes.before, seen = lanes.ties_before;
    if (r >= before && r < before + lanes.own) {
      bool found = false;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if (v[j] == cut.x) {
          w[j] = seen < cut.ties ? w_cut : 0ull;
          ++seen;
        }
        if (!found && r < before + w[j]) {
          found = true;
          a.tokens[row] = first + j;
          a.probs[row] = (float)(__ull2double_rn(w[j]) / __ull2double_rn(total));
        }
        before += w[j];
      }
    }
    run += lanes.all;
    if (r < run) return;
    ahead = shfl64(lanes.ties_before + equal, 31);
  }
}

template <typename T>
int launch_sample_rows(const SampleArgs& a, int64_t rows, cudaStream_t s) {
  if (rows > INT32_MAX) return MOE_ERR_UNSUPPORTED;
  if (launch_pdl(k_sample_rows<T>, dim3(static_cast<unsigned>(rows)), dim3(kRowThreads), 0, s, a) !=
      cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

}  // namespace
}  // namespace moe
