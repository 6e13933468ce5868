// What the sampler's kernels share: the logits of each type, their weights, the
// filters' targets (formulas in sample_tokens.cu).
#pragma once

#include "paged.cuh"

namespace moe {
namespace {

constexpr uint32_t kAll = 0xffffffffu;

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int vocab, cluster;
  const float *uniforms, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int64_t* tokens;
  float* probs;
  uint64_t wait_ns;
};

// Logits as keys: unsigned integers of the same order, NaN as -inf, -0 as 0.
// Every key is above 0, which stands for "no logit".
template <typename T>
struct Logit;
struct Half16 {
  using Raw = uint16_t;
  static constexpr int kVec = 8;
  // `inf`: the format's infinity, above which are NaNs.
  static __device__ __forceinline__ uint32_t key(uint32_t b, uint32_t inf) {
    if ((b & 0x7FFFu) > inf) b = 0x8000u | inf;
    if (b == 0x8000u) b = 0;
    return b & 0x8000u ? (~b & 0xFFFFu) : (b | 0x8000u);
  }
  static __device__ __forceinline__ uint32_t raw(uint32_t k) {
    return k & 0x8000u ? (k & 0x7FFFu) : (~k & 0xFFFFu);
  }
};
template <>
struct Logit<F16> : Half16 {
  static __device__ __forceinline__ uint32_t key(uint16_t b) { return Half16::key(b, 0x7C00u); }
  static __device__ __forceinline__ float of(uint16_t b) { return h2f(b); }
  static __device__ __forceinline__ float value(uint32_t k) { return of((uint16_t)raw(k)); }
  static __device__ __forceinline__ uint32_t key_near(float x) { return key(f2h(x)); }
};
template <>
struct Logit<BF16> : Half16 {
  static __device__ __forceinline__ uint32_t key(uint16_t b) { return Half16::key(b, 0x7F80u); }
  static __device__ __forceinline__ float of(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
  static __device__ __forceinline__ float value(uint32_t k) { return of((uint16_t)raw(k)); }
  static __device__ __forceinline__ uint32_t key_near(float x) { return key(BF16::one(x)); }
};
template <>
struct Logit<float> {
  using Raw = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float of(float x) { return x; }
  static __device__ __forceinline__ uint32_t key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
  }
  static __device__ __forceinline__ uint32_t key_near(float x) { return key(x); }
};

__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) { return __shfl_sync(kAll, v, lane); }

// trunc(2^40 e) for e in [0, 1] as two limbs of 20 bits.  Added to 2^23 and
// rounded down, a number below 2^23 leaves its whole part in the low bits of the
// sum: every step is exact, and none is a conversion, whose pipe has an eighth of
// the rate.
struct Limbs {
  uint32_t hi, lo;
  __device__ __forceinline__ uint64_t value() const { return ((uint64_t)hi << 20) + lo; }
};
constexpr uint32_t kLimbBias = 0x4B000000u;  // the bits of 2^23
__device__ __forceinline__ Limbs limbs_biased(float e) {
  const float scale = 1048576.f, whole = 8388608.f;
  const float hi = __fmaf_rz(e, scale, whole);
  const float lo = __fmaf_rz(fmaf(e, scale, whole - hi), scale, whole);
  return Limbs{__float_as_uint(hi), __float_as_uint(lo)};
}
__device__ __forceinline__ Limbs limbs(float e) {
  const Limbs w = limbs_biased(e);
  return Limbs{w.hi - kLimbBias, w.lo - kLimbBias};
}
__device__ __forceinline__ uint64_t weight(float e) { return limbs(e).value(); }

// (x - m) / temperature, correctly rounded: the product with the reciprocal in two
// floats is off by less than a unit in the last place, and one correction by the
// remainder then rounds as the division does (Markstein 1990).
struct Softmax {
  float m, inverse, rest, divisor;
  __device__ __forceinline__ Softmax(float m, float temperature) : m(m) {
    inverse = __frcp_rn(temperature);
    divisor = inverse != 0.f ? temperature : 0.f;  // infinite: nothing to correct
    rest = inverse * fmaf(-inverse, divisor, 1.f);
  }
  // NaN where it, or a reciprocal, is out of range.
  __device__ __forceinline__ float quotient(float x) const {
    const float d = x - m, q = fmaf(d, inverse, d * rest);
    return fmaf(fmaf(-q, divisor, d), inverse, q);
  }
  // m finite.  Below -104 it is 0, and what is NaN there is too.
  __device__ __forceinline__ float exp(float x) const {
    const float q = quotient(x), e = expf(q);
    return q >= -104.f ? e : 0.f;
  }
};

// A warp's sum, in every lane: 27 bits at a time, of which 32 fit 32 bits.
__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
  const uint32_t lo = __reduce_add_sync(kAll, (uint32_t)v & 0x7FFFFFFu);
  const uint32_t mid = __reduce_add_sync(kAll, (uint32_t)(v >> 27) & 0x7FFFFFFu);
  const uint32_t hi = __reduce_add_sync(kAll, (uint32_t)(v >> 54));
  return ((uint64_t)hi << 54) + ((uint64_t)mid << 27) + lo;
}

// What top-p asks of a total weight, and the point of it that u stands for.
__device__ __forceinline__ uint64_t need_of(float p, uint64_t total) {
  const double want = ceil(__dmul_rn((double)p, __ull2double_rn(total)));
  const uint64_t n = want >= 1.0 ? __double2ull_rz(want) : 1ull;
  return n < total ? n : total;
}
__device__ __forceinline__ uint64_t draw_of(float u, uint64_t total) {
  const double at = floor(__dmul_rn((double)u, __ull2double_rn(total)));
  const uint64_t r = at >= 1.0 ? __double2ull_rz(at) : 0ull;
  return r < total ? r : total - 1;
}

// Sums of 32 pieces of a row in order (lane i: the weight above the cut in piece
// i, and how many there equal the cut), of whose ties with the cut the first
// `ties` are kept, `ahead` lying before all pieces -> the kept weight and the ties
// before the piece, its kept weight, that of all.
struct Piece {
  uint64_t before, ties_before, own, all;
};
__device__ __forceinline__ Piece place_pieces(uint64_t w, uint64_t equal, uint64_t ahead,
                                              uint64_t ties, uint64_t w_cut) {
  const int lane = threadIdx.x & 31;
  uint64_t seen = equal;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(kAll, seen, o);
    if (lane >= o) seen += v;
  }
  seen += ahead - equal;
  const uint64_t own =
      w + (seen >= ties ? 0ull : (ties - seen < equal ? ties - seen : equal)) * w_cut;
  uint64_t run = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t v = __shfl_up_sync(kAll, run, o);
    if (lane >= o) run += v;
  }
  return Piece{run - own, seen, own, shfl64(run, 31)};
}

// n <= FEW candidates of a row (values of the logits' order and indices, which hold
// every logit that the filters may keep): applies the filters and draws.  THREADS /
// FEW threads per candidate compare it with an equal share of the others.  k = 0:
// no top-k; need: what top-p asks for, 0: of the sum of these.  weights: FEW values
// of shared memory, parts: one for each warp.
template <int THREADS, int FEW, class V, class I, class Exp>
__device__ __forceinline__ void finish_few(const SampleArgs& a, int64_t row, int n, const V* values,
                                           const I* indices, uint64_t* weights, int k, float p,
                                           float min_p, uint64_t need, float u, Exp exp_of,
                                           uint64_t* parts) {
  constexpr int kTeam = THREADS / FEW, kWarpsOf = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto block_sum = [&](uint64_t v) {  // in every thread
    v = warp_sum64(v);
    __syncthreads();
    if (lane == 0) parts[warp] = v;
    __syncthreads();
    return warp_sum64(lane < kWarpsOf ? parts[lane & (kWarpsOf - 1)] : 0ull);
  };
  auto team_sum = [&](auto v) {
#pragma unroll
    for (int o = 1; o < kTeam; o <<= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
  };
  const int i = threadIdx.x / kTeam, share = threadIdx.x % kTeam;
  const bool real = i < n, first = share == 0;
  const V own = real ? values[i] : V(0);
  const uint32_t index = real ? (uint32_t)indices[i] : 0u;
  const float e = real ? exp_of(own) : 0.f;
  uint64_t w = weight(e);
  if (real && first) weights[i] = w;
  __syncthreads();
  uint32_t place = 0;   // in the order by falling logit and rising index
  uint64_t before = 0;  // weights ahead of it
  if (real)
    for (int j = share; j < n; j += kTeam) {
      const V v = values[j];
      const bool ahead = v > own || (v == own && (uint32_t)indices[j] < index);
      place += ahead;
      before += ahead ? weights[j] : 0ull;
    }
  place = team_sum(place);
  before = team_sum(before);
  bool keep = real && (k == 0 || place < (uint32_t)k);
  if (p < 1.f && need == 0) need = need_of(p, block_sum(keep && first ? w : 0ull));
  keep = keep && (!(p < 1.f) || before < need) && e >= min_p;
  if (!keep) w = 0;
  const uint64_t total = block_sum(first ? w : 0ull);  // its barriers order the weights too
  if (real && first) weights[i] = w;
  __syncthreads();
  uint64_t run = 0;  // kept weights of lower indices
  if (keep)
    for (int j = share; j < n; j += kTeam) run += (uint32_t)indices[j] < index ? weights[j] : 0ull;
  run = team_sum(run);
  const uint64_t r = draw_of(u, total);
  if (keep && first && r >= run && r < run + w) {
    a.tokens[row] = index;
    a.probs[row] = (float)(__ull2double_rn(w) / __ull2double_rn(total));
  }
}

}  // namespace
}  // namespace moe
