// Trees of drafted tokens over a paged cache: what a node sees, and the rows that have
// met an infinity or NaN they do not see.  Shared by the attention kernels for trees.
#pragma once

#include "paged.cuh"

namespace moe {

struct TreeRows {
  KvPages kv;
  const uint16_t* q;
  int64_t q_seq, q_node;        // elements from one sequence's (node's) queries to the next
  uint16_t* out;                // [seqs, nodes, heads, HD]
  const int32_t *lengths, *counts;
  const uint64_t* visible;      // [seqs, nodes, words]
  int64_t vis_seq, vis_node;
  int nodes, words, heads, group;
  float scale_log2;
};

// The kernel for few rows (tree_attention_few.cu): whether it takes a call, and the call.
bool tree_is_few(const TreeRows& r);
int tree_attention_few(const TreeRows& r, int hd, bool bf16, cudaStream_t s);

// A sequence's cached positions, and those with its nodes; false if out of range.  No
// sequence, or none of its nodes there: no keys, nothing to compute.
__device__ __forceinline__ bool span(const TreeRows& a, int b, int& len, int& keys) {
  const int64_t most = (int64_t)a.kv.max_pages * a.kv.page_size;
  const int n = a.lengths[b], have = a.counts ? a.counts[b] : a.nodes;
  const int real = min(have, a.nodes);
  len = keys = 0;
  if (n < 0 || real <= 0) return have <= a.nodes;
  keys = static_cast<int>(min((int64_t)n + real, most));
  len = min(n, keys);
  return have <= a.nodes && (int64_t)n + real <= most;
}

// Which of the 64 keys from j0 on a node sees.
__device__ __forceinline__ uint64_t seen_keys(const TreeRows& a, int b, int node, int len, int keys,
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

// The same for trees of up to 64 nodes, whose word w is at hand.
__device__ __forceinline__ uint64_t seen_keys(uint64_t w, int len, int keys, int j0) {
  const int off = len - j0, real = keys - j0;
  const uint64_t mask = off >= 64 ? ~0ull : off > 0 ? w << off | ((1ull << off) - 1) : off > -64 ? w >> -off : 0;
  return real >= 64 ? mask : real <= 0 ? 0 : mask & ((1ull << real) - 1);
}

// Whether a node sees no key at all.
__device__ __forceinline__ bool blind(const TreeRows& a, int b, int node, int len, int keys) {
  bool none = len == 0;
  for (int j = 0; j < keys && none; j += 64) none = seen_keys(a, b, node, len, keys, j) == 0;
  return none;
}

// A page that the kernel's own look-up has checked already.
__device__ __forceinline__ int64_t checked_page(const TreeRows& a, int b, int entry) {
  const int64_t page = entry < a.kv.max_pages ? a.kv.table[b * a.kv.table_stride + entry] : -1;
  return page >= 0 && page < a.kv.num_pages ? page : 0;
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

// One row by the formula, by one warp: 32 keys a step, one to a lane, then the
// values of those that the node sees, HD / 32 dims to a lane; dims [from, to) are written.  For rows that met an
// infinity or NaN among the values of a node they do not see (a probability of 0
// does not silence it).  131072 keys take some 10 ms, 45 with every warp of the GPU at it.
template <typename T, int HD>
__device__ __noinline__ void redo_row(const TreeRows& a, int b, int node, int head, int len, int keys,
                                      int from, int to) {
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
      const int64_t p = checked_page(a, b, j / page), in = ((int64_t)kv_head * page + j % page) * HD;
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
    if (w * 64 + lane * 2 >= from && w * 64 + lane * 2 < to)
      *reinterpret_cast<uint32_t*>(out + w * 64 + lane * 2) = T::pack(acc[w].x * inv, acc[w].y * inv);
}

// A row whose result is not finite: computed again if a value of a node that it does not
// see is not.
template <typename T, int HD>
__device__ __noinline__ void mend_row(const TreeRows& a, int b, int node, int head, int len, int keys,
                                      int from, int to) {
  const int lane = threadIdx.x & 31, page = a.kv.page_size;
  __syncwarp();
  uint32_t met = 0;
  for (int j = len; j < keys; ++j) {
    if (seen_keys(a, b, node, len, keys, j) & 1) continue;
    const uint16_t* v = a.kv.v + checked_page(a, b, j / page) * a.kv.v_stride +
                        ((int64_t)(head / a.group) * page + j % page) * HD;
#pragma unroll
    for (int w = 0; w < HD / 64; ++w)
      met = trace_odd<T>(*reinterpret_cast<const uint32_t*>(v + w * 64 + lane * 2), met);
  }
  if (__any_sync(0xffffffffu, met)) redo_row<T, HD>(a, b, node, head, len, keys, from, to);
}

}  // namespace moe
