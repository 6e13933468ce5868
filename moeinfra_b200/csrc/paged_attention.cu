// Attention of one new token per sequence over a paged key/value cache.
//
//   o[b, h] = sum_j softmax_j(scale q[b,h] . k_j) v_j   over the lengths[b] keys of b,
//
// query head h reading KV head h / (heads / kv_heads).  One pass over the keys
// with the running maximum m, sum l and weighted sum O of the softmax:
//   m' = max(m, s_j);  l' = l 2^(m-m') + 2^(s_j-m');  O' = O 2^(m-m') + 2^(s_j-m') v_j
// (s in units of log2 e).  Two such triples over disjoint keys join the same way.
//
// Bound by memory: every key and value is read once for all query heads of
// its KV head (4 flops a byte per head, far below the tensor cores' rate), so
// what counts is bytes in flight and an even split.
//   * Rows come in chunks of 16 keys.  Where it pays (whole_units), each
//     (sequence, KV head) is a CTA's, its chunks cut evenly over 8 warps, or over 4
//     with two CTAs to an SM, one's start and end under the other's loads.
//   * Else all chunks form one line: sequence by sequence, KV head by KV head.  The
//     line is cut evenly over the CTAs and within a CTA over its 8 warps, whatever
//     the lengths are; the cuts are found on the device from the lengths, so a
//     captured graph follows them.
//   * Each warp owns a ring of chunks in shared memory that it fills with
//     cp.async (rows past a sequence's end as zeros: what lies there is never
//     read) and never waits for another warp: 192 KB in flight per SM at most.
//   * S^T = K Q^T and O^T = V^T P^T on mma.sync 16 x 8 x 16: keys, then head
//     dimensions, fill the 16 rows and the query heads of a group the 8
//     columns, so a group of 4 wastes half a tile instead of three quarters.
//     (tcgen05 wants 128 rows; with at most 16 heads to a key they would be
//     empty, and the memory bound is already reached.)
//   * Pieces of a (sequence, KV head) are joined in the order of their keys:
//     within a CTA through shared memory, between CTAs by the last of them to
//     finish.  The sums' order depends on the shapes, the lengths and the GPU only.
// Measured in a graph with a workspace given (32 / 8 heads of 128): 64 sequences of
// about 576 fp16 29.3 us (152 MB, 5.2 TB/s), 64 of 2048 82 us (6.5 TB/s, what a plain
// copy reaches), four of about 100000 bf16 263 us (6.6 TB/s); one of 72 4.0 us, a chain
// of latencies.  Heads of 64: 64 of about 576 bf16 14.8 us (5.1 TB/s).
#include "paged.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

constexpr int kMaxWarps = 8;        // of a CTA that is alone on its SM; with two to an SM it has half
constexpr int kChunk = 16;          // keys per chunk (a page holds whole chunks)
constexpr int kMaxSeqs = 4095;      // what they need of shared memory: see line_bytes
// Places in the line are 32-bit, and a share's end or a look ahead may lie a little
// past the last one.
constexpr int64_t kMostChunks = INT32_MAX - 4096;
// Smallest share of a CTA in chunks when the line is cut: below it a CTA's
// pieces cost more to join than they save (1 x 4096: 13.9 us with 8, 9.8 with 16,
// 10.0 with 32; 32 x 100: 10.9, 11.2, 13.6).
constexpr int kMinShare = 16;

struct PagedArgs {
  const uint16_t* q;
  int64_t q_stride;       // elements from one sequence's row to the next
  uint16_t* out;          // [B, heads, HD]
  const int32_t* lengths;
  KvPages kv;
  float scale_log2;       // scale * log2(e)
  int heads, per_seq;     // query heads; units (head tiles) of a sequence
  int tile;               // query heads of a unit, at most 8 * NT
  int parts;              // units of a KV head (more than one above 16 heads)
  int page_chunks;        // chunks of a page
  int page_shift;         // log2 of that, or -1
  int* counts;            // [CTAs]: pieces written of the unit that starts in a CTA; zero between calls
  float* part;            // [CTAs][2] pieces
  float* warp_part;       // [CTAs][kMaxWarps] pieces
};

// A piece in memory: O [heads of a tile][HD + 4] fp32 (the pad keeps the 4
// heads that a quad writes in different banks), then m and l per head.
template <int HD, int NT>
constexpr int piece_floats() { return NT * 8 * (HD + 4) + 2 * NT * 8; }

template <int HD>
constexpr int stages() { return HD == 128 ? 3 : 6; }  // 192 KB of ring either way
template <int HD>
constexpr int stage_bytes() { return 2 * kChunk * HD * 2; }
template <int HD, int WARPS>
constexpr int ring_bytes() { return WARPS * stages<HD>() * stage_bytes<HD>(); }
// The line in shared memory: prefix sums of the chunk counts, and the rows of each
// sequence's last chunk (1 to 16) in a byte.
constexpr int line_bytes(int seqs) { return (seqs + 1) * 4 + seqs; }
template <int HD, bool WHOLE, int WARPS>
constexpr int smem_bytes(int seqs) { return ring_bytes<HD, WARPS>() + (WHOLE ? 0 : line_bytes(seqs)); }
// At most what the kernel's __shared__ arrays take, paddings included.
template <int HD, int NT, int WARPS>
constexpr int static_bytes() {
  return 16 * (WARPS * stages<HD>() + 2 * WARPS + 2) + 4 * (WARPS + 2 * WARPS * 2 * NT * 8) + 256;
}

// Chunk x of the line: its sequence b, unit u (head tile) in it, the unit's
// number of chunks n and the chunk's place kc in it.  prefix counts the chunks
// of one unit per sequence.
struct Where {
  int b, u, n, kc;
};
__device__ __forceinline__ Where where(int x, const int* prefix, int seqs, int per_seq) {
  int lo = 0, hi = seqs;  // last b with prefix[b] * per_seq <= x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] * per_seq <= x) lo = mid;
    else hi = mid;
  }
  const int n = prefix[lo + 1] - prefix[lo];
  const uint32_t r = x - prefix[lo] * per_seq, u = r / (uint32_t)n;
  return Where{lo, (int)u, n, (int)(r - u * n)};
}

__device__ __forceinline__ int clamp_len(int len, const KvPages& kv) {
  const int64_t most = (int64_t)kv.max_pages * kv.page_size;
  return len < 0 ? 0 : (len > most ? static_cast<int>(most) : len);
}

// One lane's HD / 32 values of output row (b, h), divided by the softmax's sum.
template <typename T, int HD>
__device__ __forceinline__ void write_row(const PagedArgs& a, int b, int h, int lane,
                                          const float (&acc)[HD / 32], float sum) {
  constexpr int kVec = HD / 32;
  const float inv = __fdividef(1.f, sum);
  uint32_t* o = reinterpret_cast<uint32_t*>(a.out + ((int64_t)b * a.heads + h) * HD + lane * kVec);
#pragma unroll
  for (int v = 0; v < kVec; v += 2) o[v / 2] = T::pack(acc[v] * inv, acc[v + 1] * inv);
}

// WHOLE: CTA x has unit x to itself (see whole_units).  Then nothing depends on
// the other sequences' lengths, and the unit's pages, its queries and its
// length are read at once instead of one after the other.
template <typename T, int HD, int NT, bool WHOLE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, kMaxWarps / WARPS) k_paged_attention(const PagedArgs a) {
  constexpr int kWarps = WARPS, kThreads = WARPS * 32;
  constexpr int S = stages<HD>(), kHeads = NT * 8, kPitch = HD + 4;
  constexpr int kRow = HD * 2;                  // bytes of a row
  constexpr int kTile = kChunk * kRow;          // bytes of a chunk's keys (or values)
  extern __shared__ __align__(128) unsigned char smem[];
  // Of an SM's 228 KB each CTA loses one.
  static_assert(smem_bytes<HD, WHOLE, WARPS>(kMaxSeqs) + static_bytes<HD, NT, WARPS>() <=
                    228 * 1024 * WARPS / kMaxWarps - 1024,
                "shared memory");
  int* prefix = reinterpret_cast<int*>(smem + ring_bytes<HD, WARPS>());
  unsigned char* s_rest = reinterpret_cast<unsigned char*>(prefix + a.kv.seqs + 1);
  __shared__ int s_scan[kWarps];
  __shared__ int4 s_info[kWarps][S];            // b, u, rows that count, bit 0 first / bit 1 last
  __shared__ int4 s_piece[2 * kWarps];           // b (or -1), u, bit 0 first / bit 1 last
  __shared__ float s_ml[2 * kWarps][2][kHeads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const KvPages& kv = a.kv;
  const int per_seq = a.per_seq;
  // Rows sit at their own pitch, 16-byte pieces exchanged by the low bits of
  // the row: the 8 rows of an ldmatrix tile touch all banks.
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) +
                        warp * S * stage_bytes<HD>();
  constexpr int kPieces = HD / 8, kRows = 32 / kPieces, kSame = 8 / kRows;
  const int cp_row = lane / kPieces, cp_piece = lane % kPieces;
  uint32_t cp_at[kSame];  // the pattern repeats after 8 rows
#pragma unroll
  for (int i = 0; i < kSame; ++i) {
    const int r = i * kRows + cp_row;
    cp_at[i] = ring + r * kRow + ((cp_piece ^ r) << 4);
  }
  const int cp_el = cp_row * HD + cp_piece * 8;
  uint32_t qf[NT][HD / 16][2];
  auto load_q = [&](uint32_t (&dst)[NT][HD / 16][2], int b, int u) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool real = nt * 8 + g < a.tile;
      const uint16_t* src =
          a.q + b * a.q_stride + (int64_t)(u * a.tile + (real ? nt * 8 + g : 0)) * HD + 2 * t4;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        dst[nt][kk][0] = !real ? 0u : *reinterpret_cast<const uint32_t*>(src + kk * 16);
        dst[nt][kk][1] = !real ? 0u : *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8);
      }
    }
  };
  if (tid < 2 * kWarps) s_piece[tid] = make_int4(-1, 0, 0, 0);
  pdl_trigger();
  pdl_wait();

  int lo, hi, share = 0;  // this CTA's chunks (WHOLE: counted in the unit)
  int own_b = 0, own_u = 0, own_len = 0;
  int64_t own_page[2] = {};  // WHOLE: pages of the chunks lane and lane + 32
  if constexpr (WHOLE) {
    own_b = blockIdx.x / (uint32_t)per_seq;
    own_u = blockIdx.x - own_b * per_seq;
    const int len = a.lengths[own_b];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int kc = lane + 32 * i, entry = a.page_shift >= 0 ? kc >> a.page_shift : kc / a.page_chunks;
      own_page[i] = entry < kv.max_pages ? kv.table[own_b * kv.table_stride + entry] : -1;
    }
    load_q(qf, own_b, own_u);
    own_len = clamp_len(len, kv);
    if (own_len != len && tid == 0) set_device_error(kErrPage);
    lo = 0;
    hi = (own_len + kChunk - 1) / kChunk;
  }
  // Prefix sums of the sequences' chunk counts.
  if constexpr (!WHOLE) {
  int run = 0;
  for (int b0 = 0; b0 < kv.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < kv.seqs) {
      const int len = a.lengths[b], c = clamp_len(len, kv);
      if (c != len && blockIdx.x == 0) set_device_error(kErrPage);
      n = (c + kChunk - 1) / kChunk;
      s_rest[b] = c - (n - 1) * kChunk;  // not used where n is 0
    }
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s_scan[warp] = inc;
    __syncthreads();
    int before = run, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      all += s_scan[w];
    }
    if (b < kv.seqs) prefix[b] = before + inc - n;
    run += all;
    __syncthreads();
  }
  if (tid == 0) prefix[kv.seqs] = run;
  __syncthreads();
  const int total = run * per_seq;
  share = max((int)(((uint32_t)total + gridDim.x - 1) / gridDim.x), kMinShare);
  lo = (int)min((int64_t)blockIdx.x * share, (int64_t)total);
  hi = min(lo + share, total);
  }
  const int each = (hi - lo + kWarps - 1) / kWarps;
  const int ws = min(lo + warp * each, hi), we = min(ws + each, hi);

  // ---- this warp's chunks [ws, we) ----
  // Places of the next 32 chunks, one per lane (computed once per 32).
  int d_base = ws;
  int64_t d_k = 0, d_v = 0;
  int d_u = 0, d_b = 0, d_rows = 0, d_ends = 0;
  auto look_up = [&](int base) {
    d_base = base;
    const int x = base + lane;
    Where w{own_b, own_u, hi, x};
    int64_t page = 0;
    int entry = 0;
    if constexpr (WHOLE) {
      const int64_t p0 = __shfl_sync(0xffffffffu, own_page[0], x & 31);
      const int64_t p1 = __shfl_sync(0xffffffffu, own_page[1], x & 31);
      page = x < 32 ? p0 : p1;
    }
    if (x >= we) return;
    if constexpr (!WHOLE) w = where(x, prefix, kv.seqs, per_seq);
    entry = a.page_shift >= 0 ? w.kc >> a.page_shift : w.kc / a.page_chunks;
    if (!WHOLE || x >= 64) page = kv.table[w.b * kv.table_stride + entry];
    if (page < 0 || page >= kv.num_pages) {
      set_device_error(kErrPage);
      page = 0;
    }
    const int head = a.parts == 1 ? w.u : w.u / a.parts;
    const int64_t in_page =
        ((int64_t)head * kv.page_size + (w.kc - entry * a.page_chunks) * kChunk) * HD;
    d_k = page * kv.k_stride + in_page;
    d_v = page * kv.v_stride + in_page;
    d_u = w.u;
    d_b = w.b;
    d_ends = (w.kc == 0 ? 1 : 0) | (w.kc == w.n - 1 ? 2 : 0);
    d_rows = d_ends < 2 ? kChunk : WHOLE ? own_len - w.kc * kChunk : s_rest[w.b];
  };

  // A unit's queries are loaded when its first chunk is issued, ahead of their
  // use, where the registers allow it (not for 16 heads of 128).
  constexpr bool kAhead = !WHOLE && NT * HD <= 128;
  uint32_t qn[NT][HD / 16][2];
  int ahead_b = -1, ahead_u = 0;  // whose queries qn holds

  auto issue = [&](int x, int stage) {
    if (x < we) {
      if (x - d_base == 32) look_up(x);
      const int from = x - d_base;
      const int64_t ok = __shfl_sync(0xffffffffu, d_k, from), ov = __shfl_sync(0xffffffffu, d_v, from);
      const int rows = __shfl_sync(0xffffffffu, d_rows, from);
      if (lane == from) s_info[warp][stage] = make_int4(d_b, d_u, d_rows, d_ends);
      const uint32_t off = stage * stage_bytes<HD>();
      const uint16_t *pk = kv.k + ok + cp_el, *pv = kv.v + ov + cp_el;
#pragma unroll
      for (int i = 0; i < kChunk / kRows; ++i) {
        const uint32_t at = cp_at[i % kSame] + off + i / kSame * 8 * kRow;
        const bool take = i * kRows + cp_row < rows;
        cp_async16(at, pk + i * kRows * HD, take);
        cp_async16(at + kTile, pv + i * kRows * HD, take);
      }
      if constexpr (kAhead) {
        const int ends = __shfl_sync(0xffffffffu, d_ends, from);
        if (ahead_b < 0 && ((ends & 1) || x == ws)) {
          ahead_b = __shfl_sync(0xffffffffu, d_b, from);
          ahead_u = __shfl_sync(0xffffffffu, d_u, from);
          load_q(qn, ahead_b, ahead_u);
        }
      }
    }
    cp_async_commit();
  };

  float o[NT][HD / 16][4];
  float m[NT][2], l[NT][2];
  int cur_b = -1, cur_u = 0;  // the unit at hand
  bool cur_first = false;
  if (ws < we) look_up(ws);
#pragma unroll 1
  for (int s = 0; s < S - 1; ++s) issue(ws + s, s);
  int stage = 0;
  for (int x = ws; x < we; ++x) {
    const int next = stage == 0 ? S - 1 : stage - 1;
    __syncwarp();  // every lane is done with the stage that is refilled now
    issue(x + S - 1, next);
    cp_async_wait<S - 1>();
    __syncwarp();
    const int4 info = s_info[warp][stage];
    if (cur_b < 0) {  // a new unit: its queries, an empty softmax
      cur_b = info.x;
      cur_u = info.y;
      cur_first = info.w & 1;
      if (kAhead && ahead_b == cur_b && ahead_u == cur_u) {
        ahead_b = -1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            qf[nt][kk][0] = qn[nt][kk][0];
            qf[nt][kk][1] = qn[nt][kk][1];
          }
      } else if (!WHOLE) {
        load_q(qf, cur_b, cur_u);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
    }
    const uint32_t kt = ring + stage * stage_bytes<HD>(), vt = kt + kTile;
    const int mi = lane >> 3, r8 = lane & 7;
    float sc[NT][2][4] = {};
    {
      const uint32_t row = kt + (r8 + (mi & 1) * 8) * kRow;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t kf[4];
        ldsm4(kf, row + (((kk * 2 + (mi >> 1)) ^ r8) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(sc[nt][kk & 1], kf, qf[nt][kk][0], qf[nt][kk][1]);
      }
    }
    uint32_t pf[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = (sc[nt][0][i] + sc[nt][1][i]) * a.scale_log2;
        if (g + (i >> 1) * 8 >= info.z) s[i] = -INFINITY;
      }
      float mx[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], off));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], off));
      }
      if (__any_sync(0xffffffffu, mx[0] > m[nt][0] || mx[1] > m[nt][1])) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float nm = fmaxf(m[nt][c], mx[c]);
          const float f = m[nt][c] == nm ? 1.f : exp2_approx(m[nt][c] - nm);
          m[nt][c] = nm;
          l[nt][c] *= f;
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            o[nt][i][c] *= f;
            o[nt][i][2 + c] *= f;
          }
        }
      }
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ref = m[nt][i & 1] == -INFINITY ? 0.f : m[nt][i & 1];
        p[i] = exp2_approx(s[i] - ref + T::kProbShift);
        l[nt][i & 1] += p[i];
      }
      // Rows are keys here and have to be columns for the product with V.
      pf[nt][0] = transpose8x8(T::pack(p[0], p[1]));
      pf[nt][1] = transpose8x8(T::pack(p[2], p[3]));
    }
    {
      const uint32_t row = vt + (r8 + (mi >> 1) * 8) * kRow;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        uint32_t vf[4];
        ldsm4_trans(vf, row + (((i * 2 + (mi & 1)) ^ r8) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][i], vf, pf[nt][0], pf[nt][1]);
      }
    }
    stage = stage + 1 == S ? 0 : stage + 1;
    const bool unit_ends = info.w & 2;
    if (!unit_ends && x + 1 < we) continue;

    // ---- the warp's piece of this unit is done ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], off);
    if (cur_first && unit_ends) {  // the whole unit: write it
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = nt * 8 + 2 * t4 + c;
          if (col >= a.tile) continue;
          const float inv = __fdividef(1.f, l[nt][c]);
          uint16_t* dst = a.out + ((int64_t)cur_b * a.heads + cur_u * a.tile + col) * HD;
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            dst[i * 16 + g] = T::one(o[nt][i][c] * inv);
            dst[i * 16 + 8 + g] = T::one(o[nt][i][2 + c] * inv);
          }
        }
    } else {  // the warp's first piece to global memory, its last one to its ring
      const bool last = x + 1 == we;
      const int slot = 2 * warp + (last ? 1 : 0);
      if (last) {
        cp_async_wait<0>();
        __syncwarp();
      }
      float* dst = last ? reinterpret_cast<float*>(smem + warp * S * stage_bytes<HD>())
                        : a.warp_part + ((int64_t)blockIdx.x * kWarps + warp) * piece_floats<HD, NT>();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int col = nt * 8 + 2 * t4 + c;
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            dst[col * kPitch + i * 16 + g] = o[nt][i][c];
            dst[col * kPitch + i * 16 + 8 + g] = o[nt][i][2 + c];
          }
          if (g == 0) {
            s_ml[slot][0][col] = m[nt][c];
            s_ml[slot][1][col] = l[nt][c];
          }
        }
      if (lane == 0)
        s_piece[slot] = make_int4(cur_b, cur_u, (cur_first ? 1 : 0) | (unit_ends ? 2 : 0), 0);
    }
    cur_b = -1;
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- join the warps' pieces, unit by unit, in the order of the keys ----
  // Lane i holds slot i; every warp sees the same slots and takes its share of
  // the (unit, head) sums, one row of HD values each.  A warp holds at most one
  // piece of a unit, so a sum has at most kWarps terms: all are read at once.
  constexpr int kVec = HD / 32;
  const int4 held = s_piece[lane & (2 * kWarps - 1)];
  const bool full = lane < 2 * kWarps && held.x >= 0;
  const uint32_t used = __ballot_sync(0xffffffffu, full);
  const uint32_t firsts = __ballot_sync(0xffffffffu, full && (held.z & 1));
  const uint32_t lasts = __ballot_sync(0xffffffffu, full && (held.z & 2));
  // A sum begins at the first piece and after each last one.
  const uint32_t below = used & ((1u << lane) - 1);
  uint32_t starts = __ballot_sync(
      0xffffffffu, full && (below == 0 || (lasts >> (31 - __clz(below)) & 1)));
  int open = 0;              // pieces of units that other CTAs share: bit 0 and 1 as the slot
  int turn = 0;
  while (starts) {
    const int i = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t range = used & ~((1u << i) - 1) & (starts ? (starts & -starts) - 1 : ~0u);
    const int b = WHOLE ? own_b : __shfl_sync(0xffffffffu, held.x, i);
    const int u = WHOLE ? own_u : __shfl_sync(0xffffffffu, held.y, i);
    const bool first = firsts & range, last = lasts & range, all = WHOLE || (first && last);
    float* dst = a.part + ((int64_t)blockIdx.x * 2 + (first ? 1 : 0)) * piece_floats<HD, NT>();
    if (!all) open |= first ? 2 : 1;
    for (int col = (warp - turn) & (kWarps - 1); col < a.tile; col += kWarps) {
      float ms[kWarps], val[kWarps][kVec], mm = -INFINITY, ll = 0.f, acc[kVec] = {};
      uint32_t rest = range;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const int sk = rest ? __ffs(rest) - 1 : -1;
        rest &= rest - 1;
        ms[k] = -INFINITY;
        if (sk < 0) continue;
        const float* p =
            ((sk & 1) ? reinterpret_cast<const float*>(smem + (sk >> 1) * S * stage_bytes<HD>())
                      : a.warp_part + ((int64_t)blockIdx.x * kWarps + (sk >> 1)) * piece_floats<HD, NT>()) +
            col * kPitch + lane * kVec;
#pragma unroll
        for (int v = 0; v < kVec; ++v) val[k][v] = p[v];
        ms[k] = s_ml[sk][0][col];
        mm = fmaxf(mm, ms[k]);
      }
      rest = range;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        if (!rest) continue;
        const float f = ms[k] == mm ? 1.f : exp2_approx(ms[k] - mm);
        ll += f * s_ml[__ffs(rest) - 1][1][col];
        rest &= rest - 1;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] += f * val[k][v];
      }
      if (all) {
        write_row<T, HD>(a, b, u * a.tile + col, lane, acc, ll);
      } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v) dst[col * kPitch + lane * kVec + v] = acc[v];
        if (lane == 0) {
          dst[kHeads * kPitch + col] = mm;
          dst[kHeads * kPitch + kHeads + col] = ll;
        }
      }
    }
    turn += a.tile;
  }

  // Sequences without keys: zeros.
  if constexpr (WHOLE) {
    if (hi == 0)
      for (int col = warp; col < a.tile; col += kWarps) {
        const float none[kVec] = {};
        write_row<T, HD>(a, own_b, own_u * a.tile + col, lane, none, 1.f);
      }
  } else {
  for (int b = blockIdx.x; b < kv.seqs; b += gridDim.x) {
    if (prefix[b + 1] != prefix[b]) continue;
    uint32_t* o = reinterpret_cast<uint32_t*>(a.out + (int64_t)b * a.heads * HD);
    for (int i = tid; i < a.heads * HD / 2; i += kThreads) o[i] = 0;
  }
  if (!open) return;

  // ---- join the CTAs' pieces: the last CTA of a unit to get here does it ----
  // A unit is counted at the CTA that holds its start.  Whoever finds the count
  // full sees every piece (each CTA's are fenced before its count) and sets the
  // counter back to zero for the next launch.
  // Bit 0: the piece of the unit that the CTA's first chunk belongs to; bit 1:
  // that of its last chunk.
  __shared__ int4 s_join[2];  // b, u, first CTA, pieces (0: not the last)
  __threadfence();
  __syncthreads();
  if (tid < 2) {
    s_join[tid].w = 0;
    if (open >> tid & 1) {
      const Where w = where(tid ? hi - 1 : lo, prefix, kv.seqs, per_seq);
      const int from = prefix[w.b] * per_seq + w.u * w.n;
      const int c0 = from / share, np = (from + w.n - 1) / share - c0 + 1;
      if (atomicAdd(a.counts + c0, 1) == np - 1) {
        a.counts[c0] = 0;
        s_join[tid] = make_int4(w.b, w.u, c0, np);
      }
    }
  }
  __syncthreads();
  for (int w = 0; w < 2; ++w) {
    const int4 job = s_join[w];
    const int np = job.w;
    if (np == 0) continue;
    __threadfence();
    // Piece 0 is CTA c0's second, the others the first of the CTAs after it.
    const float* base = a.part + (int64_t)job.z * 2 * piece_floats<HD, NT>();
    for (int col = warp; col < a.tile; col += kWarps) {
      float mm = -INFINITY, ll = 0.f, acc[kVec] = {};
#pragma unroll 4
      for (int k = 0; k < np; ++k) {
        const float* p = base + (int64_t)(k == 0 ? 1 : 2 * k) * piece_floats<HD, NT>();
        const float ms = __ldcg(p + kHeads * kPitch + col), ls = __ldcg(p + kHeads * kPitch + kHeads + col);
        float val[kVec];
#pragma unroll
        for (int v = 0; v < kVec; ++v) val[v] = __ldcg(p + col * kPitch + lane * kVec + v);
        const float nm = fmaxf(mm, ms);
        const float f0 = mm == nm ? 1.f : exp2_approx(mm - nm), f1 = ms == nm ? 1.f : exp2_approx(ms - nm);
        ll = ll * f0 + ls * f1;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] = acc[v] * f0 + val[v] * f1;
        mm = nm;
      }
      write_row<T, HD>(a, job.x, job.y * a.tile + col, lane, acc, ll);
    }
  }
  }
}

template <typename T, int HD, int NT, bool WHOLE, int WARPS>
bool paged_attr() {
  return cudaFuncSetAttribute(k_paged_attention<T, HD, NT, WHOLE, WARPS>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              smem_bytes<HD, WHOLE, WARPS>(kMaxSeqs)) == cudaSuccess;
}

// Whether a call gives each unit (sequence, KV head, head tile) a CTA of its
// own, which joins nothing with others and reads its page numbers, queries and
// length at once; or cuts the line evenly.  The table's width is all that is known
// of the lengths here, so a CTA's share must not become too long where few units
// are long; and a CTA for a few chunks is a wave of latencies for each 2 to an SM.
// Measured in a graph (fp16, 32 heads of 128, 8 KV heads, own CTAs / even cut, us):
//   1 x 72 3.8 / 9.2, 8 x 576 7.1 / 10.9, 64 x 576 28.4 / 35.2, 64 x 2048 81 / 92,
//   64 ragged up to 1972 46.9 / 54.7; but 1 x 1024 8.8 / 7.9, one of 2048 and 63 of
//   16 19.5 / 9.4, one of 4096 and 63 of 16 35.7 / 14.3;
//   512 units of 48 6.8 / 11.8, of 100 8.8 / 13.8; but 2048 units of 48 26 / 12.6, of
//   100 32 / 31, of 160 38.7 / 41.6, of 256 51 / 58.
bool whole_units(int64_t units, int64_t chunks) {
  const int64_t sms = sm_count();
  if (units <= sms) return chunks <= 64;
  return chunks <= 128 && (chunks >= 12 || units <= 4 * sms);
}

struct Shape {
  int parts, tile, nt;
  int64_t units, chunks;
  int ctas;
  bool whole;
};
Shape shape_of(int64_t seqs, int kv_heads, int group, int64_t max_tokens) {
  Shape s;
  // Groups above 16 heads are read by several units, of equal numbers of heads: 24 by
  // two of 12, but a prime number by as many units of one head, each of which reads
  // the keys (from L2 at best: 64 sequences of about 576, 1 KV head of 128, 17 heads
  // 35.8 us, 16 heads 11.3).
  s.parts = static_cast<int>(ceil_div(group, 16));
  while (group % s.parts) ++s.parts;
  s.tile = group / s.parts;
  s.nt = s.tile <= 8 ? 1 : 2;
  s.units = seqs * kv_heads * s.parts;
  s.chunks = ceil_div(max_tokens, kChunk);
  s.whole = whole_units(s.units, s.chunks);
  s.ctas = s.whole ? static_cast<int>(s.units) : sm_count();
  return s;
}

// The counters lead, so that calls of any shape keep them at the same place.  The
// pieces follow, as many as a cut line has: whether a call cuts it changes back and
// forth with the number of sequences and the table's width, and a workspace made
// for the largest batch has to serve the smaller ones.
constexpr size_t kCountBytes = 4096;
size_t workspace_size(const Shape& s, int hd) {
  return kCountBytes +
         sizeof(float) * sm_count() * (2 + kMaxWarps) * (s.nt * 8 * (hd + 4) + 2 * s.nt * 8);
}

template <typename T, int HD, int NT, bool WHOLE, int WARPS>
int launch_paged(PagedArgs& a, const Shape& sh, cudaStream_t s) {
  if (!once_per_device(reinterpret_cast<const void*>(&paged_attr<T, HD, NT, WHOLE, WARPS>),
                       &paged_attr<T, HD, NT, WHOLE, WARPS>))
    return MOE_ERR_CUDA;
  a.part = a.warp_part + (size_t)sh.ctas * kMaxWarps * piece_floats<HD, NT>();
  if (launch_pdl(k_paged_attention<T, HD, NT, WHOLE, WARPS>, dim3(sh.ctas), dim3(WARPS * 32),
                 smem_bytes<HD, WHOLE, WARPS>(a.kv.seqs), s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <typename T, int HD, int NT>
int launch_tile(PagedArgs& a, const Shape& sh, cudaStream_t s) {
  if (!sh.whole) return launch_paged<T, HD, NT, false, kMaxWarps>(a, sh, s);
  return sh.units <= sm_count() ? launch_paged<T, HD, NT, true, kMaxWarps>(a, sh, s)
                                : launch_paged<T, HD, NT, true, kMaxWarps / 2>(a, sh, s);
}

template <typename T, int HD>
int launch_wide(PagedArgs& a, const Shape& sh, cudaStream_t s) {
  return sh.nt == 1 ? launch_tile<T, HD, 1>(a, sh, s) : launch_tile<T, HD, 2>(a, sh, s);
}

}  // namespace
}  // namespace moe

extern "C" size_t moe_paged_attention_workspace_size(int64_t seqs, int64_t max_pages,
                                                     int64_t page_size, int64_t heads,
                                                     int64_t kv_heads, int64_t head_dim) {
  using namespace moe;
  if (seqs < 1 || kv_heads < 1 || heads < kv_heads || max_pages < 0 || page_size < 1 ||
      (head_dim != 64 && head_dim != 128) || seqs > kMaxSeqs || heads > 4096)
    return 0;
  const Shape sh = shape_of(seqs, kv_heads, heads / kv_heads, max_pages * page_size);
  return workspace_size(sh, static_cast<int>(head_dim));
}

extern "C" int moe_paged_attention(const moe_paged_attention_args_t* args) {
  using namespace moe;
  if (!args) return MOE_ERR_INVALID_ARG;
  const moe_paged_attention_args_t& c = *args;
  if (const int st = check_pages(c.kv); st != MOE_OK) return st;
  const int64_t hd = c.kv.head_dim;
  const float scale = static_cast<float>(c.scale);
  if (c.heads < 1 || c.heads > 4096 || c.heads % c.kv.kv_heads || !(scale > 0.f && scale < INFINITY) ||
      c.q_stride < c.heads * hd)
    return MOE_ERR_INVALID_ARG;
  if (c.kv.page_size % kChunk || c.kv.seqs > kMaxSeqs) return MOE_ERR_UNSUPPORTED;
  if (c.kv.seqs == 0) return MOE_OK;
  if (!c.q || !c.lengths || !c.out ||
      (c.kv.max_pages > 0 &&
       (!c.kv.k_pages || !c.kv.v_pages || !c.kv.block_table || c.kv.num_pages < 1)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(c.q) || !aligned16(c.out) || (c.q_stride & 7)) return MOE_ERR_ALIGNMENT;
  const Shape sh = shape_of(c.kv.seqs, static_cast<int>(c.kv.kv_heads),
                            static_cast<int>(c.heads / c.kv.kv_heads), c.kv.max_pages * c.kv.page_size);
  if (sh.units * sh.chunks > kMostChunks) return MOE_ERR_UNSUPPORTED;
  if (!c.workspace || c.workspace_bytes < (int64_t)workspace_size(sh, static_cast<int>(hd)))
    return MOE_ERR_WORKSPACE;
  if (!aligned16(c.workspace)) return MOE_ERR_ALIGNMENT;
  PagedArgs a{};
  a.q = c.q;
  a.q_stride = c.q_stride;
  a.out = c.out;
  a.lengths = c.lengths;
  a.kv = pages_of(c.kv);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.heads = static_cast<int>(c.heads);
  a.per_seq = static_cast<int>(c.kv.kv_heads) * sh.parts;
  a.tile = sh.tile;
  a.parts = sh.parts;
  a.page_chunks = a.kv.page_size / kChunk;
  a.page_shift = -1;
  for (int i = 0; i < 27; ++i)
    if (a.page_chunks == 1 << i) a.page_shift = i;
  a.counts = static_cast<int*>(c.workspace);
  a.warp_part = reinterpret_cast<float*>(static_cast<char*>(c.workspace) + kCountBytes);
  cudaStream_t s = static_cast<cudaStream_t>(c.stream);
  if (c.kv.dtype == MOE_DTYPE_F16)
    return hd == 64 ? launch_wide<F16, 64>(a, sh, s) : launch_wide<F16, 128>(a, sh, s);
  return hd == 64 ? launch_wide<BF16, 64>(a, sh, s) : launch_wide<BF16, 128>(a, sh, s);
}
