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
//   * The caches' rows, as chunks of 16 keys, form one line: sequence by
//     sequence, KV head by KV head.  The line is cut evenly over the CTAs and
//     within a CTA over its 8 warps, whatever the lengths are; the cuts are
//     found on the device from the lengths, so a captured graph follows them.
//   * Each warp owns a ring of chunks in shared memory that it fills with
//     cp.async (rows past a sequence's end as zeros: what lies there is never
//     read) and never waits for another warp: 192 KB in flight per SM at most.
//   * S^T = K Q^T and O^T = V^T P^T on mma.sync 16 x 8 x 16: keys, then head
//     dimensions, fill the 16 rows and the query heads of a group the 8
//     columns, so a group of 4 wastes half a tile instead of three quarters.
//     (tcgen05 wants 128 rows; with at most 16 heads to a key they would be
//     empty, and the memory bound is already reached.)
//   * Pieces of a (sequence, KV head) are joined in the order of their keys:
//     within a CTA through shared memory, between CTAs by a second small
//     launch.  The sums' order depends on the lengths and the GPU only.
#include "paged.cuh"

namespace moe {
namespace {

MOE_DEFINE_ERROR_WORD()

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kChunk = 16;          // keys per chunk (a page holds whole chunks)
constexpr int kMaxSeqs = 8191;      // their chunk counts' prefix sums sit in shared memory
// Smallest share of a CTA in chunks when the line is cut: below it a CTA's
// pieces cost more to join than they save.
constexpr int kMinShare = 16;

struct PagedArgs {
  const uint16_t* q;
  int64_t q_stride;       // elements from one sequence's row to the next
  uint16_t* out;          // [B, heads, HD]
  const int32_t* lengths;
  KvPages kv;
  float scale_log2;       // scale * log2(e)
  int group;              // query heads per KV head
  int parts;              // head tiles of a group (more than one above 16 heads)
  bool whole;             // one CTA per unit: no cut, no second launch
  float* part;            // [CTAs][2] pieces
  float* warp_part;       // [CTAs][kWarps] pieces
  int2* meta;             // [CTAs]: the unit whose pieces start in the CTA, their count
};

// A piece in memory: O [heads of a tile][HD + 4] fp32 (the pad keeps the 4
// heads that a quad writes in different banks), then m and l per head.
template <int HD, int NT>
constexpr int piece_floats() { return NT * 8 * (HD + 4) + 2 * NT * 8; }

template <int HD>
constexpr int stages() { return HD == 128 ? 3 : 6; }  // 192 KB of ring either way
template <int HD>
constexpr int stage_bytes() { return 2 * kChunk * HD * 2; }
template <int HD>
constexpr int ring_bytes() { return kWarps * stages<HD>() * stage_bytes<HD>(); }
template <int HD>
int smem_bytes(int seqs) { return ring_bytes<HD>() + (seqs + 1) * 4; }

// Chunk x of the line: its sequence, unit (head tile of a sequence), and place.
struct Where {
  int b, unit, n, kc;
};
__device__ __forceinline__ Where where(int x, const int* prefix, int seqs, int per_seq) {
  int lo = 0, hi = seqs;  // last b with prefix[b] <= x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x) lo = mid;
    else hi = mid;
  }
  const int n = (prefix[lo + 1] - prefix[lo]) / per_seq;
  const int r = x - prefix[lo], u = r / n;
  return Where{lo, lo * per_seq + u, n, r - u * n};
}

__device__ __forceinline__ int clamp_len(int len, const KvPages& kv) {
  const int64_t most = (int64_t)kv.max_pages * kv.page_size;
  return len < 0 ? 0 : (len > most ? static_cast<int>(most) : len);
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kThreads, 1) k_paged_attention(const PagedArgs a) {
  constexpr int S = stages<HD>(), kHeads = NT * 8, kPitch = HD + 4;
  constexpr int kRow = HD * 2;                  // bytes of a row
  constexpr int kTile = kChunk * kRow;          // bytes of a chunk's keys (or values)
  extern __shared__ __align__(128) unsigned char smem[];
  int* prefix = reinterpret_cast<int*>(smem + ring_bytes<HD>());
  __shared__ int s_scan[kWarps];
  __shared__ int4 s_info[kWarps][S];            // unit, b, rows that count, bit 0 first / bit 1 last
  __shared__ int s_unit[2 * kWarps], s_ends[2 * kWarps];
  __shared__ float s_ml[2 * kWarps][2][kHeads];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const KvPages& kv = a.kv;
  const int per_seq = kv.kv_heads * a.parts;
  pdl_trigger();
  pdl_wait();

  // Prefix sums of the sequences' chunk counts (all units of a sequence).
  int run = 0;
  for (int b0 = 0; b0 < kv.seqs; b0 += kThreads) {
    const int b = b0 + tid;
    int n = 0;
    if (b < kv.seqs) {
      const int len = a.lengths[b], c = clamp_len(len, kv);
      if (c != len && blockIdx.x == 0) set_device_error(kErrPage);
      n = (c + kChunk - 1) / kChunk * per_seq;
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
  if (tid < 2 * kWarps) s_unit[tid] = -1;
  __syncthreads();
  const int total = run;

  // Sequences without keys: zeros.
  for (int b = blockIdx.x; b < kv.seqs; b += gridDim.x) {
    if (prefix[b + 1] != prefix[b]) continue;
    uint32_t* o = reinterpret_cast<uint32_t*>(a.out + (int64_t)b * kv.kv_heads * a.group * HD);
    for (int i = tid; i < kv.kv_heads * a.group * HD / 2; i += kThreads) o[i] = 0;
  }

  int lo, hi, share = 0;  // this CTA's chunks
  if (a.whole) {
    const int b = blockIdx.x / per_seq, u = blockIdx.x % per_seq;
    const int n = (prefix[b + 1] - prefix[b]) / per_seq;
    lo = prefix[b] + u * n;
    hi = lo + n;
  } else {
    share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, kMinShare);
    lo = (int)min((int64_t)blockIdx.x * share, (int64_t)total);
    hi = min(lo + share, total);
  }
  const int each = (hi - lo + kWarps - 1) / kWarps;
  const int ws = min(lo + warp * each, hi), we = min(ws + each, hi);

  // ---- this warp's chunks [ws, we) ----
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) +
                        warp * S * stage_bytes<HD>();
  // Rows sit at their own pitch, 16-byte pieces exchanged by the low bits of
  // the row: the 8 rows of an ldmatrix tile touch all banks.
  constexpr int kPieces = HD / 8, kRows = 32 / kPieces;
  const int cp_row = lane / kPieces, cp_piece = lane % kPieces;
  // Places of the next 32 chunks, one per lane (computed once per 32).
  int d_base = ws;
  int64_t d_k = 0, d_v = 0;
  int d_unit = 0, d_b = 0, d_rows = 0, d_ends = 0;
  auto look_up = [&](int base) {
    d_base = base;
    const int x = base + lane;
    if (x >= we) return;
    const Where w = where(x, prefix, kv.seqs, per_seq);
    const int p0 = w.kc * kChunk;
    int64_t page = kv.table[w.b * kv.table_stride + p0 / kv.page_size];
    if (page < 0 || page >= kv.num_pages) {
      set_device_error(kErrPage);
      page = 0;
    }
    const int head = (w.unit - w.b * per_seq) / a.parts;
    const int64_t in_page = ((int64_t)head * kv.page_size + p0 % kv.page_size) * HD;
    d_k = page * kv.k_stride + in_page;
    d_v = page * kv.v_stride + in_page;
    d_unit = w.unit;
    d_b = w.b;
    d_rows = min(kChunk, clamp_len(a.lengths[w.b], kv) - p0);
    d_ends = (w.kc == 0 ? 1 : 0) | (w.kc == w.n - 1 ? 2 : 0);
  };
  auto issue = [&](int x, int stage) {
    if (x < we) {
      if (x - d_base == 32) look_up(x);
      const int from = x - d_base;
      const int64_t ok = __shfl_sync(0xffffffffu, d_k, from), ov = __shfl_sync(0xffffffffu, d_v, from);
      const int rows = __shfl_sync(0xffffffffu, d_rows, from);
      if (lane == from) s_info[warp][stage] = make_int4(d_unit, d_b, d_rows, d_ends);
      const uint32_t dst = ring + stage * stage_bytes<HD>();
#pragma unroll
      for (int i = 0; i < kChunk / kRows; ++i) {
        const int r = i * kRows + cp_row;
        const uint32_t at = dst + r * kRow + ((cp_piece ^ (r & 7)) << 4);
        const int64_t el = (int64_t)r * HD + cp_piece * 8;
        cp_async16(at, kv.k + ok + el, r < rows);
        cp_async16(at + kTile, kv.v + ov + el, r < rows);
      }
    }
    cp_async_commit();
  };

  uint32_t qf[NT][HD / 16][2];
  float o[NT][HD / 16][4];
  float m[NT][2], l[NT][2];
  int cur = -1, cur_b = 0;
  bool cur_first = false;

  auto head_of = [&](int unit, int nt, int col) {  // query head of a column, or -1
    const int u = unit % per_seq, h = (u % a.parts) * kHeads + nt * 8 + col;
    return h < a.group ? u / a.parts * a.group + h : -1;
  };
  if (ws < we) look_up(ws);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) issue(ws + s, s);
  int stage = 0;
  for (int x = ws; x < we; ++x) {
    const int next = stage == 0 ? S - 1 : stage - 1;
    __syncwarp();  // every lane is done with the stage that is refilled now
    issue(x + S - 1, next);
    cp_async_wait<S - 1>();
    __syncwarp();
    const int4 info = s_info[warp][stage];
    if (info.x != cur) {  // a new unit: its queries, an empty softmax
      cur = info.x;
      cur_b = info.y;
      cur_first = info.w & 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = head_of(cur, nt, g);
        const uint16_t* src = a.q + cur_b * a.q_stride + (int64_t)(h < 0 ? 0 : h) * HD + 2 * t4;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          qf[nt][kk][0] = h < 0 ? 0u : *reinterpret_cast<const uint32_t*>(src + kk * 16);
          qf[nt][kk][1] = h < 0 ? 0u : *reinterpret_cast<const uint32_t*>(src + kk * 16 + 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[nt][kk][i] = 0.f;
        }
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
          const int h = head_of(cur, nt, 2 * t4 + c);
          if (h < 0) continue;
          const float inv = 1.f / l[nt][c];
          uint16_t* dst = a.out + ((int64_t)cur_b * kv.kv_heads * a.group + h) * HD;
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
      if (lane == 0) {
        s_unit[slot] = cur;
        s_ends[slot] = (cur_first ? 1 : 0) | (unit_ends ? 2 : 0);
      }
    }
    cur = -1;
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- join the warps' pieces, unit by unit, in the order of the keys ----
  // Lane k holds the k-th piece of the CTA; every warp sees the same list and
  // takes its share of the (unit, head) sums, one row of HD values each.
  const int held = lane < 2 * kWarps ? s_unit[lane] : -1;
  const uint32_t used = __ballot_sync(0xffffffffu, held >= 0);
  const int pieces = __popc(used);
  int slot = 0;
  for (uint32_t rest = used, k = 0; rest; rest &= rest - 1, ++k)
    if (lane == (int)k) slot = __ffs(rest) - 1;
  const int unit_k = __shfl_sync(0xffffffffu, held, slot);
  const int ends_k = lane < pieces ? s_ends[slot] : 0;
  const int unit_before = __shfl_up_sync(0xffffffffu, unit_k, 1);
  uint32_t starts = __ballot_sync(0xffffffffu, lane < pieces && (lane == 0 || unit_k != unit_before));
  const uint32_t firsts = __ballot_sync(0xffffffffu, ends_k & 1);
  const uint32_t lasts = __ballot_sync(0xffffffffu, ends_k & 2);
  const float* src = (slot & 1) ? reinterpret_cast<const float*>(smem + (slot >> 1) * S * stage_bytes<HD>())
                                : a.warp_part + ((int64_t)blockIdx.x * kWarps + (slot >> 1)) * piece_floats<HD, NT>();
  int2 start = make_int2(-1, 0);
  int turn = 0;
  while (starts) {
    const int i = __ffs(starts) - 1;
    starts &= starts - 1;
    const int j = starts ? __ffs(starts) - 1 : pieces;
    const uint32_t range = ((1u << j) - 1) & ~((1u << i) - 1);
    const int unit = __shfl_sync(0xffffffffu, unit_k, i);
    const bool first = firsts & range, last = lasts & range;
    const int cols = min(kHeads, a.group - unit % a.parts * kHeads);
    float* dst = a.part + ((int64_t)blockIdx.x * 2 + (first ? 1 : 0)) * piece_floats<HD, NT>();
    for (int col = 0; col < cols; ++col, turn = turn + 1 == kWarps ? 0 : turn + 1) {
      if (turn != warp) continue;
      const bool mine = lane >= i && lane < j;
      const float ms = mine ? s_ml[slot][0][col] : -INFINITY;
      float mm = ms;
#pragma unroll
      for (int off = 16; off; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
      const float f = ms == mm ? 1.f : exp2_approx(ms - mm);
      float ll = mine ? f * s_ml[slot][1][col] : 0.f;
#pragma unroll
      for (int off = 16; off; off >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
      constexpr int kVec = HD / 32;
      float acc[kVec] = {};
#pragma unroll 4
      for (int k = i; k < j; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float* p = reinterpret_cast<const float*>(
                             __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(src), k)) +
                         col * kPitch + lane * kVec;
#pragma unroll
        for (int v = 0; v < kVec; ++v) acc[v] += fk * p[v];
      }
      if (first && last) {
        const float inv = 1.f / ll;
        const int h = head_of(unit, col >> 3, col & 7);
        uint32_t* o32 = reinterpret_cast<uint32_t*>(
            a.out + ((int64_t)(unit / per_seq) * kv.kv_heads * a.group + h) * HD + lane * kVec);
#pragma unroll
        for (int v = 0; v < kVec; v += 2) o32[v / 2] = T::pack(acc[v] * inv, acc[v + 1] * inv);
      } else {
#pragma unroll
        for (int v = 0; v < kVec; ++v) dst[col * kPitch + lane * kVec + v] = acc[v];
        if (lane == 0) {
          dst[kHeads * kPitch + col] = mm;
          dst[kHeads * kPitch + kHeads + col] = ll;
        }
      }
    }
    if (first && !last) {  // further pieces lie in the CTAs after this one
      const int b = unit / per_seq, n = (prefix[b + 1] - prefix[b]) / per_seq;
      const int end = prefix[b] + (unit - b * per_seq + 1) * n;
      start = make_int2(unit, (end - 1) / share - (int)blockIdx.x + 1);
    }
  }
  if (!a.whole && tid == 0) a.meta[blockIdx.x] = start;
}

// Joins the pieces of the unit that starts in CTA x of the first launch and
// ends in another; one block per head of the tile, one thread per dimension.
template <typename T, int HD, int NT>
__global__ void __launch_bounds__(HD) k_paged_join(const PagedArgs a) {
  constexpr int kHeads = NT * 8, kPitch = HD + 4, kPiece = piece_floats<HD, NT>();
  pdl_trigger();
  pdl_wait();
  const int2 meta = a.meta[blockIdx.x];
  if (meta.x < 0) return;
  const int col = blockIdx.y, d = threadIdx.x;
  const int per_seq = a.kv.kv_heads * a.parts, u = meta.x % per_seq;
  const int h = u % a.parts * kHeads + col;
  if (h >= a.group) return;
  // Piece 0 is the CTA's second, the others the first of the CTAs after it.
  const float* base = a.part + (int64_t)blockIdx.x * 2 * kPiece;
  float mm = -INFINITY, ll = 0.f, oo = 0.f;
#pragma unroll 4
  for (int i = 0; i < meta.y; ++i) {
    const float* p = base + (int64_t)(i == 0 ? 1 : 2 * i) * kPiece;
    const float ms = p[kHeads * kPitch + col], ls = p[kHeads * kPitch + kHeads + col];
    const float os = p[col * kPitch + d];
    const float nm = fmaxf(mm, ms);
    const float f0 = mm == nm ? 1.f : exp2_approx(mm - nm), f1 = ms == nm ? 1.f : exp2_approx(ms - nm);
    ll = ll * f0 + ls * f1;
    oo = oo * f0 + os * f1;
    mm = nm;
  }
  a.out[((int64_t)(meta.x / per_seq) * a.kv.kv_heads * a.group + u / a.parts * a.group + h) * HD + d] =
      T::one(oo / ll);
}

template <typename T, int HD, int NT>
bool paged_attr() {
  return cudaFuncSetAttribute(k_paged_attention<T, HD, NT>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              smem_bytes<HD>(kMaxSeqs)) == cudaSuccess;
}

// Whether a call gives each unit (sequence, KV head, head tile) a CTA of its
// own: few units and a table that holds at most 64 chunks (1024 tokens) each.
// Its 8 warps then read up to 8 chunks one after the other, which takes no
// longer than the second launch that joins a cut would.
bool whole_units(int64_t units, int64_t chunks) { return units <= sm_count() && chunks <= 64; }

struct Shape {
  int parts, nt;
  int64_t units, chunks;
  int ctas;
  bool whole;
};
Shape shape_of(int64_t seqs, int kv_heads, int group, int64_t max_tokens) {
  Shape s;
  s.nt = group <= 8 ? 1 : 2;
  s.parts = static_cast<int>(ceil_div(group, 16));
  s.units = seqs * kv_heads * s.parts;
  s.chunks = ceil_div(max_tokens, kChunk);
  s.whole = whole_units(s.units, s.chunks);
  s.ctas = s.whole ? static_cast<int>(s.units) : sm_count();
  return s;
}

size_t workspace_floats(const Shape& s, int hd) {
  if (s.whole) return (size_t)s.ctas * kWarps * (s.nt * 8 * (hd + 4) + 2 * s.nt * 8);
  return (size_t)s.ctas * (2 + kWarps) * (s.nt * 8 * (hd + 4) + 2 * s.nt * 8) + (size_t)s.ctas * 2;
}

template <typename T, int HD, int NT>
int launch_paged(PagedArgs& a, const Shape& sh, float* ws, cudaStream_t s) {
  if (!once_per_device(reinterpret_cast<const void*>(&paged_attr<T, HD, NT>), &paged_attr<T, HD, NT>))
    return MOE_ERR_CUDA;
  a.warp_part = ws;
  a.part = ws + (size_t)sh.ctas * kWarps * piece_floats<HD, NT>();
  a.meta = reinterpret_cast<int2*>(a.part + (size_t)sh.ctas * 2 * piece_floats<HD, NT>());
  if (launch_pdl(k_paged_attention<T, HD, NT>, dim3(sh.ctas), dim3(kThreads),
                 smem_bytes<HD>(a.kv.seqs), s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  if (sh.whole) return MOE_OK;
  const int cols = a.group < NT * 8 ? a.group : NT * 8;
  if (launch_pdl(k_paged_join<T, HD, NT>, dim3(sh.ctas, cols), dim3(HD), 0, s, a) != cudaSuccess)
    return MOE_ERR_CUDA;
  MOE_CHECK_LAUNCH();
  return MOE_OK;
}

template <typename T>
int launch_typed(PagedArgs& a, const Shape& sh, int hd, float* ws, cudaStream_t s) {
  if (hd == 64)
    return sh.nt == 1 ? launch_paged<T, 64, 1>(a, sh, ws, s) : launch_paged<T, 64, 2>(a, sh, ws, s);
  return sh.nt == 1 ? launch_paged<T, 128, 1>(a, sh, ws, s) : launch_paged<T, 128, 2>(a, sh, ws, s);
}

}  // namespace
}  // namespace moe

extern "C" size_t moe_paged_attention_workspace_size(int seqs, int max_pages, int page_size,
                                                     int heads, int kv_heads, int head_dim) {
  using namespace moe;
  if (seqs < 1 || kv_heads < 1 || heads < kv_heads || max_pages < 0 || page_size < 1 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  const Shape sh = shape_of(seqs, kv_heads, heads / kv_heads, (int64_t)max_pages * page_size);
  return workspace_floats(sh, head_dim) * sizeof(float);
}

extern "C" int moe_paged_attention(const uint16_t* q, int64_t q_stride, uint16_t* k_pages,
                                   uint16_t* v_pages, int64_t k_page_stride,
                                   int64_t v_page_stride, int64_t num_pages, int page_size,
                                   const int32_t* block_table, int64_t table_stride, int seqs,
                                   int max_pages, const int32_t* lengths, int heads, int kv_heads,
                                   int head_dim, int dtype, float scale, uint16_t* out,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  using namespace moe;
  if (seqs < 0 || max_pages < 0 || heads < 1 || kv_heads < 1 || heads % kv_heads || num_pages < 0 ||
      page_size < 1 || !(scale > 0.f) || heads > 4096)
    return MOE_ERR_INVALID_ARG;
  if (dtype != MOE_DTYPE_F16 && dtype != MOE_DTYPE_BF16) return MOE_ERR_UNSUPPORTED;
  if ((head_dim != 64 && head_dim != 128) || page_size % kChunk || seqs > kMaxSeqs)
    return MOE_ERR_UNSUPPORTED;
  const int64_t page_elems = (int64_t)kv_heads * page_size * head_dim;
  if (q_stride < (int64_t)heads * head_dim || table_stride < max_pages ||
      (num_pages > 1 && (k_page_stride < page_elems || v_page_stride < page_elems)))
    return MOE_ERR_INVALID_ARG;
  if (seqs == 0) return MOE_OK;
  if (!q || !lengths || !out || (max_pages > 0 && (!k_pages || !v_pages || !block_table || num_pages < 1)))
    return MOE_ERR_INVALID_ARG;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out) ||
      (q_stride & 7) || (k_page_stride & 7) || (v_page_stride & 7))
    return MOE_ERR_ALIGNMENT;
  const Shape sh = shape_of(seqs, kv_heads, heads / kv_heads, (int64_t)max_pages * page_size);
  // Chunk numbers are 32-bit on the device.
  if ((int64_t)max_pages * page_size > INT32_MAX || sh.units * sh.chunks > INT32_MAX)
    return MOE_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < workspace_floats(sh, head_dim) * sizeof(float))
    return MOE_ERR_WORKSPACE;
  if (!aligned16(workspace)) return MOE_ERR_ALIGNMENT;
  PagedArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.out = out;
  a.lengths = lengths;
  a.kv = KvPages{k_pages, v_pages, k_page_stride, v_page_stride, num_pages, block_table,
                 table_stride, seqs, max_pages, page_size, kv_heads};
  a.scale_log2 = scale * 1.4426950408889634f;
  a.group = heads / kv_heads;
  a.parts = sh.parts;
  a.whole = sh.whole;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* ws = static_cast<float*>(workspace);
  return dtype == MOE_DTYPE_F16 ? launch_typed<F16>(a, sh, head_dim, ws, s)
                                : launch_typed<BF16>(a, sh, head_dim, ws, s);
}
