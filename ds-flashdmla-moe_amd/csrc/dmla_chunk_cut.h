// How chunk attention's work is cut over its workgroups, and where the rows of a piece are cut for its careful passes.
//
// All of it is arithmetic on lengths, tables and latents that the threads of a workgroup do together.  Beside plain C++ it
// uses what dmla_common.h and dmla_pipe.h define and what a kernel has by itself (threadIdx, barriers, ballots): the
// file that includes this one brings them, and tests/test_chunk_cut.py runs this code on the CPU, a thread for a lane.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace dmla {
namespace {

constexpr int kPage = 64;
constexpr int kTile = 32;                                  // keys of a tile
constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 128;                                 // of a workgroup
constexpr int kNarrowRows = 32;                            // up to here the waves share the rows' scores

// Pointers say that they are to global memory: taken out of a copy of the arguments, the compiler would not know.
template <typename T>
using Global = DMLA_GLOBAL T*;

struct ChunkParams {
  Global<const bf16> q;
  Global<const char> kv;
  Global<const int32_t> block_table, seqlens;
  Global<const int32_t> cu;       // nullable: one query per sequence
  Global<bf16> o;
  Global<float> lse;              // nullable
  Global<float> part_o;           // [2 ranges, 128 rows, 512] normalised partial outputs
  Global<float> part_lse;         // [2 ranges, 128 rows], log2 units
  Global<i32x4> links;            // [ranges] (RangeLink)
  int64_t q_st, q_sh, kv_sp, kv_ss, bt_sb, o_st, o_sh;   // kv strides in bytes
  int T, B, H, num_pages, max_pages, causal, n_ranges, groups;
  FastDiv hdiv;          // division by H
  float scale_log2;
  float two_by_h, weight_scale;   // 2 / H, 2^-weight_shift
  int weight_shift;
};

// A sequence's queries: q0 .. q0 + n - 1, the newest of its len tokens.
struct Sequence {
  int q0, n, len;
};
__device__ __forceinline__ Sequence sequence(const ChunkParams& p, int b) {
  Sequence s;
  s.len = (int)min((int64_t)max(p.seqlens[b], 0), (int64_t)p.max_pages * kPage);
  if (p.cu == nullptr) {
    s.q0 = b;
    s.n = 1;
  } else {
    s.q0 = min(max(p.cu[b], 0), p.T);
    s.n = min(max(p.cu[b + 1], s.q0), p.T) - s.q0;
  }
  return s;
}

// Up to 128 rows of a sequence from row0 on, the key tiles [t0, t1) of them, and where their output goes: slot < 0 to o, else
// a part.
struct Piece {
  Sequence s;
  int b, row0, rows, t0, t1, slot;
};

// A piece runs once, against each row's largest score in the first tile.  Where scores have climbed more than kHeadroom
// above it, or an output is not a number or infinite, it runs the careful way: a row's reference is the largest score
// that was seen, and a row sees nothing of later tokens, as a probability of 0 times a latent that is not a number is
// none either.  So the rows are cut where a later row's token holds such a latent or begins a page outside the pool, and
// the rows before it run without it.  Both are rare, and the loop holds neither rescaling nor tests.
struct Pass {
  bool careful;
  int from, to;   // rows with a limit in [from, to) are written
};

// The next rows to run the careful way, from the limit `from` on: up to a later token whose latents are not all finite,
// or the first one of a page outside the pool.
__device__ __forceinline__ Pass careful_pass(const ChunkParams& p, const Piece& pc, DMLA_LDS int* flag, int from, int lim_last) {
  const int wave = uniform(threadIdx.x >> 6);
  int to = 0x7fffffff;
  for (int j = max(from + 1, 0) + wave; j <= min(lim_last, pc.t1 * kTile - 1); j += kWaves) {
    const int page = uniform(p.block_table[pc.b * p.bt_sb + j / kPage]);
    if (page < 0 || page >= p.num_pages) {   // page 0 stands in for it; its first token's row and all behind see it
      if (j % kPage != 0) continue;
      to = j;
      break;
    }
    const u32x4 v = *reinterpret_cast<Global<const u32x4>>(p.kv + page * p.kv_sp + j % kPage * p.kv_ss + 16 * fresh_lane_id());
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) odd = odd || (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
    if (__any(odd)) {
      to = j;
      break;
    }
  }
  __syncthreads();   // every wave has read from these words that a pass follows
  if (fresh_lane_id() == 0) flag[wave] = to;
  __syncthreads();
  to = uniform(min(min(flag[0], flag[1]), min(flag[2], flag[3])));
  __syncthreads();
  return Pass{true, from, to};
}

// ---- cutting the work ---------------------------------------------------------------------------------
// The row tiles (128 rows) of all sequences, in order, each with its key tiles behind some virtual ones (what starting
// and ending a piece costs), are cut into ranges of equal weight, one per workgroup: no list, no plan kernel, no order
// of workgroups.  Every workgroup works the cut out from the lengths.  A row tile that spans ranges leaves a part in
// each, merged by chunk_combine_kernel: range r writes the part that it begins with to slot 2 r (a row tile that an
// earlier range began) and the one that it ends with to slot 2 r + 1.
//
// Weights are estimates in closed form, in key tiles (one of a few rows takes as long as one of 128: 32 sequences x
// 16 heads, four of them with chunks of 460 tokens, 343 us, 506 when it weighed half).  The first n row tiles of a
// sequence whose first query is token `base` weigh A(n) = n (c + (base + 31) / 32) + 2 n (n + 1) / H (row tile i ends
// at token base + 128 (i + 1) / H, causal), where c is what a start and end cost; of more queries than tokens the first row
// tiles weigh c alone, and the growth starts behind them.  A range's end is the next one's start
// by the same arithmetic, so nothing is lost or done twice where they are off.  They are integers (of fp32 products,
// ascending in n whatever the rounding); where the host finds that they could pass 2^30, all are taken in units of
// 2^weight_shift.
// (c of 7 and the one more: four prompts of 300 to 1900 tokens x 128 heads 814 us; 863 with 5, 829 with 9.)
constexpr int kMaxRanges = 256;
constexpr int kCost = 7, kNarrowCost = 5;
constexpr int kMinWidth = 3;    // of a range
// Little work (a weight of kFine and less) is cut in row tiles of 32 rows: their queries and outputs take a
// quarter of the time, and there are four times as many to spread (one token x 128 heads over 5000 / 20000 tokens: 27 / 36
// us, 33 / 40 in row tiles of 128; over 40000, weight 1260, 50 and 45).
constexpr int kFine = 900;
constexpr int kRowsLog2 = 7, kNarrowLog2 = 5;
static_assert(1 << kRowsLog2 == kRows && 1 << kNarrowLog2 == kNarrowRows, "row tiles");
// Tiles: a cut this near to a row tile's end moves there, or a quarter of a range's width.  (512 queries x 128 heads over
// 32 pages each, two row tiles a range: 262 us, 288 with 8; 256 queries x 128 heads over 8192 tokens 514 us, 501 with 8.)
constexpr int kSnap = 12;

struct Place {   // in the row tiles and key tiles of all sequences
  int b, rt, t;
};
struct Window {   // the sequences of 256 at a time, and what the threads share
  int q0[kThreads], n[kThreads], len[kThreads];
  int tmp[kWaves];
  Place at, end;        // where the next piece begins, and the range's end
  int first;            // sequence of the window
  int rows_log2;        // rows of a row tile
  i32x4 piece[2][3];   // q0, row0, rows, n; len, b, t0, t1; slot: this one and the next
};

// (Rows of a row tile: 2^rows_log2.)
__device__ __forceinline__ int row_tiles(const ChunkParams& p, const Sequence& s, int rows_log2) { return (s.n * p.H + (1 << rows_log2) - 1) >> rows_log2; }
__device__ __forceinline__ int key_tiles(const ChunkParams& p, const Sequence& s, int rt, int rows_log2) {
  const int last = fast_div(min((rt + 1) << rows_log2, s.n * p.H) - 1, p.hdiv);
  const int end = p.causal ? s.len - s.n + last + 1 : s.len;
  return (max(end, 0) + kTile - 1) / kTile;
}
struct Weights {
  int cost, none;       // none: row tiles before the first that has a token
  float base, growth;   // of a row tile, and how much more each one behind those weighs
};
__device__ __forceinline__ Weights weights(const ChunkParams& p, const Sequence& s, int rows_log2) {
  const bool few = s.n * p.H <= kNarrowRows || rows_log2 == kNarrowLog2;
  Weights w = {few ? kNarrowCost : kCost, 0, 0.f, 0.f};
  const int tiles = ((p.causal ? max(s.len - s.n, 0) : s.len) + kTile - 1) / kTile;
  w.base = (float)(w.cost + tiles);
  w.none = p.causal ? max(s.n - s.len, 0) * p.H >> rows_log2 : 0;
  w.growth = !p.causal ? 0.f : rows_log2 == kNarrowLog2 ? 0.25f * p.two_by_h : p.two_by_h;
  return w;
}
// A(n), one more for each row tile: none is without a weight, or no range would hold it.
__device__ __forceinline__ int weight(const ChunkParams& p, const Weights& w, int n) {
  const int m = max(n - w.none, 0);
  return n + (int)(((float)m * (w.base + w.growth * (float)(m + 1)) + (float)(n - m) * w.base) * p.weight_scale);
}
// The place at weight y of sequence b.
__device__ __forceinline__ Place place_of(const ChunkParams& p, int b, const Sequence& s, int y, int width, int rows_log2) {
  const Weights w = weights(p, s, rows_log2);
  int lo = 0, hi = row_tiles(p, s, rows_log2) - 1;   // the last row tile that begins at or before y
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (weight(p, w, mid) <= y) lo = mid; else hi = mid - 1;
  }
  const int nt = key_tiles(p, s, lo, rows_log2), snap = min(kSnap, width >> 2 << p.weight_shift);
  const int64_t in = (int64_t)(y - weight(p, w, lo)) << p.weight_shift;
  int t = (int)min((int64_t)nt, max((int64_t)0, in - w.cost));
  if (t <= snap) t = 0;
  if (t > 0 && nt - t <= snap) return Place{b, lo + 1, 0};
  return Place{b, lo, t};
}

// What the combine reads of a range: x the rows of a row tile that begins in it and goes on in the next (0: none), their
// packed query q0 and first row, w how its first part goes on: 1 it ends here, 2 it does not.
typedef i32x4 RangeLink;

// The window from sequence b0 on; this thread's sequence.
__device__ __forceinline__ Sequence load_window(const ChunkParams& p, DMLA_LDS Window* win, int b0) {
  const int tid = threadIdx.x;
  __syncthreads();   // the window is read
  Sequence s = {0, 0, 0};
  if (b0 + tid < p.B) s = sequence(p, b0 + tid);
  win->q0[tid] = s.q0;
  win->n[tid] = s.n;
  win->len[tid] = s.len;
  if (tid == 0) win->first = b0;
  return s;
}
__device__ __forceinline__ Sequence known(const DMLA_LDS Window* win, int i) {
  return Sequence{uniform(win->q0[i]), uniform(win->n[i]), uniform(win->len[i])};
}

// The range's end and its first place; whether it has any.
__device__ __forceinline__ bool cut(const ChunkParams& p, DMLA_LDS Window* win, int range) {
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  // Inclusive sum over the threads and their total.
  auto scan = [&](int v, int& sum) {
    v = lane_scan(v);
    __syncthreads();   // every wave has read the sums of a scan before
    if (lane == 63) win->tmp[wave] = v;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) v += win->tmp[w];
      sum += win->tmp[w];
    }
    return v;
  };
  int total = 0, upto = 0, mine = 0, sum = 0, rows_log2 = kRowsLog2;
  Sequence s = {0, 0, 0};
  for (int b0 = 0; b0 < p.B; b0 += kThreads) {
    s = load_window(p, win, b0);
    mine = weight(p, weights(p, s, rows_log2), row_tiles(p, s, rows_log2));
    upto = scan(mine, sum);
    total += sum;
  }
  if (total <= kFine && p.B <= kThreads && p.weight_shift == 0) {
    rows_log2 = kNarrowLog2;
    mine = weight(p, weights(p, s, rows_log2), row_tiles(p, s, rows_log2));
    upto = scan(mine, total);
  }
  const int n = max(1, min(p.n_ranges, total / max(1, kMinWidth >> p.weight_shift)));
  const int width = total / n, rest = total - width * n;
  const int x0 = range * width + range * rest / n, x1 = (range + 1) * width + (range + 1) * rest / n;
  if (tid == 0) {
    p.links[range] = i32x4{0, 0, 0, 0};
    // (Starts that do not ascend can add up to anything; then there may be no place, and nothing to do.)
    win->at.b = win->at.rt = win->at.t = 0;
    win->end.b = win->end.rt = win->end.t = 0;
    win->rows_log2 = rows_log2;
  }
  if (range >= n || x0 >= x1) return false;
  __syncthreads();
  // The places of x0 and x1, by the threads whose sequences hold them; x1 at the end of one is that end.
  for (int b0 = 0, before = 0; b0 < p.B && before < x1; b0 += kThreads, before += sum) {
    if (p.B > kThreads) {
      s = load_window(p, win, b0);
      mine = weight(p, weights(p, s, rows_log2), row_tiles(p, s, rows_log2));
      upto = scan(mine, sum);
    }
    const int lo = before + upto - mine, hi = before + upto;
    auto put = [](DMLA_LDS Place* to, const Place& v) {
      to->b = v.b;
      to->rt = v.rt;
      to->t = v.t;
    };
    if (lo <= x0 && x0 < hi) put(&win->at, place_of(p, b0 + tid, s, x0 - lo, width, rows_log2));
    if (lo < x1 && x1 <= hi) put(&win->end, x1 == hi ? Place{b0 + tid, row_tiles(p, s, rows_log2), 0} : place_of(p, b0 + tid, s, x1 - lo, width, rows_log2));
  }
  __syncthreads();
  const int b = uniform(win->at.b), first = uniform(win->first);
  if (b < first || b >= first + kThreads) {
    load_window(p, win, b);
    __syncthreads();
  }
  return true;
}

// The next piece of the range (rows 0: none).  What it goes by is in LDS and not in registers: run_piece has none to
// spare, and a value reloaded from scratch memory would wait for every copy and store in flight.
__device__ __forceinline__ void next_piece(const ChunkParams& p, DMLA_LDS Window* win, DMLA_LDS i32x4* to, int range) {
  const int tid = threadIdx.x, lane = tid & 63;
  Place at = {uniform(win->at.b), uniform(win->at.rt), uniform(win->at.t)};
  const int rows_log2 = uniform(win->rows_log2);
  const Place end = {uniform(win->end.b), uniform(win->end.rt), uniform(win->end.t)};
  Sequence s;
  for (;;) {
    if (!(at.b < end.b || (at.b == end.b && (at.rt < end.rt || (at.rt == end.rt && at.t < end.t))))) {
      if (tid == 0) to[0] = i32x4{0, 0, 0, 0};
      return;
    }
    int first = uniform(win->first);
    s = known(win, at.b - first);
    if (at.rt < row_tiles(p, s, rows_log2)) break;
    // The next sequence with queries (there is one, end.b at the latest): 256 looked at together.
    int b = at.b + 1;
    for (;; b = first + kThreads) {
      if (b >= first + kThreads) {
        load_window(p, win, b);
        __syncthreads();
        first = b;
      }
      int found = kThreads;
      for (int i0 = (b - first) & ~63; i0 < kThreads; i0 += 64) {
        const unsigned long long m = __ballot(i0 + lane >= b - first && win->n[i0 + lane] > 0);
        if (m != 0) {
          found = i0 + __builtin_ctzll(m);
          break;
        }
      }
      if (found < kThreads) {
        b = first + found;
        break;
      }
    }
    at = Place{uniform(b), 0, 0};
  }
  const int row0 = at.rt << rows_log2, rows = min(s.n * p.H - row0, 1 << rows_log2);
  const bool whole = !(at.b == end.b && at.rt == end.rt);   // to its end
  __syncthreads();   // the place is read
  if (tid == 0) {
    to[0] = i32x4{s.q0, row0, rows, s.n};
    to[1] = i32x4{s.len, at.b, at.t, whole ? key_tiles(p, s, at.rt, rows_log2) : end.t};
    to[2] = i32x4{at.t > 0 ? 2 * range : whole ? -1 : 2 * range + 1, 0, 0, 0};
    Global<RangeLink> link = p.links + range;
    if (at.t > 0) {
      (*link)[3] = whole ? 1 : 2;
    } else if (!whole) {
      (*link)[0] = rows;
      (*link)[1] = s.q0;
      (*link)[2] = row0;
    }
    win->at.b = at.b;
    win->at.rt = whole ? at.rt + 1 : at.rt;
    win->at.t = whole ? 0 : end.t;
  }
}

// At least the weight that the kernel adds up, in row tiles of `rows` rows (but for two a row tile, from roundings up): a
// row tile has no more keys than the table, however many queries have no token.
inline int64_t chunk_weight(int64_t T, int64_t B, int64_t H, int64_t max_pages, int64_t rows) {
  const int64_t tiles = T * H / rows + std::min(B, T);
  return tiles * (kCost + 3 + max_pages * (kPage / kTile));
}
inline int chunk_weight_shift(int64_t T, int64_t B, int64_t H, int64_t max_pages) {
  int shift = 0;
  while (chunk_weight(T, B, H, max_pages, kRows) >> shift > (int64_t)1 << 30) ++shift;
  return shift;
}

}  // namespace
}  // namespace dmla
