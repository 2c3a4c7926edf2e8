// Eviction from the paged latent cache by accumulated attention weight.
//
// A sequence of N tokens above the budget K keeps its first S tokens (sinks), its newest R, and of the
// middle ones the K - S - R with the largest accounts (the lower index first among equals; NaN counts as
// the largest).  Attention does not depend on the order of the rows, since a row carries its position,
// so the pages are compacted with as few copies as possible:
//   * sinks, and kept middle rows below K - R, stay where they are;
//   * the other kept middle rows, in order, fill the freed places below K - R, in order;
//   * the newest R rows move down to [K - R, K), in order.
// Cutting 4096 + 64 tokens back to 4096 with R = 256 then moves at most 64 + 256 rows, where closing every
// gap would move nearly all.  No reference counterpart.
//
// The selection is a radix select of the accounts' keys (digits of 11, 11 and 10 bits) and a pass in index
// order that lists the freed places and the rows that fill them.
//   * Up to kOneTokens tokens one workgroup per sequence holds the accounts in registers and does it all in one
//     launch.  Whole calls on 4-bit pages, cut to 4096 tokens: 64 sequences of 8192 tokens 36 us (chunked as below
//     80), one of 16384 25 us (38).
//   * Longer block tables: up to kMaxChunks workgroups per sequence, a launch per digit and one for the lists.  A
//     chunk's counts go through the workspace and every workgroup adds up all chunks', so nothing is cleared
//     beforehand and nothing depends on the order of atomics.  No chunk straddles the end of the kept low
//     places: how many places a chunk frees, or how many rows it moves, follows from its counts alone.
// Then come the middle moves, together with a copy of the newest rows into the workspace where their old and new
// places overlap (N - K < R), and the newest rows' move.  A middle move's destination is a freed place and its
// source lies at or past K - R, so those moves depend on nothing; the newest rows overwrite such sources and
// therefore come last.
// Bound: the moved rows' bytes, twice, and where few rows move the launches' latency.  64 sequences of 4096 to 8192
// bf16 tokens cut to 4096: 66 us (selection 12, moves 41 and 9; 229 MB, 3.5 TB/s); one of 131072 cut
// to 32768: 53 us, of which the four selection launches take 38.
#include <algorithm>

#include "dmla_common.h"
#include "dmla_host.h"

namespace dmla {
namespace {

constexpr int kPage = 64;
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kDigitBits = 11, kBins = 1 << kDigitBits;
constexpr int kOneTokens = 16 * kSelThreads;   // tokens that a workgroup holds in registers
constexpr int kMaxChunks = 32;
constexpr int kPiece = 8;          // tokens of a thread at a time
constexpr int kMoveRows = 32;      // rows that a workgroup moves at a time
constexpr int kMoveBatch = 5;      // 16-byte pieces of a thread in flight (32 bf16 rows are nine for each thread)

struct EvictArgs {
  char* pool;
  const int32_t* block_table;
  const int32_t* seqlens;
  const float* mass;
  int32_t* new_lens;
  int32_t* src;
  float* mass_out;
  int32_t* bad;          // nullable
  int64_t kv_sp, kv_ss;  // bytes
  int64_t bt_sb, m_sb, mo_sb, src_sb;
  int B, mass_len, num_pages, max_pages, width;   // width: entries of a row of src
  int budget, recent, sink;
  int row_chunks;        // 16-byte pieces of a row
  int32_t* info;         // [B][2]: tokens cut from the sequence (0: untouched), middle rows to move
  int32_t* free_at;      // [B][budget - recent - sink] freed places, and the rows that fill them
  int32_t* late_at;
  char* stage;           // [B][recent] rows
  int chunks;            // workgroups of a sequence, long tables only, as the next three
  int32_t* counts;       // [2][B][chunks][kBins]
  int32_t* above;        // [B][chunks]: tokens of a chunk whose key lies above the digits picked so far
  int32_t* sel;          // [2][B][2]: those digits, and how many of the tokens that share them are kept
  FastDiv per_row;       // division by row_chunks
};

// An integer that orders like the account: larger is better, -0 equals 0, NaN above everything.
__device__ __forceinline__ unsigned rank_key(float f) {
  unsigned u = __float_as_uint(f);
  if (f != f) return 0xffffffffu;
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix of v over the workgroup; total gets the sum.  tmp: kSelWaves ints.
__device__ __forceinline__ int scan_exclusive(int v, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = lane_scan(v);
  __syncthreads();   // tmp is free
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    const int t = tmp[w];
    before += w < wave ? t : 0;
    sum += t;
  }
  total = sum;
  return before + x - v;
}

struct Shared {
  int hist[kBins];
  int tmp[kSelWaves];
  int pick[2];                     // the digit that holds the last kept key, and how many keys lie above it
  int kept[kMaxChunks], equal[kMaxChunks];
};

// A sequence's cut: N tokens down to the budget.
struct Cut {
  int n, lo, hi, low_end, want;   // the middle tokens [lo, hi), and the places [lo, low_end) of the kept ones
};
__device__ __forceinline__ Cut cut_of(const EvictArgs& a, int b) {
  Cut c;
  c.n = min(max(a.seqlens[b], 0), a.max_pages * kPage);
  c.lo = a.sink;
  c.hi = c.n - a.recent;
  c.low_end = a.budget - a.recent;
  c.want = c.low_end - c.lo;
  return c;
}

// Whether the sequence is cut: it is longer than the budget and its pages are all in the pool.
__device__ __forceinline__ bool is_cut(const EvictArgs& a, int b, const Cut& c) {
  int bad = 0;
  if (c.n > a.budget)
    for (int i = threadIdx.x; i < (c.n + kPage - 1) / kPage; i += kSelThreads) {
      const int page = a.block_table[b * a.bt_sb + i];
      bad |= page < 0 || page >= a.num_pages;
    }
  bad = __syncthreads_or(bad);
  if (bad && a.bad != nullptr && threadIdx.x == 0) a.bad[0] = 1;
  return c.n > a.budget && !bad;
}

// The outputs of a sequence that stays as it is, by the threads first, first + step, ...
__device__ __forceinline__ void leave(const EvictArgs& a, int b, const Cut& c, int first, int step) {
  if (first == 0) {
    a.new_lens[b] = c.n;
    a.info[2 * b] = 0;
    a.info[2 * b + 1] = 0;
  }
  for (int i = first; i < a.width; i += step) a.src[b * a.src_sb + i] = i < c.n ? i : -1;
  for (int i = first; i < a.mass_len; i += step) a.mass_out[b * a.mo_sb + i] = i < c.n ? a.mass[b * a.m_sb + i] : 0.f;
}

// Digits: bits 21.., 10.. and 0.. of the key.
__device__ __forceinline__ int digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__device__ __forceinline__ int digit_bins(int d) { return d == 2 ? 1 << 10 : kBins; }

// Thread t brings the counts of the bins top = bins - 1 - 2 t and top - 1; the digit whose bin holds the left-th key
// from above becomes part of prefix, and left counts within it.  Returns the digit.
__device__ __forceinline__ int pick_digit(Shared& sh, int d, int top, int c0, int c1, unsigned& prefix, int& left) {
  int total;
  const int above = scan_exclusive(c0 + c1, sh.tmp, total);
  if (above < left && left <= above + c0) {
    sh.pick[0] = top;
    sh.pick[1] = above;
  } else if (above + c0 < left && left <= above + c0 + c1) {
    sh.pick[0] = top - 1;
    sh.pick[1] = above + c0;
  }
  __syncthreads();
  const int digit = sh.pick[0];
  prefix |= (unsigned)digit << digit_shift(d);
  left -= sh.pick[1];
  return digit;
}

// Exclusive prefix, over the waves, of a count that is the same in all lanes of a wave; total gets the sum.
__device__ __forceinline__ int scan_waves(int v, int* tmp, int& total) {
  const int wave = uniform(threadIdx.x >> 6);
  __syncthreads();   // tmp is free
  if ((threadIdx.x & 63) == 0) tmp[wave] = v;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    const int t = uniform(tmp[w]);
    before += w < wave ? t : 0;
    sum += t;
  }
  total = sum;
  return before;
}

// Where the lists and the count of equal keys stand.
struct Seen {
  int equal, freed, late;
};

// A thread's kJ tokens: a wave holds 64 kJ consecutive ones, 64 at a time, so that ranks within it are bit counts.
template <int kJ>
__device__ __forceinline__ int token_of(int i0, int j) {
  return i0 + (int)(threadIdx.x >> 6) * 64 * kJ + 64 * j + (int)(threadIdx.x & 63);
}

// The accounts of a thread's tokens that lie in [from, to), and their bits.
template <int kJ>
__device__ __forceinline__ unsigned load_accounts(const float* mass, int i0, int from, int to, float (&v)[kJ]) {
  unsigned in = 0;
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const int i = token_of<kJ>(i0, j);
    const bool is = i >= from && i < to;
    v[j] = is ? mass[i] : 0.f;
    in |= is ? 1u << j : 0u;
  }
  return in;
}

// The middle tokens from i0 on (those with their bit of in set), whose accounts are v: which of them stay, which
// places below low_end are freed, which rows fill them.
template <int kJ>
__device__ __forceinline__ void place(const EvictArgs& a, int b, const Cut& c, Shared& sh, const float (&v)[kJ], unsigned in,
                                      int i0, unsigned key, int left, Seen& seen) {
  auto rank_in = [](unsigned long long m) { return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, 0)); };
  unsigned kept = 0, equal = 0;   // a bit per j
  int n_equal = 0;                // of the wave
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const unsigned k = rank_key(v[j]), bit = in & 1u << j;
    kept |= k > key ? bit : 0u;
    equal |= k == key ? bit : 0u;
    n_equal += __popcll(__ballot(equal >> j & 1));
  }
  int sum;
  int rank0 = seen.equal + scan_waves(n_equal, sh.tmp, sum);
  seen.equal += sum;
  const int top = c.low_end - token_of<kJ>(i0, 0);   // tokens with 64 j < top lie below low_end
  unsigned below = 0;
  int counts = 0;   // of the wave: freed places, and rows to move in the upper half; 64 kJ kSelWaves fit 16 bits
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const unsigned bit = 1u << j;
    const unsigned long long m = __ballot(equal >> j & 1);
    kept |= rank0 + rank_in(m) < left ? equal & bit : 0u;
    rank0 += __popcll(m);
    below |= 64 * j < top ? bit : 0u;
    counts += __popcll(__ballot((in & below & ~kept) >> j & 1)) | __popcll(__ballot((kept & ~below) >> j & 1)) << 16;
  }
  const unsigned freed = in & below & ~kept, late = kept & ~below, stay = kept & below;
  const int before = scan_waves(counts, sh.tmp, sum);
  int32_t* free_at = a.free_at + (int64_t)b * c.want + seen.freed + (before & 0xffff);
  int32_t* late_at = a.late_at + (int64_t)b * c.want + seen.late + (before >> 16);
  int32_t* src = a.src + b * a.src_sb;
  float* out = a.mass_out + b * a.mo_sb;
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const int i = token_of<kJ>(i0, j);
    const unsigned long long f = __ballot(freed >> j & 1), l = __ballot(late >> j & 1);
    if (freed >> j & 1) free_at[rank_in(f)] = i;
    if (late >> j & 1) late_at[rank_in(l)] = i;
    if (stay >> j & 1) {
      src[i] = i;
      out[i] = v[j];
    }
    free_at += __popcll(f);
    late_at += __popcll(l);
  }
  seen.freed += sum & 0xffff;
  seen.late += sum >> 16;
}

template <int kJ>
__device__ __forceinline__ void count_digit(int* hist, int d, unsigned prefix, const float (&v)[kJ], unsigned in) {
  const unsigned mask = d == 0 ? 0u : ~0u << digit_shift(d - 1);
#pragma unroll
  for (int j = 0; j < kJ; ++j) {
    const unsigned key = rank_key(v[j]);
    if ((in >> j & 1) && (key & mask) == prefix) atomicAdd(&hist[(key >> digit_shift(d)) & (digit_bins(d) - 1)], 1);
  }
}

// One workgroup per sequence, tables of up to kJ tokens a thread.
template <int kJ>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x;
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const Cut c = cut_of(a, b);
    float v[kJ];   // read beside the check of the pages
    const unsigned in = load_accounts(a.mass + b * a.m_sb, 0, c.lo, c.hi, v);
    if (!is_cut(a, b, c)) {
      leave(a, b, c, tid, kSelThreads);
      continue;
    }
    unsigned prefix = 0;
    int left = c.want;   // how many are still to be taken from the tokens whose key matches prefix
    Seen seen = {0, 0, 0};
    if (c.want > 0) {
      for (int d = 0; d < 3; ++d) {
        const int bins = digit_bins(d);
        for (int i = tid; i < bins; i += kSelThreads) sh.hist[i] = 0;
        __syncthreads();
        count_digit(sh.hist, d, prefix, v, in);
        __syncthreads();
        const int top = bins - 1 - 2 * tid;
        pick_digit(sh, d, top, top >= 0 ? sh.hist[top] : 0, top >= 1 ? sh.hist[top - 1] : 0, prefix, left);
      }
      place(a, b, c, sh, v, in, 0, prefix, left, seen);
    }
    if (tid == 0) {
      a.new_lens[b] = a.budget;
      a.info[2 * b] = c.n - a.budget;
      a.info[2 * b + 1] = seen.late;
    }
  }
}

// ---- long tables ----
// Chunks of a cut sequence: first those of [lo, low_end), then those of [low_end, hi).
struct Chunks {
  int span, n_low, n;
  __device__ __forceinline__ Chunks(const Cut& c, int most) {
    const int each = (c.hi - c.lo + most - 3) / (most - 2);   // the two parts' last chunks may be short
    span = max(1, (each + kSelThreads - 1) / kSelThreads) * kSelThreads;
    n_low = (c.want + span - 1) / span;
    n = n_low + (c.hi - c.low_end + span - 1) / span;
  }
  __device__ __forceinline__ int from(const Cut& c, int k) const { return k < n_low ? c.lo + k * span : c.low_end + (k - n_low) * span; }
  __device__ __forceinline__ int to(const Cut& c, int k) const { return min(from(c, k) + span, k < n_low ? c.low_end : c.hi); }
};

// Launch d = 0 .. 2 counts digit d of every chunk, d = 3 writes the lists; each first picks digit d - 1.  Grid: x
// over the chunks, y over sequences.
template <int kD>
__global__ void __launch_bounds__(kSelThreads) evict_chunk_kernel(EvictArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, k = blockIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  constexpr int kBatch = 8;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const Cut c = cut_of(a, b);
    if constexpr (kD == 0) {
      const bool cut = is_cut(a, b, c);
      if (!cut) {
        leave(a, b, c, k * kSelThreads + tid, a.chunks * kSelThreads);
        continue;
      }
      if (k == 0 && tid == 0) a.info[2 * b] = c.n - a.budget;
    } else {
      if (a.info[2 * b] == 0) continue;
    }
    const Chunks ch(c, a.chunks);
    auto counts_of = [&](int d, int chunk) { return a.counts + (((int64_t)(d & 1) * a.B + b) * a.chunks + chunk) * kBins; };
    auto sel_of = [&](int d) { return a.sel + ((int64_t)(d & 1) * a.B + b) * 2; };   // of launch d
    unsigned prefix = kD > 1 ? (unsigned)sel_of(kD - 1)[0] : 0u;
    int left = kD > 1 ? sel_of(kD - 1)[1] : c.want;
    // What does not depend on the pick is on its way beside it: the chunk's first accounts, and in the last launch
    // the counts of the chunks w and w + 16 by wave w, and in lane i the tokens of chunk i above the earlier digits.
    const float* mass = a.mass + b * a.m_sb;
    const bool work = k < ch.n && c.want > 0;
    const int from = work ? ch.from(c, k) : 0, to = work ? ch.to(c, k) : 0;
    float v[kPiece];
    unsigned in = load_accounts(mass, from, from, to, v);
    constexpr int kEach = kMaxChunks / kSelWaves, kCounts = (1 << 10) / 64;
    int counts[kD == 3 ? kEach : 1][kCounts];
    int above = 0;
    if constexpr (kD == 3) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
#pragma unroll
        for (int x = 0; x < kCounts; ++x) counts[i][x] = counts_of(2, min(wave + kSelWaves * i, ch.n - 1))[64 * x + lane];
      above = a.above[b * a.chunks + min(lane, ch.n - 1)];
    }
    if (kD > 0 && c.want > 0) {
      constexpr int d = kD - 1;
      const int top = digit_bins(d) - 1 - 2 * tid;
      int c0 = 0, c1 = 0, own = 0, own0 = 0, own1 = 0;
      if (top > 0) {
        for (int i0 = 0; i0 < ch.n; i0 += kBatch) {
          int2 x[kBatch];   // on their way together
#pragma unroll
          for (int i = 0; i < kBatch; ++i)
            x[i] = *reinterpret_cast<const int2*>(counts_of(d, min(i0 + i, ch.n - 1)) + top - 1);
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const bool is = i0 + i < ch.n, mine = i0 + i == k;
            c1 += is ? x[i].x : 0;
            c0 += is ? x[i].y : 0;
            own1 = mine ? x[i].x : own1;
            own0 = mine ? x[i].y : own0;
          }
        }
      }
      const int digit = pick_digit(sh, d, top, c0, c1, prefix, left);
      if constexpr (kD < 3) {   // of this chunk, the tokens above the digit
        scan_exclusive((top > digit ? own0 : 0) + (top - 1 > digit ? own1 : 0), sh.tmp, own);
        if (tid == 0 && k < ch.n) a.above[b * a.chunks + k] = own + (kD > 1 ? a.above[b * a.chunks + k] : 0);
        if (tid == 0 && k == 0) {
          sel_of(kD)[0] = (int)prefix;
          sel_of(kD)[1] = left;
        }
      } else {   // the tokens of a chunk above the digit, and those equal to it
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          int sum = 0, equal = 0;
#pragma unroll
          for (int x = 0; x < kCounts; ++x) {
            sum += 64 * x + lane > digit ? counts[i][x] : 0;
            equal += 64 * x + lane == digit ? counts[i][x] : 0;
          }
          sum = lane_scan(sum);
          equal = lane_scan(equal);
          if (lane == 63) {
            sh.kept[wave + kSelWaves * i] = sum;
            sh.equal[wave + kSelWaves * i] = equal;
          }
        }
      }
    }
    if constexpr (kD < 3) {
      if (work) {
        for (int i = tid; i < digit_bins(kD); i += kSelThreads) sh.hist[i] = 0;
        __syncthreads();
        count_digit(sh.hist, kD, prefix, v, in);
        for (int i0 = from + kPiece * kSelThreads; i0 < to; i0 += kPiece * kSelThreads) {
          in = load_accounts(mass, i0, from, to, v);
          count_digit(sh.hist, kD, prefix, v, in);
        }
        __syncthreads();
        for (int i = tid; i < digit_bins(kD); i += kSelThreads) counts_of(kD, k)[i] = sh.hist[i];
      }
      __syncthreads();   // hist is free for the next sequence
    } else {
      __syncthreads();
      Seen seen = {0, 0, 0};
      int late = 0;
      if (c.want > 0) {
        // lane i: chunk i's kept tokens, the places it frees and the rows it moves, and their sums over the chunks before
        static_assert(kMaxChunks <= 64, "a lane per chunk");
        const bool is = lane < ch.n;
        const int equal = is ? sh.equal[lane] : 0, equal_to = lane_scan(equal);
        const int kept = (is ? above + sh.kept[lane] : 0) + min(max(left - (equal_to - equal), 0), equal);
        const int freed = is && lane < ch.n_low ? ch.to(c, lane) - ch.from(c, lane) - kept : 0;
        const int moved = is && lane >= ch.n_low ? kept : 0;
        const int freed_to = lane_scan(freed), moved_to = lane_scan(moved);
        late = __builtin_amdgcn_readlane(moved_to, 63);
        seen.equal = __builtin_amdgcn_readlane(equal_to - equal, k);
        seen.freed = __builtin_amdgcn_readlane(freed_to - freed, k);
        seen.late = __builtin_amdgcn_readlane(moved_to - moved, k);
        if (work) {
          place(a, b, c, sh, v, in, from, prefix, left, seen);
          for (int i0 = from + kPiece * kSelThreads; i0 < to; i0 += kPiece * kSelThreads) {
            in = load_accounts(mass, i0, from, to, v);
            place(a, b, c, sh, v, in, i0, prefix, left, seen);
          }
        }
      }
      if (k == 0 && tid == 0) {
        a.new_lens[b] = a.budget;
        a.info[2 * b + 1] = late;
      }
      __syncthreads();   // kept and equal are free for the next sequence
    }
  }
}

// The outputs of a cut sequence of n tokens outside the middle, by the threads first, first + step, ...
__device__ __forceinline__ void put_ends(const EvictArgs& a, int b, int n, int first, int step) {
  const int lo = a.sink, hi = n - a.recent, low_end = a.budget - a.recent;
  int32_t* src = a.src + b * a.src_sb;
  float* out = a.mass_out + b * a.mo_sb;
  const float* mass = a.mass + b * a.m_sb;
  for (int i = first; i < lo; i += step) {
    src[i] = i;
    out[i] = mass[i];
  }
  for (int i = first; i < a.recent; i += step) {
    src[low_end + i] = hi + i;
    out[low_end + i] = mass[hi + i];
  }
  for (int i = a.budget + first; i < a.mass_len; i += step) out[i] = 0.f;
}

// Phase 0: the outputs outside the middle; the middle moves, with the outputs of the places they fill, and the newest rows into the workspace where
// they overlap their new places.  Phase 1: the newest rows to their places.  A workgroup takes kMoveRows rows at a
// time: their addresses first, then their 16-byte pieces.  Grid: x over the rows of a sequence, y over sequences.
template <int kPhase>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a) {
  __shared__ const DMLA_GLOBAL char* from[kMoveRows];
  __shared__ DMLA_GLOBAL char* to[kMoveRows];
  const int want = a.budget - a.recent - a.sink;
  auto row_at = [&](int b, int pos) {
    return a.pool + a.block_table[b * a.bt_sb + pos / kPage] * a.kv_sp + (int64_t)(pos % kPage) * a.kv_ss;
  };
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int cut = a.info[2 * b], moves = a.info[2 * b + 1];
    if (cut == 0) continue;
    const int low_end = a.budget - a.recent;
    const bool staged = cut < a.recent;
    const int64_t row_bytes = (int64_t)a.row_chunks * 16;
    char* stage = a.stage + (int64_t)b * a.recent * row_bytes;
    const int rows = kPhase == 0 ? moves + (staged ? a.recent : 0) : a.recent;
    if constexpr (kPhase == 0) put_ends(a, b, a.budget + cut, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
    for (int r0 = blockIdx.x * kMoveRows; r0 < rows; r0 += gridDim.x * kMoveRows) {
      const int n = min(kMoveRows, rows - r0);
      __syncthreads();   // the addresses before have been read
      if ((int)threadIdx.x < n) {
        const int r = r0 + threadIdx.x;
        const char* f;
        char* t;
        if (kPhase == 0 && r < moves) {
          const int late = a.late_at[(int64_t)b * want + r], freed = a.free_at[(int64_t)b * want + r];
          f = row_at(b, late);
          t = row_at(b, freed);
          a.src[b * a.src_sb + freed] = late;
          a.mass_out[b * a.mo_sb + freed] = a.mass[b * a.m_sb + late];
        } else if (kPhase == 0) {
          f = row_at(b, low_end + cut + (r - moves));
          t = stage + (r - moves) * row_bytes;
        } else {
          f = staged ? stage + r * row_bytes : row_at(b, low_end + cut + r);
          t = row_at(b, low_end + r);
        }
        from[threadIdx.x] = (const DMLA_GLOBAL char*)f;
        to[threadIdx.x] = (DMLA_GLOBAL char*)t;
      }
      __syncthreads();
      const int pieces = n * a.row_chunks;
      for (int q0 = threadIdx.x; q0 < pieces; q0 += 256 * kMoveBatch) {
        i32x4 v[kMoveBatch];
        DMLA_GLOBAL i32x4* at[kMoveBatch];
#pragma unroll
        for (int u = 0; u < kMoveBatch; ++u) {
          const int q = min(q0 + 256 * u, pieces - 1), r = fast_div(q, a.per_row), c = 16 * (q - r * a.row_chunks);
          at[u] = (DMLA_GLOBAL i32x4*)(to[r] + c);
          v[u] = *(const DMLA_GLOBAL i32x4*)(from[r] + c);
        }
#pragma unroll
        for (int u = 0; u < kMoveBatch; ++u)
          if (q0 + 256 * u < pieces) __builtin_nontemporal_store(v[u], at[u]);   // 64 sequences 66 us, plain stores 73
      }
    }
  }
}

struct EvictLayout {
  int64_t info, free_at, late_at, stage, counts, above, sel, total;   // byte offsets, multiples of 16
};
// Workgroups of a sequence: every one adds up the counts of all, so together no more than twice the chip's
// (64 sequences x 32 took 280 us where one workgroup each took 37), and 4 at least, two for either part.
int64_t evict_chunks(int64_t B) { return std::min<int64_t>(kMaxChunks, std::max<int64_t>(4, 2 * device_cu_count() / B)); }
EvictLayout evict_layout(int64_t B, int64_t cap, int64_t budget, int64_t recent, int64_t sink, int64_t row_bytes) {
  int64_t at = 0;
  auto part = [&](int64_t bytes) {
    const int64_t from = at;
    at += (bytes + 15) / 16 * 16;
    return from;
  };
  const int64_t want = budget - recent - sink, chunked = cap > kOneTokens ? B * evict_chunks(B) : 0;
  EvictLayout l;
  l.info = part(B * 8);
  l.free_at = part(B * want * 4);
  l.late_at = part(B * want * 4);
  l.stage = part(B * recent * row_bytes);
  l.counts = part(chunked * 2 * kBins * 4);
  l.above = part(chunked * 4);
  l.sel = part(chunked > 0 ? B * 16 : 0);
  l.total = at;
  return l;
}
// The layout of a call; a budget that covers the block table cuts nothing and keeps no lists.
EvictLayout evict_layout_of(int64_t B, int64_t row_bytes, int64_t max_pages, int64_t budget, int64_t recent, int64_t sink) {
  const int64_t cap = max_pages * kPage;
  return budget >= cap ? evict_layout(B, cap, 0, 0, 0, row_bytes) : evict_layout(B, cap, budget, recent, sink, row_bytes);
}

}  // namespace
}  // namespace dmla

using namespace dmla;

static bool evict_sizes_ok(int64_t B, int64_t row_bytes, int64_t max_pages, int64_t budget, int64_t recent, int64_t sink) {
  return B > 0 && B <= ((int64_t)1 << 20) && row_bytes > 0 && row_bytes % 16 == 0 && row_bytes <= 65536 && max_pages > 0 &&
         max_pages <= ((int64_t)1 << 20) && budget > 0 && recent >= 0 && sink >= 0 && recent <= budget && sink <= budget - recent;
}

extern "C" int64_t dmla_kv_evict_workspace_bytes(int64_t B, int64_t row_bytes, int64_t max_pages_per_seq, int64_t budget,
                                                 int64_t recent, int64_t sink) {
  if (!evict_sizes_ok(B, row_bytes, max_pages_per_seq, budget, recent, sink)) return 0;
  return evict_layout_of(B, row_bytes, max_pages_per_seq, budget, recent, sink).total;
}

extern "C" int dmla_kv_evict(void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens, const float* mass,
                             int32_t* new_lens, int32_t* src, float* mass_out, int32_t* bad_index_flag, int64_t B,
                             int64_t row_bytes, int64_t num_pages, int64_t max_pages_per_seq, int64_t mass_len,
                             int64_t kv_sp, int64_t kv_ss, int64_t bt_sb, int64_t m_sb, int64_t mo_sb, int64_t src_sb,
                             int64_t budget, int64_t recent, int64_t sink, void* workspace, int64_t workspace_bytes,
                             dmla_stream_t stream) {
  clear_error();
  // (Of an empty call any address does: empty tensors have none.)
  if (B != 0 && (!kv_pool || !block_table || !cache_seqlens || !mass || !new_lens || !src || !mass_out))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: null pointer argument");
  if (B < 0 || num_pages < 0 || max_pages_per_seq < 0 || mass_len < 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: negative size");
  if (budget <= 0 || recent < 0 || sink < 0 || recent > budget || sink > budget - recent)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: budget must be positive and cover recent + sink");
  if (row_bytes <= 0 || row_bytes % 16 != 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: row_bytes must be a positive multiple of 16");
  if (!aligned16(kv_pool)) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: kv_pool must be 16-byte aligned");
  if (kv_sp % 16 != 0 || kv_ss % 16 != 0 || kv_ss < row_bytes || kv_ss > ((int64_t)1 << 31) || kv_sp < kPage * kv_ss)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: strides must be multiples of 16 bytes and cover a row / page");
  if (bt_sb < max_pages_per_seq)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: block_table row stride < max_pages_per_seq");
  if (B == 0) return DMLA_OK;
  if (num_pages == 0 || max_pages_per_seq == 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: empty page pool or block table");
  if (max_pages_per_seq > ((int64_t)1 << 20) || B > ((int64_t)1 << 20) || num_pages > 0x7fffffff || row_bytes > 65536)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_kv_evict: size too large");
  const int64_t cap = max_pages_per_seq * kPage;
  if (mass_len < cap || m_sb < mass_len || mo_sb < mass_len || mass_len > ((int64_t)1 << 30))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: mass rows must cover the block table's tokens");
  const int64_t width = std::min(budget, cap);
  if (src_sb < width) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: src rows must hold min(budget, tokens) entries");
  if (mass == mass_out) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: mass_out must not be mass");
  const int64_t need = dmla_kv_evict_workspace_bytes(B, row_bytes, max_pages_per_seq, budget, recent, sink);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DMLA_ERR_WORKSPACE, "dmla_kv_evict: workspace of %lld bytes needed (got %lld)", (long long)need,
                (long long)workspace_bytes);
  if (!aligned16(workspace)) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: workspace must be 16-byte aligned");
  const bool can_cut = budget < cap;
  const EvictLayout l = evict_layout_of(B, row_bytes, max_pages_per_seq, budget, recent, sink);
  char* ws = static_cast<char*>(workspace);
  EvictArgs a = {};
  a.pool = static_cast<char*>(kv_pool);
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.mass = mass;
  a.new_lens = new_lens; a.src = src; a.mass_out = mass_out; a.bad = bad_index_flag;
  a.kv_sp = kv_sp; a.kv_ss = kv_ss; a.bt_sb = bt_sb; a.m_sb = m_sb; a.mo_sb = mo_sb; a.src_sb = src_sb;
  a.B = (int)B; a.mass_len = (int)mass_len; a.num_pages = (int)num_pages; a.max_pages = (int)max_pages_per_seq;
  a.width = (int)width;
  a.budget = (int)std::min<int64_t>(budget, 0x7fffffff); a.recent = can_cut ? (int)recent : 0; a.sink = can_cut ? (int)sink : 0;
  a.row_chunks = (int)(row_bytes / 16);
  a.info = reinterpret_cast<int32_t*>(ws + l.info);
  a.free_at = reinterpret_cast<int32_t*>(ws + l.free_at);
  a.late_at = reinterpret_cast<int32_t*>(ws + l.late_at);
  a.stage = ws + l.stage;
  a.counts = reinterpret_cast<int32_t*>(ws + l.counts);
  a.above = reinterpret_cast<int32_t*>(ws + l.above);
  a.sel = reinterpret_cast<int32_t*>(ws + l.sel);
  a.per_row = make_fastdiv((unsigned)a.row_chunks);
  const int64_t gy = std::min<int64_t>(B, 65535);
  if (cap <= kOneTokens) {
    auto select = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)gy), dim3(kSelThreads), 0, (hipStream_t)stream, a); };
    // half the tokens a thread where they are enough: 64 sequences of 8192 tokens 36.8 us, 41.5 with all
    if (cap <= kOneTokens / 2) select(evict_select_kernel<kOneTokens / kSelThreads / 2>);
    else select(evict_select_kernel<kOneTokens / kSelThreads>);
  } else {
    a.chunks = (int)evict_chunks(B);
    const dim3 grid((unsigned)a.chunks, (unsigned)gy);
    hipLaunchKernelGGL(evict_chunk_kernel<0>, grid, dim3(kSelThreads), 0, (hipStream_t)stream, a);
    if (can_cut) {
      hipLaunchKernelGGL(evict_chunk_kernel<1>, grid, dim3(kSelThreads), 0, (hipStream_t)stream, a);
      hipLaunchKernelGGL(evict_chunk_kernel<2>, grid, dim3(kSelThreads), 0, (hipStream_t)stream, a);
      hipLaunchKernelGGL(evict_chunk_kernel<3>, grid, dim3(kSelThreads), 0, (hipStream_t)stream, a);
    }
  }
  int rc = check_launch("dmla_kv_evict");
  if (rc != DMLA_OK || !can_cut) return rc;
  // About eight workgroups per CU over all sequences, no more than a sequence has groups of rows.
  const int64_t share = std::max<int64_t>(1, (int64_t)device_cu_count() * 8 / gy);
  auto launch = [&](auto kernel, int64_t rows) {
    const int64_t gx = std::min(share, std::max<int64_t>(1, (rows + kMoveRows - 1) / kMoveRows));
    hipLaunchKernelGGL(kernel, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, (hipStream_t)stream, a);
  };
  launch(evict_move_kernel<0>, std::min(budget - recent - sink, cap - budget) + recent);
  if (recent > 0) launch(evict_move_kernel<1>, recent);
  return check_launch("dmla_kv_evict(move)");
}
