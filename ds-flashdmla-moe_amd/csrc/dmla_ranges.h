// Cutting the cached tokens of a batch over the workgroups of one launch, by workgroups that read nothing
// but the lengths.
//
// The key tiles of all sequences, in order, with kCost virtual tiles before each nonempty one (what
// starting and ending a segment costs), are cut into ranges of equal weight; range r is one workgroup's
// work, and its piece of a sequence is a segment.  Every workgroup works out the same cut: one prefix
// sum over the sequences, kRangeThreads at a time, and no trip through memory.  Range r and sequence b
// share the slot r + b: from one piece to the next r or b grows, so slots are distinct, and those of one
// sequence follow each other.
#pragma once
#include "dmla_common.h"

namespace dmla {

constexpr int kRangeThreads = 256, kRangeWaves = kRangeThreads / 64;

struct RangeLds {   // the segments of one chunk of kRangeThreads sequences
  int lo[kRangeThreads], hi[kRangeThreads], ctx[kRangeThreads], nsplit[kRangeThreads];
  unsigned long long live[kRangeWaves];
  int tmp[kRangeWaves];
};

// Calls segment(b, t0, t1, ctx, nsplit) for every piece of range r, with a barrier after each, and
// owner(b, first_range, nsplit) on one thread for every sequence whose first tile lies in r (the empty
// ones: r = 0).  All kRangeThreads threads take part.  ctx is the length, at most max_tokens.
// The weights' sum stays below 2^31 (checked on the host).
template <int kTokens, int kCost, typename SegmentFn, typename OwnerFn>
__device__ __forceinline__ void for_each_segment(const int32_t* seqlens, int B, int max_tokens, int n_ranges, int min_width,
                                                 int r, RangeLds& lds, SegmentFn segment, OwnerFn owner) {
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = uniform(tid >> 6);
  auto length_of = [&](int b) { return b < B ? min(max(seqlens[b], 0), max_tokens) : 0; };
  auto weight_of = [&](int nt) { return nt > 0 ? nt + kCost : 0; };
  int ctx = length_of(tid);
  int total = 0;
  for (int c0 = 0; c0 < B; c0 += kRangeThreads)
    total += weight_of(((c0 == 0 ? ctx : length_of(c0 + tid)) + kTokens - 1) / kTokens);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o, 64);
  if (lane == 0) lds.tmp[wave] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kRangeWaves; ++w) total += lds.tmp[w];
  const int width = max(min_width, (total + n_ranges - 1) / n_ranges);
  int carry = 0;
  for (int c0 = 0; c0 < B; c0 += kRangeThreads) {
    const int b = c0 + tid;
    if (c0 > 0) ctx = length_of(b);
    const int nt = (ctx + kTokens - 1) / kTokens, w = weight_of(nt);
    int x = w;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    __syncthreads();   // tmp has been read
    if (lane == 63) lds.tmp[wave] = x;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int v = 0; v < kRangeWaves; ++v) {
      if (v < wave) before += lds.tmp[v];
      carry += lds.tmp[v];
    }
    const int first_tile = before + x - w + kCost;   // weighted position of the sequence's first tile
    const int fr = first_tile / width;
    const int ns = nt > 0 ? (first_tile + nt - 1) / width - fr + 1 : 0;
    const int64_t at = (int64_t)r * width - first_tile;   // 64 bits: the last ranges may start past the total
    const int lo = (int)min(max(at, (int64_t)0), (int64_t)nt), hi = (int)min(max(at + width, (int64_t)0), (int64_t)nt);
    lds.lo[tid] = lo;
    lds.hi[tid] = hi;
    lds.ctx[tid] = ctx;
    lds.nsplit[tid] = ns;
    const unsigned long long live = __ballot(hi > lo);
    if (lane == 0) lds.live[wave] = live;
    if (b < B && (nt > 0 ? r == fr : r == 0)) owner(b, fr, ns);
    __syncthreads();
    for (int v = 0; v < kRangeWaves; ++v) {
      const unsigned long long lv = lds.live[v];
      unsigned long long m =
          ((unsigned long long)(unsigned)uniform((int)(lv >> 32)) << 32) | (unsigned)uniform((int)(unsigned)lv);
      while (m != 0) {
        const int i = 64 * v + __builtin_ctzll(m);
        m &= m - 1;
        segment(c0 + i, uniform(lds.lo[i]), uniform(lds.hi[i]), uniform(lds.ctx[i]), uniform(lds.nsplit[i]));
        __syncthreads();
      }
    }
  }
}

}  // namespace dmla
