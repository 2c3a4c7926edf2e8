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
  int lo[kRangeThreads], hi[kRangeThreads], ctx[kRangeThreads];
  unsigned short nsplit[kRangeThreads];   // at most a part per workgroup
  unsigned long long live[kRangeWaves];
  int tmp[kRangeWaves];
};

// Whether the cut of B sequences of at most `tiles` tiles stays within 32-bit integers: their weights' sum, the
// rounding up of its division by the ranges, and the cost that stands before an empty sequence at the end.
inline bool ranges_fit(int64_t B, int64_t tiles, int64_t cost, int64_t n_ranges) {
  return B * (tiles + cost) + n_ranges + cost <= 0x7fffffff;
}

// Calls segment(b, t0, t1, ctx, nsplit) for every piece of range r, with a barrier after each, and
// owner(b, first_range, nsplit) on one thread for every sequence whose first tile lies in r (the empty
// ones: r = 0).  All threads of the workgroup take part, those past kRangeThreads in the barriers.  ctx is
// the length, at most max_tokens.
// The sums are 32-bit integers: the host has checked ranges_fit.
template <int kTokens, int kCost, typename SegmentFn, typename OwnerFn>
__device__ __forceinline__ void for_each_segment(const int32_t* seqlens, int B, int max_tokens, int n_ranges, int min_width,
                                                 int r, RangeLds& lds, SegmentFn segment, OwnerFn owner) {
  const int tid = threadIdx.x;
  const int lane = tid & 63, wave = uniform(tid >> 6);
  const bool in = tid < kRangeThreads;
  auto length_of = [&](int b) { return in && b < B ? min(max(seqlens[b], 0), max_tokens) : 0; };
  auto tiles_of = [&](int len) { return (len + kTokens - 1) / kTokens; };
  auto weight_of = [&](int nt) { return nt > 0 ? nt + kCost : 0; };
  // Sum of the threads' w up to this one; sum: over all.  The first use of lds.tmp, or after a barrier.
  auto scan = [&](int w, int& sum) {
    int x = lane_scan(w);
    if (in && lane == 63) lds.tmp[wave] = x;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int v = 0; v < kRangeWaves; ++v) {
      if (v < wave) x += lds.tmp[v];
      sum += lds.tmp[v];
    }
    return x;
  };
  int ctx = length_of(tid);
  int chunk = 0;   // weight of the chunk
  int x = scan(weight_of(tiles_of(ctx)), chunk);
  int total = chunk;
  if (B > kRangeThreads) {
    int w = 0, rest = 0;
    for (int c0 = kRangeThreads; c0 < B; c0 += kRangeThreads) w += weight_of(tiles_of(length_of(c0 + tid)));
    __syncthreads();   // tmp has been read
    scan(w, rest);
    total += rest;
  }
  const int width = max(min_width, (total + n_ranges - 1) / n_ranges);
  int carry = 0;   // weight of the chunks before
  for (int c0 = 0; c0 < B; c0 += kRangeThreads) {
    const int b = c0 + tid;
    if (c0 > 0) {
      ctx = length_of(b);
      __syncthreads();   // tmp has been read
      x = scan(weight_of(tiles_of(ctx)), chunk);
    }
    const int nt = tiles_of(ctx), w = weight_of(nt);
    const int first_tile = carry + x - w + kCost;   // weighted position of the sequence's first tile
    carry += chunk;
    const int fr = first_tile / width;
    const int ns = nt > 0 ? (first_tile + nt - 1) / width - fr + 1 : 0;
    const int64_t at = (int64_t)r * width - first_tile;   // 64 bits: the last ranges may start past the total
    const int lo = (int)min(max(at, (int64_t)0), (int64_t)nt), hi = (int)min(max(at + width, (int64_t)0), (int64_t)nt);
    const unsigned long long live = __ballot(hi > lo);
    if (in) {
      lds.lo[tid] = lo;
      lds.hi[tid] = hi;
      lds.ctx[tid] = ctx;
      lds.nsplit[tid] = (unsigned short)ns;
      if (lane == 0) lds.live[wave] = live;
    }
    if (in && b < B && (nt > 0 ? r == fr : r == 0)) owner(b, fr, ns);
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
