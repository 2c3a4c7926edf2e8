// What the two kernels of the 4-bit decode share (dmla_q4_decode.hip: 32 heads a workgroup, dmla_q4_wide.hip: 128).
#pragma once
#include "dmla_q4.h"
#include "dmla_ranges.h"

namespace dmla {

constexpr int kQ4Dqk = 576, kQ4Dv = 512, kQ4Page = 64;
constexpr int kQ4Tile = 32;                                // tokens of a key tile
constexpr int kQ4TileBytes = kQ4Tile * kQ4RowBytes;        // 12800
constexpr int kQ4Waves = 4, kQ4Threads = 64 * kQ4Waves;    // a wave per SIMD: 512 registers each
static_assert(kQ4Threads == kRangeThreads, "one workgroup cuts the ranges");
// What starting and ending a segment costs, in tiles (dmla_ranges.h), with 32 and with 128 heads a workgroup.
constexpr int kQ4Cost = 24, kQ4WideCost = 8;
// log2 headroom of P over a head's reference
constexpr float kQ4Headroom = 32.0f;
// A block scale from which values (up to 6 scales) may overflow the sums together with the headroom: below it
// 6 x 2^60 x 2^32 leaves room for 2^33 tokens.
constexpr int kQ4BigScale = 60;   // log2

struct Q4DecodeParams {
  const bf16* q;
  const char* kv;
  const int32_t* block_table;
  const int32_t* seqlens;
  bf16* o;
  float* lse;            // nullable
  float* part_o;         // [slots, H, 512]
  float* part_lse;       // [slots, H]
  int32_t* num_splits;   // [B], with split_base what the combine reads
  int32_t* split_base;
  int64_t q_sb, q_sh, kv_sp, bt_sb, o_sb, o_sh;
  int B, H, num_pages, max_pages;
  int head_groups, n_ranges, min_width;
  float scale_log2;
};

// The tiles [t0, t1) of a sequence.
struct Q4Segment {
  int b, t0, t1, ctx, nsplit, slot;
};

// The pages of a segment, 64 at a time in a register (lane i: page first + i).
struct Q4Pages {
  int first = 0, pages = 0;
  bool bad = false;   // a page outside the pool was met

  __device__ __forceinline__ void fetch(const Q4DecodeParams& p, const Q4Segment& sg, int from) {
    first = uniform(from);
    const int i = first + fresh_lane_id();
    pages = i < (sg.t1 + 1) / 2 ? p.block_table[sg.b * p.bt_sb + i] : 0;
    asm volatile("" : "+v"(pages));   // waited for here, in the rare branch, and not by every reader
  }
  // Address of a key tile; tiles come in ascending order.  A bad page reads page 0 instead.
  __device__ __forceinline__ const char* tile(const Q4DecodeParams& p, const Q4Segment& sg, int t) {
    if (t / 2 - first >= 64) fetch(p, sg, first + 64);
    int page = __builtin_amdgcn_readlane(pages, uniform((t / 2 - first) & 63));
    const bool off = page < 0 || page >= p.num_pages;
    bad = bad || off;
    page = off ? 0 : page;
    return p.kv + page * p.kv_sp + (t & 1) * kQ4TileBytes;
  }
};

// What a wave posts at the end of a segment.  It starts over from the largest scores seen if one of them is past the
// headroom, or past its reference at all where big values are in it.
constexpr int kQ4Over = 1, kQ4Climbed = 2, kQ4Big = 4;
__device__ __forceinline__ int q4_climb(float mtrue, float mref, bool big) {
  return (__any(mtrue > mref + kQ4Headroom) ? kQ4Over : 0) | (__any(mtrue > mref) ? kQ4Climbed : 0) | (__any(big) ? kQ4Big : 0);
}
__device__ __forceinline__ bool q4_repeat(int posted) {
  return (posted & kQ4Over) != 0 || (posted & (kQ4Climbed | kQ4Big)) == (kQ4Climbed | kQ4Big);
}

void launch_q4_wide(const Q4DecodeParams& p, int grid, hipStream_t stream);

}  // namespace dmla
