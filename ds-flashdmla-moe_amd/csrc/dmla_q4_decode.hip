// Paged decode over the 4-bit latent cache (row format: dmla_q4.h): one query token per sequence.
//
//   s_ht = scale q_h . k_t,  o_h = sum_t softmax(s_h)_t k_t[:512],  k_t = code x scale (exact)
//
// MI355X design:
//  * Key tiles of 32 tokens are copied global -> LDS as they lie in the cache (400 bytes per token) into
//    a ring of slots and become bf16 on the way to the MFMA, two values per instruction, scale included.
//    (The scaled MFMA would take the codes as they are, but it sums the products of an instruction in
//    fixed point, some 14 bits below the largest: scores 2^-14 of their terms off, where bf16 products
//    are exact and sum in fp32.)
//  * The score product has the keys as its rows, so a lane ends with 8 keys' scores of one head, which is
//    the operand layout that the value product takes its probabilities in.
//  * The value product needs keys along the MFMA's k.  A lane reads the codes of 32 / kHW neighbouring
//    columns -- of one scale block -- of 8 keys, converts them and joins equal columns of two keys with a
//    byte permute: 8 instructions per MFMA operand.  MFMA number j then holds column (32 / kHW) m + j in row m.
//  * Four waves per workgroup, one per SIMD with 512 registers.  A wave computes the scores and the
//    softmax of up to 32 heads (their queries: 144 registers).  kHW waves with different heads share a key
//    tile and exchange probabilities through LDS, so that each holds all their heads' outputs for 512 / kHW
//    columns (256 registers) and every code is converted for the value product by one wave only;
//    4 / kHW such groups work on different tiles and meet in LDS at the end of a segment.
//  * The value product of a tile runs one step behind its scores: one barrier per step, and the two
//    products of a step are independent.
//  * The softmax reference of a head rises only when a score passes it by 2^8 (kLazy), so outputs are
//    rarely rescaled; P keeps bf16's relative precision whatever its size, sums stay in fp32.
//  * Sequences are cut over the chip's workgroups by weight (dmla_ranges.h); sequences in several parts
//    are merged by the split-KV combine.
#include <algorithm>

#include "dmla_host.h"
#include "dmla_q4.h"
#include "dmla_ranges.h"

namespace dmla {
namespace {

constexpr int kDqk = 576, kDv = 512, kPage = 64;
constexpr int kTile = 32;                            // tokens of a key tile
constexpr int kTileBytes = kTile * kQ4RowBytes;      // 12800
constexpr int kCopies = (kTileBytes + 1023) / 1024;  // wave copies of a tile, the last one half
constexpr int kWaves = 4, kThreads = 64 * kWaves;
static_assert(kThreads == kRangeThreads, "one workgroup cuts the ranges");
constexpr float kLazy = 8.0f;

struct Q4DecodeParams {
  const bf16* q;
  const char* kv;
  const int32_t* block_table;
  const int32_t* seqlens;
  bf16* o;
  float* lse;            // nullable
  bf16* part_o;          // [slots, H, 512]
  float* part_lse;       // [slots, H]
  int32_t* num_splits;   // [B], with split_base what the combine reads
  int32_t* split_base;
  int64_t q_sb, q_sh, kv_sp, bt_sb, o_sb, o_sh;
  int B, H, num_pages, max_pages;
  int head_groups, n_ranges, min_width;
  float scale_log2;
};

template <int kNH, int kHW>
struct Shape {
  static constexpr int kKP = kWaves / kHW;              // tiles in work at once
  static constexpr int kSlotBytes = kKP * kTileBytes;
  static constexpr int kSlots = kHW == 1 ? 3 : kHW == 2 ? 5 : 8;
  static constexpr int kRingBytes = kSlots * kSlotBytes;
  static constexpr int kNB = kHW * kNH;                 // head blocks of 16 of a workgroup
  static constexpr int kHeads = kNB * 16;
  static constexpr int kCols = 32 / kHW;                // neighbouring columns of a lane
  static constexpr int kLag = kHW > 1 ? 1 : 0;          // steps the value product runs behind
  static constexpr int kXBytes = kHW > 1 ? 2 * kKP * kNB * 1024 : 16;   // P of two steps
  static constexpr int kMergeRow = 128 / kHW + 4;       // floats, padded against bank conflicts
  static constexpr int kMergeBytes = kWaves * kHeads * kMergeRow * 4;
  static constexpr int kSegCost = kHW == 1 ? 16 : kHW == 2 ? 10 : 5;
  static_assert(kKP == 1 || kMergeBytes <= kRingBytes, "the merge reuses the ring");
};

struct Segment {
  int b, t0, t1, ctx, nsplit, slot;
};

struct Lds {
  DMLA_LDS char* ring;
  DMLA_LDS char* p;        // [2][kKP][kNB][64 lanes] x 16 bytes
  DMLA_LDS float* alpha;   // [2][kKP][kHeads]: what a step multiplies the outputs by; after the last step
                           // [kKP][kHeads][2], references and sums
  DMLA_LDS int* flag;      // [kWaves]
};

// One segment: the tiles [t0, t1) of a sequence.
template <int kNH, int kHW>
__device__ __forceinline__ void run_segment(const Q4DecodeParams& p, const Segment& sg, const Lds& lds, int head0) {
  using S = Shape<kNH, kHW>;
  constexpr int kKP = S::kKP, kNB = S::kNB, kCols = S::kCols;
  const int lane = fresh_lane_id();
  const int l16 = lane & 15, g = lane >> 4;
  const int wave = uniform(threadIdx.x >> 6);
  const int hw = wave % kHW, kp = wave / kHW;
  const int n_steps = (sg.t1 - sg.t0 + kKP - 1) / kKP;
  bool bad_page = false;

  // Pages of this wave's tiles, 64 at a time in a register (lane i: page page0 + i).
  int page0 = sg.t0 / 2, pages = 0;
  auto fetch_pages = [&]() {
    const int i = page0 + lane;
    pages = i < (sg.t1 + 1) / 2 ? p.block_table[sg.b * p.bt_sb + i] : 0;
  };
  fetch_pages();
  const unsigned ring_addr = lds_addr(lds.ring);
  // This wave's share of the copies of step s's tile kp: pieces hw, hw + kHW, ...
  auto copy_step = [&](int s) {
    const int t = sg.t0 + s * kKP + kp;
    if (t >= sg.t1) return;
    if (t / 2 - page0 >= 64) {
      page0 += 64;
      fetch_pages();
    }
    int page = __builtin_amdgcn_readlane(pages, (t / 2 - page0) & 63);
    const bool bad = page < 0 || page >= p.num_pages;
    bad_page = bad_page || bad;
    page = bad ? 0 : page;
    const char* src = p.kv + page * p.kv_sp + (t & 1) * kTileBytes;
    const unsigned dst = ring_addr + (unsigned)((s % S::kSlots) * S::kSlotBytes + kp * kTileBytes);
    const int valid = sg.ctx - t * kTile;
    if (valid >= kTile) {
#pragma unroll
      for (int k = 0; k < kCopies; ++k) {
        if (k % kHW != hw) continue;
        if (k < kCopies - 1 || lane < 32) dma16(src + k * 1024, 16u * lane, dst + k * 1024);
      }
    } else {   // rows past the sequence's end re-read the tile's first row: finite data, masked below
#pragma unroll
      for (int k = 0; k < kCopies; ++k) {
        if (k % kHW != hw) continue;
        const int i = k * 64 + lane, row = i / kQ4Chunks, col = i - row * kQ4Chunks;
        if (k < kCopies - 1 || lane < 32) dma16(src, 16u * (row < valid ? i : col), dst + k * 1024);
      }
    }
  };

  bf16x8 q[kNH][kQ4KeySteps];
#pragma unroll
  for (int h = 0; h < kNH; ++h) {
    const int head = min(head0 + (hw * kNH + h) * 16 + l16, p.H - 1);
    q4_load_query(p.q + sg.b * p.q_sb + head * p.q_sh, g, q[h]);
  }

  f32x4 acc[kNB][kCols];   // O^T: row m = 4 g + i is column (512 / kHW) hw + kCols m + j, for head l16
  float mref[kNH], lsum[kNH];
#pragma unroll
  for (int h = 0; h < kNH; ++h) {
    mref[h] = kNegInf;
    lsum[h] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < kNB; ++n)
#pragma unroll
    for (int j = 0; j < kCols; ++j) acc[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16x8 pv[kNH];          // P of the wave's own heads
  float alpha[kNH];

  // S^T[key 16 kb + 4 g + i][head l16] of a tile, then P and alpha.
  auto scores = [&](int s, int t) {
    const DMLA_LDS char* tile = lds.ring + (s % S::kSlots) * S::kSlotBytes + kp * kTileBytes;
    f32x4 sc[kNH][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      Q4Key key;
      key.load(tile + (16 * kb + l16) * kQ4RowBytes, g);
#pragma unroll
      for (int h = 0; h < kNH; ++h) sc[h][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
      auto step = [&](auto a_tag) {
        constexpr int kA = decltype(a_tag)::value;
        bf16x8 k[4];
        key.octets<kA>(k);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int h = 0; h < kNH; ++h) sc[h][kb] = mfma_bf16(k[b], q[h][4 * kA + b], sc[h][kb]);
      };
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
      step(std::integral_constant<int, 2>{});
      step(std::integral_constant<int, 3>{});
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int h = 0; h < kNH; ++h) sc[h][kb] = mfma_bf16(key.rope[c], q[h][16 + c], sc[h][kb]);
    }
    const int left = sg.ctx - t * kTile;   // keys of the tile
#pragma unroll
    for (int h = 0; h < kNH; ++h) {
      float x[8], mx = kNegInf;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = sc[h][j >> 2][j & 3] * p.scale_log2;
        x[j] = 16 * (j >> 2) + 4 * g + (j & 3) < left ? x[j] : kNegInf;
        mx = fmaxf(mx, x[j]);
      }
      mx = group_max(mx);
      const bool rise = mx > mref[h] + kLazy || mref[h] == kNegInf;
      const float mnew = rise ? fmaxf(mx, mref[h]) : mref[h];
      alpha[h] = rise && mnew != kNegInf ? fast_exp2(mref[h] - mnew) : 1.f;
      mref[h] = mnew;
      lsum[h] *= alpha[h];
      const float ms = mnew == kNegInf ? 0.f : mnew;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float e = fast_exp2(x[j] - ms);
        lsum[h] += e;
        pv[h][j] = (bf16)e;
      }
    }
  };
  auto rescale = [&](int n, float al) {
    if (__any(al != 1.f)) {
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[n][j] *= al;
    }
  };
  // O^T += V^T P of step s's tile; pb(n): P of head block n.
  auto values = [&](int s, auto pb) {
    const DMLA_LDS char* tile = lds.ring + (s % S::kSlots) * S::kSlotBytes + kp * kTileBytes;
    unsigned vc[8][kCols / 8];
    float vs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {   // the keys of the scores: 4 g + j, then 16 + 4 g + j - 4
      const DMLA_LDS char* row = tile + (16 * (j >> 2) + 4 * g + (j & 3)) * kQ4RowBytes;
      const DMLA_LDS char* at = row + (256 / kHW) * hw + (kCols / 2) * l16;
      if constexpr (kCols == 32) {
        const u32x4 w = *reinterpret_cast<const DMLA_LDS u32x4*>(at);
#pragma unroll
        for (int d = 0; d < 4; ++d) vc[j][d] = w[d];
      } else if constexpr (kCols == 16) {
        const u32x2 w = *reinterpret_cast<const DMLA_LDS u32x2*>(at);
        vc[j][0] = w[0];
        vc[j][1] = w[1];
      } else {
        vc[j][0] = *reinterpret_cast<const DMLA_LDS unsigned*>(at);
      }
      vs[j] = q4_scale(*reinterpret_cast<const DMLA_LDS uint8_t*>(row + kQ4ScaleOff + (16 / kHW) * hw + l16 / kHW));
    }
    auto column_pair = [&](auto byte_tag, int d) {
      constexpr int kB = decltype(byte_tag)::value;
      unsigned e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = __builtin_bit_cast(unsigned, q4_pair<kB>(vc[j][d], vs[j]));
      u32x4 even, odd;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        even[r] = __builtin_amdgcn_perm(e[2 * r + 1], e[2 * r], 0x05040100u);
        odd[r] = __builtin_amdgcn_perm(e[2 * r + 1], e[2 * r], 0x07060302u);
      }
#pragma unroll
      for (int n = 0; n < kNB; ++n) {
        const int j = 8 * d + 2 * kB;
        acc[n][j] = mfma_bf16(__builtin_bit_cast(bf16x8, even), pb(n), acc[n][j]);
        acc[n][j + 1] = mfma_bf16(__builtin_bit_cast(bf16x8, odd), pb(n), acc[n][j + 1]);
      }
    };
#pragma unroll
    for (int d = 0; d < kCols / 8; ++d) {
      column_pair(std::integral_constant<int, 0>{}, d);
      column_pair(std::integral_constant<int, 1>{}, d);
      column_pair(std::integral_constant<int, 2>{}, d);
      column_pair(std::integral_constant<int, 3>{}, d);
    }
  };
  // P and alpha of step s through LDS, between the waves of a group.
  auto post = [&](int s) {
#pragma unroll
    for (int h = 0; h < kNH; ++h) {
      const int n = hw * kNH + h, at = (s & 1) * kKP + kp;
      *reinterpret_cast<DMLA_LDS bf16x8*>(lds.p + (at * kNB + n) * 1024 + lane * 16) = pv[h];
      if (g == 0) lds.alpha[(at * kNB + n) * 16 + l16] = alpha[h];
    }
  };
  auto shared_values = [&](int s) {
    const int at = (s & 1) * kKP + kp;
    bf16x8 pall[kNB];
#pragma unroll
    for (int n = 0; n < kNB; ++n) {
      pall[n] = lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(lds.p + (at * kNB + n) * 1024 + lane * 16));
      rescale(n, lds.alpha[(at * kNB + n) * 16 + l16]);
    }
    values(s, [&](int n) { return pall[n]; });
  };

  // Copies run kSlots - 1 - kLag steps ahead: at step s the slot of step s - 1 - kLag is refilled.
  constexpr int kAhead = S::kSlots - 1 - S::kLag;
  for (int s = 0; s < kAhead && s < n_steps; ++s) copy_step(s);
  for (int s = 0; s < n_steps; ++s) {
    // This wave's copies of step s have landed; those of the kAhead - 1 steps after it stay in flight.
    constexpr int kFlight = kAhead - 1;
    constexpr int kMost = (kCopies + kHW - 1) / kHW, kLeast = kCopies / kHW;
    if (s + kFlight >= n_steps - 1) wait_vm<0>();   // the last steps' tiles need not exist
    else if (hw < kCopies % kHW || kCopies % kHW == 0) wait_vm<kFlight * kMost>();
    else wait_vm<kFlight * kLeast>();
    wait_lds();   // this wave's reads of the slot that is refilled below are done
    if constexpr (kHW > 1) __syncthreads();   // and everybody's; all copies of step s have landed
    if (s + kAhead < n_steps) copy_step(s + kAhead);
    const int t = sg.t0 + s * kKP + kp;
    if constexpr (kHW > 1) {
      if (s > 0) shared_values(s - 1);
      if (t < sg.t1) {
        scores(s, t);
        post(s);
      }
    } else {
      if (t >= sg.t1) continue;
      scores(s, t);
#pragma unroll
      for (int h = 0; h < kNH; ++h) rescale(h, alpha[h]);
      values(s, [&](int n) { return pv[n]; });
    }
  }
  if constexpr (kHW > 1) {
    __syncthreads();
    if (sg.t0 + (n_steps - 1) * kKP + kp < sg.t1) shared_values(n_steps - 1);
  }

  // ---- the segment's output ----
#pragma unroll
  for (int h = 0; h < kNH; ++h) lsum[h] = group_sum(lsum[h]);
  wait_vm<0>();
  wait_lds();
  __syncthreads();   // the ring and the exchange are free
  if (g == 0) {
#pragma unroll
    for (int h = 0; h < kNH; ++h) {
      const int at = (kp * S::kHeads + (hw * kNH + h) * 16 + l16) * 2;
      lds.alpha[at] = mref[h];
      lds.alpha[at + 1] = lsum[h];
    }
  }
  if (lane == 0) lds.flag[wave] = bad_page ? 1 : 0;
  __syncthreads();
  const float nanv = __builtin_nanf("");
  const bool poison = (lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]) != 0;
  // Reference and sum of a head of the workgroup over the tile groups.
  auto joined = [&](int hd, float& top, float& sum) {
    top = kNegInf;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < kKP; ++k) top = fmaxf(top, lds.alpha[(k * S::kHeads + hd) * 2]);
#pragma unroll
    for (int k = 0; k < kKP; ++k) {
      const float m = lds.alpha[(k * S::kHeads + hd) * 2], l = lds.alpha[(k * S::kHeads + hd) * 2 + 1];
      sum += m == kNegInf ? l : l * fast_exp2(m - top);   // no finite reference: 0, or NaN
    }
    if (poison) sum = nanv;
  };
  auto out_row = [&](int head) {
    return sg.nsplit == 1 ? p.o + sg.b * p.o_sb + head * p.o_sh : p.part_o + ((int64_t)sg.slot * p.H + head) * kDv;
  };
  auto put_lse = [&](int head, float top, float sum) {
    const float lse = sum == 0.f ? kNegInf : (top + __log2f(sum)) * kLn2;
    if (sg.nsplit > 1) p.part_lse[(int64_t)sg.slot * p.H + head] = lse;
    else if (p.lse != nullptr) p.lse[sg.b * p.H + head] = lse;
  };
  if constexpr (kKP == 1) {
#pragma unroll
    for (int n = 0; n < kNB; ++n) {
      const int head = head0 + 16 * n + l16;
      if (head >= p.H) continue;
      float top, sum;
      joined(16 * n + l16, top, sum);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      bf16* orow = out_row(head) + (kDv / kHW) * hw;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < kCols / 8; ++d) {
          bf16x8 v;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = (bf16)(acc[n][8 * d + j][i] * inv);
          *reinterpret_cast<bf16x8*>(orow + kCols * (4 * g + i) + 8 * d) = v;
        }
      if (g == 0 && hw == n % kHW) put_lse(head, top, sum);
    }
  } else {
    // The tile groups' outputs meet in LDS, one row index i of the accumulators a round (512 / 4
    // columns of all heads): each group's at the common reference.
    DMLA_LDS float* merge = reinterpret_cast<DMLA_LDS float*>(lds.ring);
    float fac[kNB];
#pragma unroll
    for (int n = 0; n < kNB; ++n) {
      float top, sum;
      joined(16 * n + l16, top, sum);
      const float m = lds.alpha[(kp * S::kHeads + 16 * n + l16) * 2];
      fac[n] = m == kNegInf ? 0.f : fast_exp2(m - top);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int n = 0; n < kNB; ++n) {
        DMLA_LDS float* at = merge + ((wave * kNB + n) * 16 + l16) * S::kMergeRow + kCols * g;
#pragma unroll
        for (int d = 0; d < kCols / 4; ++d) {
          f32x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = acc[n][4 * d + j][i] * fac[n];
          *reinterpret_cast<DMLA_LDS f32x4*>(at + 4 * d) = v;
        }
      }
      __syncthreads();
#pragma unroll
      for (int it = 0; it < S::kHeads * 16 / kThreads; ++it) {
        const int item = it * kThreads + threadIdx.x;
        const int hd = item >> 4, cc = (item & 15) * 8;   // head, and 8 of the round's 128 columns
        const int w0 = cc / (128 / kHW), lc = cc % (128 / kHW);   // the wave that holds them, and where
        const int head = head0 + hd;
        float top, sum;
        joined(hd, top, sum);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
#pragma unroll
        for (int k = 0; k < kKP; ++k) {
          const DMLA_LDS float* from = merge + ((k * kHW + w0) * S::kHeads + hd) * S::kMergeRow + lc;
          v0 += *reinterpret_cast<const DMLA_LDS f32x4*>(from);
          v1 += *reinterpret_cast<const DMLA_LDS f32x4*>(from + 4);
        }
        if (head < p.H) {
          bf16x8 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = (bf16)(v0[j] * inv);
            v[4 + j] = (bf16)(v1[j] * inv);
          }
          *reinterpret_cast<bf16x8*>(out_row(head) + (kDv / kHW) * w0 + kCols * (4 * (lc / kCols) + i) + lc % kCols) = v;
          if (i == 0 && cc == 0) put_lse(head, top, sum);
        }
      }
      __syncthreads();   // read out before the next round writes
    }
  }
}

// One workgroup per range (dmla_ranges.h) and head group.
template <int kNH, int kHW>
__global__ __launch_bounds__(kThreads, 1) void q4_decode_kernel(Q4DecodeParams p) {
  using S = Shape<kNH, kHW>;
  __shared__ __attribute__((aligned(1024))) char ring[S::kRingBytes];
  __shared__ __attribute__((aligned(1024))) char p_mem[S::kXBytes];
  __shared__ __attribute__((aligned(16))) float alpha[2 * S::kKP * S::kHeads];
  __shared__ __attribute__((aligned(16))) int flag[kWaves];
  __shared__ __attribute__((aligned(16))) RangeLds ranges;
  const Lds lds = {(DMLA_LDS char*)ring, (DMLA_LDS char*)p_mem, (DMLA_LDS float*)alpha, (DMLA_LDS int*)flag};
  // The head groups of a range run 8 ids apart, on one XCD: the second read of its pages hits that L2.
  const int id = blockIdx.x;
  const int hg = (id / 8) % p.head_groups;
  const int r = (id / (8 * p.head_groups)) * 8 + id % 8;
  if (r >= p.n_ranges) return;
  for_each_segment<kTile, S::kSegCost>(
      p.seqlens, p.B, p.max_pages * kPage, p.n_ranges, p.min_width, r, ranges,
      [&](int b, int t0, int t1, int ctx, int nsplit) {
        run_segment<kNH, kHW>(p, Segment{b, t0, t1, ctx, nsplit, r + b}, lds, hg * S::kHeads);
      },
      [&](int b, int first_range, int nsplit) {
        if (hg != 0) return;
        p.num_splits[b] = nsplit;
        p.split_base[b] = first_range + b;
      });
}

// Heads of a workgroup, by the number of heads: see kShapes' use in the launch.
int wg_heads(int64_t H) { return H <= 16 ? 16 : H <= 32 ? 32 : H <= 64 ? 64 : 128; }
int64_t q4_ranges(int64_t H) {
  const int64_t hg = (H + wg_heads(H) - 1) / wg_heads(H);
  return std::max<int64_t>(1, device_cu_count() / hg);
}

}  // namespace
}  // namespace dmla

using namespace dmla;

static int64_t q4_plan_bytes(int64_t B) { return (B * 8 + 255) / 256 * 256; }

extern "C" int64_t dmla_decode_q4_workspace_bytes(int64_t B, int64_t H) {
  if (B <= 0 || H <= 0 || B > ((int64_t)1 << 20) || H > ((int64_t)1 << 16)) return 0;
  return q4_plan_bytes(B) + (q4_ranges(H) + B) * H * (int64_t)(kDv * 2 + 4);
}

extern "C" int dmla_decode_paged_q4(const void* q, const void* kv_pool, const int32_t* block_table,
                                    const int32_t* cache_seqlens, void* o, float* lse, int64_t B, int64_t H,
                                    int64_t d_qk, int64_t d_v, int64_t num_pages, int64_t max_pages_per_seq,
                                    int64_t q_sb, int64_t q_sh, int64_t kv_sp, int64_t bt_sb, int64_t o_sb, int64_t o_sh,
                                    float softmax_scale, void* workspace, int64_t workspace_bytes, dmla_stream_t stream) {
  clear_error();
  if (!q || !kv_pool || !block_table || !cache_seqlens || !o)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: null pointer argument");
  if (B < 0 || H < 0 || num_pages < 0 || max_pages_per_seq < 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: negative size");
  if (d_qk != kDqk || d_v != kDv)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_decode_paged_q4: only d_qk=576, d_v=512 is compiled (got %lld, %lld)",
                (long long)d_qk, (long long)d_v);
  if (!(softmax_scale > 0.f) || !__builtin_isfinite(softmax_scale))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: softmax_scale must be finite and > 0");
  if (!aligned16(q) || !aligned16(kv_pool) || !aligned16(o))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: q/kv_pool/o must be 16-byte aligned");
  if (!mult8(q_sb) || !mult8(q_sh) || !mult8(o_sb) || !mult8(o_sh))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: strides must be multiples of 8 elements");
  if (kv_sp % 16 != 0 || kv_sp < kPage * kQ4RowBytes)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: page stride must be a multiple of 16 bytes and cover a page");
  if (bt_sb < max_pages_per_seq)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: block_table row stride < max_pages_per_seq");
  if (H > ((int64_t)1 << 16) || B > ((int64_t)1 << 20) || max_pages_per_seq > ((int64_t)1 << 24) || num_pages > 0x7fffffff ||
      B * (max_pages_per_seq * 2 + 16) >= ((int64_t)1 << 31))
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_decode_paged_q4: size too large");
  if (B == 0 || H == 0) return DMLA_OK;
  if (num_pages == 0 || max_pages_per_seq == 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: empty page pool or block table");
  const int64_t need = dmla_decode_q4_workspace_bytes(B, H);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DMLA_ERR_WORKSPACE, "dmla_decode_paged_q4: workspace of %lld bytes needed (got %lld)", (long long)need,
                (long long)workspace_bytes);
  if (!aligned16(workspace)) return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: workspace must be 16-byte aligned");
  const int64_t R = q4_ranges(H), slots = R + B;
  char* ws = static_cast<char*>(workspace);
  Q4DecodeParams p = {};
  p.q = static_cast<const bf16*>(q);
  p.kv = static_cast<const char*>(kv_pool);
  p.block_table = block_table;
  p.seqlens = cache_seqlens;
  p.o = static_cast<bf16*>(o);
  p.lse = lse;
  p.num_splits = reinterpret_cast<int32_t*>(ws);
  p.split_base = p.num_splits + B;
  p.part_o = reinterpret_cast<bf16*>(ws + q4_plan_bytes(B));
  p.part_lse = reinterpret_cast<float*>(p.part_o + slots * H * kDv);
  p.q_sb = q_sb; p.q_sh = q_sh; p.kv_sp = kv_sp; p.bt_sb = bt_sb; p.o_sb = o_sb; p.o_sh = o_sh;
  p.B = (int)B; p.H = (int)H; p.num_pages = (int)num_pages; p.max_pages = (int)max_pages_per_seq;
  p.head_groups = (int)((H + wg_heads(H) - 1) / wg_heads(H));
  p.n_ranges = (int)R;
  p.scale_log2 = softmax_scale * kLog2e;
  const dim3 grid((unsigned)((R + 7) / 8 * 8 * p.head_groups));
  switch (wg_heads(H)) {
    case 16: p.min_width = 32; hipLaunchKernelGGL((q4_decode_kernel<1, 1>), grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
    case 32: p.min_width = 32; hipLaunchKernelGGL((q4_decode_kernel<2, 1>), grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
    case 64: p.min_width = 16; hipLaunchKernelGGL((q4_decode_kernel<2, 2>), grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
    default: p.min_width = 8; hipLaunchKernelGGL((q4_decode_kernel<2, 4>), grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
  }
  const int rc = check_launch("dmla_decode_paged_q4");
  if (rc != DMLA_OK) return rc;
  // Sequences in one part were written above; the others, and the empty ones, come from the combine.
  CombineArgs c = {};
  c.part_o16 = p.part_o;
  c.part_lse = p.part_lse;
  c.split_base = p.split_base;
  c.num_splits = p.num_splits;
  c.o = p.o;
  c.lse = lse;
  c.B = (int)B; c.H = (int)H; c.max_splits = (int)R + 1; c.d = kDv;
  c.mean_splits = (int)((R + B - 1) / B);
  c.skip_single = 1;
  c.po_ss = H * kDv; c.po_sh = kDv;
  c.lse_ss = H; c.lse_sh = 1;
  c.o_sb = o_sb; c.o_sh = o_sh;
  return launch_lse_combine(c, (hipStream_t)stream, "dmla_decode_paged_q4(combine)");
}
