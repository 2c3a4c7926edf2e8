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
//  * The softmax reference of a head is its largest score in the segment's first tile; P may grow to 2^32
//    past it (bf16 keeps its relative precision whatever the size, sums stay in fp32), and a segment
//    whose scores climb further starts over from their exact maximum.
//  * Sequences are cut over the chip's workgroups by weight (dmla_ranges.h); sequences in several parts
//    are merged by the split-KV combine.
#include <algorithm>
#include <type_traits>

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
constexpr float kHeadroom = 32.0f;   // log2 headroom of P over a head's reference

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

// The output accumulators fill the AGPR file.  Where ordinary code touches them, the compiler gives them a
// home among the VGPRs as well and spills the queries; these accesses leave them where they are.  The
// compiler does not see into the assembly, so agpr_settle() keeps them clear of MFMAs on the same register.
__device__ __forceinline__ float agpr_read(float x) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(x));
  return v;
}
// Longer than any MFMA takes to write its result, or a write to reach one.
__device__ __forceinline__ void agpr_settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// One step of the score product, x += k q (x = k q for the first of a tile).  In assembly because the
// AGPRs have no room for x beside the accumulators and the compiler gives every MFMA of a kernel the same
// register file.  It does not see the waits that such an operand needs, so they are here: two states after
// a VALU write of an operand or another step on x (both pass while the matrix core is busy).  score_done()
// stands between the last step and the first read of x.
template <bool kFirst>
__device__ __forceinline__ void score_step(f32x16& x, const bf16x8& k, const bf16x8& q) {
  if constexpr (kFirst) asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(x) : "v"(k), "v"(q));
  else asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(x) : "v"(k), "v"(q));
}
__device__ __forceinline__ void score_done(f32x16& x) { asm("s_nop 15\n\ts_nop 7" : "+v"(x)); }

// f(0), f(1), .., f(kN - 1) with compile-time arguments.
template <int kN, typename F, int kI = 0>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (kI < kN) {
    f(std::integral_constant<int, kI>{});
    static_for<kN, F, kI + 1>(f);
  }
}

// Nothing moves across: the order of a pipelined loop body is the source's.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

template <int kHW>
struct Shape {
  static constexpr int kKP = kWaves / kHW;              // tiles in work at once
  static constexpr int kSlotBytes = kKP * kTileBytes;
  static constexpr int kSlots = kHW == 1 ? 3 : kHW == 2 ? 4 : 6;
  static constexpr int kRingBytes = kSlots * kSlotBytes;
  static constexpr int kHeads = 32 * kHW;               // heads of a workgroup
  static constexpr int kCols = 16 / kHW;                // neighbouring columns of a lane
  static constexpr int kLag = kHW > 1 ? 1 : 0;          // steps the value product runs behind
  static constexpr int kQRegs = kHW == 1 ? kQ4Steps : 24;   // query operands in registers, the others in LDS
  static constexpr int kQLds = kQ4Steps - kQRegs;
  static constexpr int kQBytes = kQLds > 0 ? kHW * kQLds * 1024 : 16;
  static constexpr int kXBytes = kHW > 1 ? 2 * kWaves * 2048 : 16;   // P of two steps
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
  DMLA_LDS char* q;        // [kHW][kQLds][64 lanes] x 16 bytes
  DMLA_LDS char* p;        // [2][kKP][kHW][2][64 lanes] x 16 bytes
  DMLA_LDS float* stat;    // [kKP][kHeads][2]: references and sums
  DMLA_LDS int* flag;      // [kWaves]
};

// One segment: the tiles [t0, t1) of a sequence.
template <int kHW>
__device__ __forceinline__ void run_segment(const Q4DecodeParams& p, const Segment& sg, const Lds& lds, int head0) {
  using S = Shape<kHW>;
  constexpr int kKP = S::kKP, kCols = S::kCols;
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int hw = wave % kHW, kp = wave / kHW;
  const int n_steps = (sg.t1 - sg.t0 + kKP - 1) / kKP;
  bool bad_page = false;

  // Pages of this wave's tiles, 64 at a time in a register (lane i: page page0 + i).
  int page0 = 0, pages = 0;
  auto fetch_pages = [&](int from) {
    page0 = uniform(from);
    const int i = page0 + fresh_lane_id();
    pages = i < (sg.t1 + 1) / 2 ? p.block_table[sg.b * p.bt_sb + i] : 0;
    asm volatile("" : "+v"(pages));   // waited for here, in the rare branch, and not by every reader
  };
  const unsigned ring_addr = lds_addr(lds.ring);
  // LDS address of this wave's tile of step s, a scalar that the compiler cannot see through: it would keep
  // an address per read up to date in the loop otherwise.
  auto tile_addr = [&](int s) {
    unsigned a = ring_addr + (unsigned)((s % S::kSlots) * S::kSlotBytes + kp * kTileBytes);
    asm("" : "+s"(a));
    return a;
  };
  // Address lane_off + add as one register; the reads through it carry their constant parts as offsets.
  auto lds_at = [&](int lane_off, unsigned add) {
    unsigned a;
    asm("v_add_u32 %0, %1, %2" : "=v"(a) : "v"(lane_off), "s"(add));
    return reinterpret_cast<const DMLA_LDS char*>(static_cast<uintptr_t>(a));
  };
  // This wave's share of the copies of step s's tile kp: pieces hw, hw + kHW, ...
  auto copy_step = [&](int s) {
    const int t = min(sg.t0 + s * kKP + kp, sg.t1 - 1);   // past the end: the last tile, all masked
    if (t / 2 - page0 >= 64) fetch_pages(page0 + 64);
    int page = __builtin_amdgcn_readlane(pages, uniform((t / 2 - page0) & 63));
    const bool bad = page < 0 || page >= p.num_pages;
    bad_page = bad_page || bad;
    page = bad ? 0 : page;
    const char* src = p.kv + page * p.kv_sp + (t & 1) * kTileBytes;
    const unsigned dst = tile_addr(s);
    const int valid = sg.ctx - t * kTile;
    const int ln = fresh_lane_id();   // nothing of this is kept across the loop
#pragma unroll
    for (int i = 0; i < (kCopies + kHW - 1) / kHW; ++i) {
      const int k = i * kHW + hw;
      if (k >= kCopies) continue;
      const int c = k * 64 + ln;
      unsigned off = 16u * c;
      if (valid < kTile) {   // rows past the sequence's end re-read the tile's first row: finite data, masked below
        const int row = c / kQ4Chunks;
        off = row < valid ? off : 16u * (c - row * kQ4Chunks);
      }
      if (k < kCopies - 1 || ln < 32) dma16(src, off, dst + k * 1024);
    }
  };
  // Copies run kAhead steps ahead: at step s the slot of step s - 1 - kLag is refilled.
  constexpr int kAhead = S::kSlots - 1 - S::kLag;
  auto start_copies = [&]() {
    fetch_pages(sg.t0 / 2);
    for (int s = 0; s < kAhead && s < n_steps; ++s) copy_step(s);
  };
  start_copies();

  bf16x8 q[S::kQRegs];
  DMLA_LDS char* q_lds = lds.q + hw * S::kQLds * 1024 + lane * 16;
  {
    const bf16* src = p.q + sg.b * p.q_sb + min(head0 + hw * 32 + l32, p.H - 1) * p.q_sh;
#pragma unroll
    for (int c = 0; c < kQ4Steps; ++c) {
      const bf16x8 v = q4_query_operand(src, hl, c);
      if (c < S::kQRegs) q[c] = v;
      else *reinterpret_cast<DMLA_LDS bf16x8*>(q_lds + (c - S::kQRegs) * 1024) = v;   // the same from every kp
    }
  }
  auto query_lds = [&](int c) {
    return lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(q_lds + (c - S::kQRegs) * 1024));
  };

  f32x16 acc[kHW][kCols];   // O^T of 32 heads and 32 columns: row m is column (512 / kHW) hw + kCols m + j
  float mref = kNegInf, mtrue = kNegInf, lsum = 0.f;   // reference, largest score seen, sum
  bf16x8 pv[2];             // P of the wave's own heads, 16 keys each

  // S^T[key 8 (i / 4) + 4 hl + i % 4][head l32] of a tile.
  // before_end runs while the last steps are in the matrix core.
  auto scores = [&](int s, int t, auto before_end) -> f32x16 {
    const unsigned tile = tile_addr(s);
    const DMLA_LDS char* codes = lds_at(l32 * kQ4RowBytes + 128 * hl, tile);
    const DMLA_LDS char* rope = lds_at(l32 * kQ4RowBytes + kQ4RopeOff + 16 * hl, tile);
    // Blocks of four steps: codes are read two blocks ahead and converted one block ahead, a quarter of
    // the next block's beside each MFMA; the queries kept in LDS are read one block ahead.
    constexpr int kBlocks = kQ4LatentSteps / 4;
    f32x16 x;
    u32x4 w[3];
    bf16x8 k[2][4], qx[2][4];
    const u32x2 scales = *reinterpret_cast<const DMLA_LDS u32x2*>(lds_at(l32 * kQ4RowBytes + kQ4ScaleOff + 8 * hl, tile));
    auto codes_of = [&](int a) { return *reinterpret_cast<const DMLA_LDS u32x4*>(codes + 16 * a); };
    w[0] = codes_of(0);
    w[1] = codes_of(1);
    auto fetch_queries = [&](int a) {
      if (4 * a >= S::kQRegs && a <= kBlocks) {
#pragma unroll
        for (int j = 0; j < 4; ++j) qx[a & 1][j] = query_lds(4 * a + j);
      }
    };
    auto query = [&](int a, int j) { return 4 * a < S::kQRegs ? q[4 * a < S::kQRegs ? 4 * a + j : 0] : qx[a & 1][j]; };
    {
      const float sc = q4_key_scale<0>(scales);
#pragma unroll
      for (int j = 0; j < 4; ++j) k[0][j] = q4_octet(w[0][j], sc);
    }
    fetch_queries(0);
    in_order();
    auto block = [&](auto a_tag) {
      constexpr int a = decltype(a_tag)::value;
      if constexpr (a + 2 < kBlocks) w[(a + 2) % 3] = codes_of(a + 2);
      fetch_queries(a + 1);
      float sc = 0.f;
      if constexpr (a + 1 < kBlocks) {
        sc = q4_key_scale<a + 1>(scales);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) k[(a + 1) & 1][j] = lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(rope + 32 * j));
      }
      in_order();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (a == 0 && j == 0) score_step<true>(x, k[0][0], query(0, 0));
        else score_step<false>(x, k[a & 1][j], query(a, j));
        if constexpr (a + 1 < kBlocks) k[(a + 1) & 1][j] = q4_octet(w[(a + 1) % 3][j], sc);
        in_order();
      }
    };
    static_for<kBlocks>(block);
    before_end();
    in_order();
#pragma unroll
    for (int j = 0; j < 4; ++j) score_step<false>(x, k[kBlocks & 1][j], query(kBlocks, j));
    in_order();
    score_done(x);
    const int left = t < sg.t1 ? sg.ctx - t * kTile : 0;   // keys of the tile
    if (left < kTile) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 8 * (i >> 2) + 4 * hl + (i & 3) < left ? x[i] : kNegInf;
    }
    return x;
  };
  auto tile_max = [&](const f32x16& x) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    return half_max(mx) * p.scale_log2;   // scale > 0
  };
  // The softmax of a tile in kPieces pieces, which the value product of another tile takes between its
  // MFMAs: the maximum, then an element at a time.
  constexpr int kPieces = 21;
  float mx_part[4];
  float ms = 0.f;
  auto softmax_piece = [&](const f32x16& x, auto i_tag) {
    constexpr int i = decltype(i_tag)::value;
    if constexpr (i < 4) {
      mx_part[i] = fmaxf(fmaxf(x[4 * i], x[4 * i + 1]), fmaxf(x[4 * i + 2], x[4 * i + 3]));
    } else if constexpr (i == 4) {
      const float mx = half_max(fmaxf(fmaxf(mx_part[0], mx_part[1]), fmaxf(mx_part[2], mx_part[3])));
      mtrue = fmaxf(mtrue, mx * p.scale_log2);   // scale > 0
      ms = mref == kNegInf ? 0.f : mref;
    } else if constexpr (i < kPieces) {
      constexpr int e = i - 5;
      const float v = fast_exp2(__builtin_fmaf(x[e], p.scale_log2, -ms));
      lsum += v;
      pv[e >> 3][e & 7] = (bf16)v;
    }
  };
  auto softmax = [&](const f32x16& x) {
    static_for<kPieces>([&](auto i) { softmax_piece(x, i); });
  };

  // O^T += V^T P of step s's tile, in groups of a column pair: while a group's MFMAs run, the next group's
  // codes are converted and between(i) is called after MFMA i, i = 0 .. 31.
  constexpr int kWords = kCols >= 8 ? kCols / 8 : 1;   // words of codes per key
  constexpr int kPairs = kCols / 2;                    // groups per 16 keys
  struct Codes {
    unsigned c[8][kWords];
    float s[8];
    bf16x8 p[kHW];
  };
  Codes cv[2];
  // Codes, scales and probabilities of the keys from 16 u on; read_p(n, u): P of head block n.
  auto read_codes = [&](int s, int u, auto read_p) {
    const unsigned tile = tile_addr(s);
    const DMLA_LDS char* codes = lds_at(4 * hl * kQ4RowBytes + (256 / kHW) * hw + (kCols / 2) * l32, tile);
    const DMLA_LDS char* scales = lds_at(4 * hl * kQ4RowBytes + kQ4ScaleOff + (16 / kHW) * hw + l32 / (2 * kHW), tile);
#pragma unroll
    for (int j = 0; j < 8; ++j) {   // the keys of the lane's scores
      const int row = (16 * u + 8 * (j >> 2) + (j & 3)) * kQ4RowBytes;
      const DMLA_LDS char* at = codes + row;
      if constexpr (kCols == 16) {
        const u32x2 w = *reinterpret_cast<const DMLA_LDS u32x2*>(at);
        cv[u].c[j][0] = w[0];
        cv[u].c[j][1] = w[1];
      } else if constexpr (kCols == 8) {
        cv[u].c[j][0] = *reinterpret_cast<const DMLA_LDS unsigned*>(at);
      } else {
        cv[u].c[j][0] = *reinterpret_cast<const DMLA_LDS uint16_t*>(at);
      }
      cv[u].s[j] = q4_scale(*reinterpret_cast<const DMLA_LDS uint8_t*>(scales + row));
    }
#pragma unroll
    for (int n = 0; n < kHW; ++n) cv[u].p[n] = read_p(n, u);
  };
  u32x4 even[2], odd[2];   // operands of two groups
  // Keys 2 r and 2 r + 1 of group gi's operands.
  auto convert = [&](auto g_tag, int r) {
    constexpr int gi = decltype(g_tag)::value, u = gi / kPairs, cp = gi % kPairs;
    const unsigned a = __builtin_bit_cast(unsigned, q4_pair<cp % 4>(cv[u].c[2 * r][cp / 4], cv[u].s[2 * r]));
    const unsigned b = __builtin_bit_cast(unsigned, q4_pair<cp % 4>(cv[u].c[2 * r + 1][cp / 4], cv[u].s[2 * r + 1]));
    even[gi & 1][r] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    odd[gi & 1][r] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  };
  auto values = [&](int s, auto read_p, auto between) {
#pragma unroll
    for (int r = 0; r < 4; ++r) convert(std::integral_constant<int, 0>{}, r);
    read_codes(s, 1, read_p);
    in_order();
    static_for<2 * kPairs>([&](auto g_tag) {
      constexpr int gi = decltype(g_tag)::value, u = gi / kPairs, cp = gi % kPairs;
      static_for<2 * kHW>([&](auto i_tag) {
        constexpr int i = decltype(i_tag)::value, n = i / 2, j = 2 * cp + (i & 1);
        acc[n][j] = mfma32_bf16(__builtin_bit_cast(bf16x8, (i & 1) ? odd[gi & 1] : even[gi & 1]), cv[u].p[n], acc[n][j]);
        if constexpr (gi + 1 < 2 * kPairs) {   // four quarters over the group's MFMAs
          if constexpr (kHW == 4) {
            if constexpr (i % 2 == 0) convert(std::integral_constant<int, gi + 1>{}, i / 2);
          } else if constexpr (kHW == 2) {
            convert(std::integral_constant<int, gi + 1>{}, i);
          } else {
            convert(std::integral_constant<int, gi + 1>{}, 2 * i);
            convert(std::integral_constant<int, gi + 1>{}, 2 * i + 1);
          }
        }
        between(std::integral_constant<int, gi * 2 * kHW + i>{});
        in_order();
      });
    });
  };
  // P of step s through LDS, between the waves of a group.
  auto post = [&](int s) {
    const int at = (s & 1) * kWaves + kp * kHW + hw;
#pragma unroll
    for (int u = 0; u < 2; ++u) *reinterpret_cast<DMLA_LDS bf16x8*>(lds.p + (2 * at + u) * 1024 + lane * 16) = pv[u];
  };
  auto shared_p = [&](int s) {
    const unsigned at = (unsigned)(2048 * ((s & 1) * kWaves + kp * kHW));
    const DMLA_LDS char* from = lds_at(lane * 16, lds_addr(lds.p) + at);
    return [from](int n, int u) { return lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(from + 2048 * n + 1024 * u)); };
  };

  auto arrive = [&](int s, bool copy) {
    // This wave's copies of step s have landed; those of the kAhead - 1 steps after it stay in flight.
    constexpr int kFlight = kAhead - 1;
    constexpr int kMost = (kCopies + kHW - 1) / kHW, kLeast = kCopies / kHW;
    if (s + kFlight >= n_steps) wait_vm<0>();   // the last steps have fewer behind them
    else if (hw < kCopies % kHW || kCopies % kHW == 0) wait_vm<kFlight * kMost>();
    else wait_vm<kFlight * kLeast>();
    wait_lds();   // this wave's reads of the slot that is refilled below are done
    if constexpr (kHW > 1) __syncthreads();   // and everybody's; all copies of step s have landed
    if (copy && s + kAhead < n_steps) copy_step(s + kAhead);
  };
  // The reference of a head is its first tile's largest score.  Where scores have climbed more than
  // kHeadroom above it, the segment starts over from the largest that was seen: rare, and the loop holds
  // no rescaling of the outputs.
  for (bool again = false;; again = true) {
    arrive(0, true);
    const f32x16 x0 = scores(0, sg.t0 + kp, [] {});
    mref = again ? mtrue : tile_max(x0);
    lsum = 0.f;
    if constexpr (kHW > 1) {
      softmax(x0);
      post(0);
    }
    // Zeros by the matrix core, a whole accumulator at a time: element by element the compiler would
    // assemble them elsewhere and move them.
#pragma unroll
    for (int n = 0; n < kHW; ++n)
#pragma unroll
      for (int j = 0; j < kCols; ++j) acc[n][j] = mfma32_bf16(bf16x8{}, bf16x8{}, f32x16{});
    wait_vm<0>();   // whatever the compiler has in flight, so that it does not wait for it in the loop
    if constexpr (kHW > 1) {
      // One step more than there are tiles, whose scores are all masked: no branch in the loop.
#pragma nounroll
      for (int s = 1; s <= n_steps; ++s) {
        arrive(s, true);
        const auto read_p = shared_p(s - 1);
        const f32x16 x = scores(s, sg.t0 + s * kKP + kp, [&] { read_codes(s - 1, 0, read_p); });
        values(s - 1, read_p, [&](auto i) { softmax_piece(x, i); });
        post(s);
      }
    } else {
#pragma nounroll
      for (int s = 0; s < n_steps; ++s) {
        arrive(s, s > 0);
        softmax(scores(s, sg.t0 + s * kKP + kp, [] {}));
        const auto own_p = [&](int, int u) { return pv[u]; };
        read_codes(s, 0, own_p);
        values(s, own_p, [](auto) {});
      }
    }
    const bool over = __any(mtrue > mref + kHeadroom);
    if (lane == 0) lds.flag[wave] = over ? 1 : 0;
    wait_vm<0>();
    wait_lds();
    __syncthreads();   // flags posted; the ring and the exchange are free
    const bool repeat = (lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]) != 0;
    __syncthreads();   // flags read
    if (again || !repeat) break;
    start_copies();
  }

  // ---- the segment's output ----
  lsum = half_sum(lsum);
  agpr_settle();
  if (hl == 0) {
    const int at = (kp * S::kHeads + hw * 32 + l32) * 2;
    lds.stat[at] = mref;
    lds.stat[at + 1] = lsum;
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
    for (int k = 0; k < kKP; ++k) top = fmaxf(top, lds.stat[(k * S::kHeads + hd) * 2]);
#pragma unroll
    for (int k = 0; k < kKP; ++k) {
      const float m = lds.stat[(k * S::kHeads + hd) * 2], l = lds.stat[(k * S::kHeads + hd) * 2 + 1];
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
  // A lane holds, for each q = 0..3, 4 kCols neighbouring columns from kCols (8 q + 4 hl) of its wave's
  // 512 / kHW on: value n of them is accumulator n % kCols, register 4 q + n / kCols.
  if constexpr (kKP == 1) {
#pragma unroll
    for (int n = 0; n < kHW; ++n) {
      const int head = head0 + 32 * n + l32;
      if (head >= p.H) continue;
      float top, sum;
      joined(32 * n + l32, top, sum);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      bf16* orow = out_row(head) + (kDv / kHW) * hw;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
        for (int d = 0; d < kCols / 2; ++d) {
          bf16x8 v;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = (bf16)(agpr_read(acc[n][(8 * d + j) % kCols][4 * q4 + (8 * d + j) / kCols]) * inv);
          *reinterpret_cast<bf16x8*>(orow + kCols * (8 * q4 + 4 * hl) + 8 * d) = v;
        }
      if (hl == 0 && hw == n) put_lse(head, top, sum);
    }
  } else {
    // The tile groups' outputs meet in LDS, one q a round (a quarter of the columns of all heads),
    // each group's at the common reference.
    DMLA_LDS float* merge = reinterpret_cast<DMLA_LDS float*>(lds.ring);
    float fac[kHW];
#pragma unroll
    for (int n = 0; n < kHW; ++n) {
      float top, sum;
      joined(32 * n + l32, top, sum);
      const float m = lds.stat[(kp * S::kHeads + 32 * n + l32) * 2];
      fac[n] = m == kNegInf ? 0.f : fast_exp2(m - top);
    }
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
#pragma unroll
      for (int n = 0; n < kHW; ++n) {
        DMLA_LDS float* at = merge + (wave * S::kHeads + 32 * n + l32) * S::kMergeRow + 4 * kCols * hl;
#pragma unroll
        for (int d = 0; d < kCols; ++d) {
          f32x4 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = agpr_read(acc[n][(4 * d + j) % kCols][4 * q4 + (4 * d + j) / kCols]) * fac[n];
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
          const int half = lc / (4 * kCols);
          *reinterpret_cast<bf16x8*>(out_row(head) + (kDv / kHW) * w0 + kCols * (8 * q4 + 4 * half) + lc % (4 * kCols)) = v;
          if (q4 == 0 && cc == 0) put_lse(head, top, sum);
        }
      }
      __syncthreads();   // read out before the next round writes
    }
  }
}

// One workgroup per range (dmla_ranges.h) and head group.
template <int kHW>
__global__ __launch_bounds__(kThreads, 1) void q4_decode_kernel(Q4DecodeParams p) {
  using S = Shape<kHW>;
  __shared__ __attribute__((aligned(1024))) char ring[S::kRingBytes];
  __shared__ __attribute__((aligned(1024))) char q_mem[S::kQBytes];
  __shared__ __attribute__((aligned(1024))) char p_mem[S::kXBytes];
  __shared__ __attribute__((aligned(16))) float stat[2 * kWaves * 32];
  __shared__ __attribute__((aligned(16))) int flag[kWaves];
  __shared__ __attribute__((aligned(16))) RangeLds ranges;
  const Lds lds = {(DMLA_LDS char*)ring, (DMLA_LDS char*)q_mem, (DMLA_LDS char*)p_mem, (DMLA_LDS float*)stat, (DMLA_LDS int*)flag};
  // The head groups of a range run 8 ids apart, on one XCD: the second read of its pages hits that L2.
  const int id = blockIdx.x;
  const int hg = (id / 8) % p.head_groups;
  const int r = (id / (8 * p.head_groups)) * 8 + id % 8;
  if (r >= p.n_ranges) return;
  for_each_segment<kTile, S::kSegCost>(
      p.seqlens, p.B, p.max_pages * kPage, p.n_ranges, p.min_width, r, ranges,
      [&](int b, int t0, int t1, int ctx, int nsplit) {
        run_segment<kHW>(p, Segment{b, t0, t1, ctx, nsplit, r + b}, lds, hg * S::kHeads);
      },
      [&](int b, int first_range, int nsplit) {
        if (hg != 0) return;
        p.num_splits[b] = nsplit;
        p.split_base[b] = first_range + b;
      });
}

int wg_heads(int64_t H) { return H <= 32 ? 32 : H <= 64 ? 64 : 128; }
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
    case 32: p.min_width = 32; hipLaunchKernelGGL(q4_decode_kernel<1>, grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
    case 64: p.min_width = 16; hipLaunchKernelGGL(q4_decode_kernel<2>, grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
    default: p.min_width = 8; hipLaunchKernelGGL(q4_decode_kernel<4>, grid, dim3(kThreads), 0, (hipStream_t)stream, p); break;
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
