// Paged decode over the 4-bit latent cache (row format: dmla_q4.h): one query token per sequence.  This
// kernel takes up to 64 heads, and small batches of any; dmla_q4_wide.hip the others.
//
//   s_ht = scale q_h . k_t,  o_h = sum_t softmax(s_h)_t k_t[:512],  k_t = code x scale (exact)
//
// MI355X design:
//  * Key tiles of 32 tokens are copied global -> LDS as they lie in the cache (400 bytes per token) into
//    a ring of slots and become bf16 on the way to the MFMA, two values per instruction, scale included.
//    (The scaled MFMA would take the codes as they are, but it sums the products of an instruction in
//    fixed point, some 14 bits below the largest: scores 2^-14 of their terms off, where bf16 products
//    are exact and sum in fp32.)
//  * The score product has the keys as its rows, so a lane ends with 16 keys' scores of one head, which are, 8 by 8,
//    two operands of the value product's probabilities as it takes them.
//  * Probabilities enter the value product rounded to bf16 (2^-8 of each at most, of no common sign), sums stay in fp32.
//    The values need bf16's exponents, so fp16 probabilities would not do, and two bf16 halves of each would
//    double that product: 100 MFMAs a tile for 68, in the wide kernel of a loop that the matrix units bound.
//  * The value product needs keys along the MFMA's k.  A lane reads the codes of 16 neighbouring columns of
//    8 keys, converts them and joins equal columns of two keys with a byte permute: 8 instructions per MFMA
//    operand.  MFMA number j then holds column 16 m + j in row m.
//  * Four waves per workgroup, one per SIMD with 512 registers.  A wave computes the scores, the softmax and
//    the outputs (256 registers) of 32 heads for tiles of its own, without a barrier; the waves meet in LDS
//    at the end of a segment.
//  * The softmax reference of a head is its largest score in the wave's first tile; P may grow to 2^32
//    past it (bf16 keeps its relative precision whatever the size, sums stay in fp32), and a segment
//    whose scores climb further starts over from their exact maximum.  So does one whose scores climb at all
//    where the latents reach 2^60, since 2^32 times those might leave fp32.
//  * Sequences are cut over the chip's workgroups by weight (dmla_ranges.h); sequences in several parts
//    are merged by the split-KV combine, from fp32.  Parts in bf16 saved 10 of 104 us at 64 sequences x 128 heads and 4
//    of 74 at 16 heads, and cost precision: outputs 1.5 times as far from 64 bits as the rounding of an exact result
//    (with P's rounding beside it), where fp32 parts leave 1.2 times.
//
// Bound: the cache's bytes, read at some 4.3 TB/s from scattered pages of 25.6 KB (a plain reduction over such a
// pool reads 3.9), and close to them one wave's instruction issue at the clock that power leaves: an instruction takes
// it 4 to 5 cycles whatever its kind, and a tile 750 of them.  With all pages scattered over 420 MB a tile of four
// waves' takes 0.79 us, with all-zero data 0.65 (5.0 TB/s).  Measured: 64 sequences of 2048 to 16384 tokens (229 MB) x
// 16 heads 75 us with the combine, 3.1 TB/s; one of 5000 x 128 heads 26 us, latency; 256 workgroups take 0.61 us a tile
// and 15 us besides while the pages lie in the last cache.
#include <algorithm>

#include "dmla_host.h"
#include "dmla_q4_decode.h"

namespace dmla {
namespace {

constexpr int kDqk = kQ4Dqk, kDv = kQ4Dv, kPage = kQ4Page, kTile = kQ4Tile, kTileBytes = kQ4TileBytes;
constexpr int kCopies = (kTileBytes + 1023) / 1024;  // wave copies of a tile, the last one half
constexpr int kWaves = kQ4Waves, kThreads = kQ4Threads;
constexpr int kHeads = 32;                     // heads of a workgroup
constexpr int kSlotBytes = kWaves * kTileBytes, kSlots = 3;
constexpr int kRingBytes = kSlots * kSlotBytes;
constexpr int kMergeRow = 128 + 4;             // floats, padded against bank conflicts
static_assert(kWaves * kHeads * kMergeRow * 4 <= kRingBytes, "the merge reuses the ring");

struct Lds {
  DMLA_LDS char* ring;
  DMLA_LDS float* stat;    // [kWaves][kHeads][2]: references and sums
  DMLA_LDS int* flag;      // [kWaves]
};

// One segment: the tiles [t0, t1) of a sequence.
__device__ __forceinline__ void run_segment(const Q4DecodeParams& p, const Q4Segment& sg, const Lds& lds, int head0) {
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int n_steps = (sg.t1 - sg.t0 + kWaves - 1) / kWaves;
  const unsigned ring_addr = lds_addr(lds.ring) + wave * kTileBytes;
  // LDS address of this wave's tile of step s, a scalar that the compiler cannot see through.
  auto tile_addr = [&](int s) {
    unsigned a = ring_addr + (unsigned)((s % kSlots) * kSlotBytes);
    asm("" : "+s"(a));
    return a;
  };
  auto lds_at = [&](int lane_off, unsigned add) { return lds_ptr<const char>(lds_sum(lane_off, add)); };
  Q4Pages pages;
  auto copy_step = [&](int s) {
    const int t = min(sg.t0 + s * kWaves + wave, sg.t1 - 1);   // past the end: the last tile, all masked
    const char* src = pages.tile(p, sg, t);
    const unsigned dst = tile_addr(s);
    const int valid = sg.ctx - t * kTile;
    const int ln = fresh_lane_id();   // nothing of this is kept across the loop
#pragma unroll
    for (int k = 0; k < kCopies; ++k) {
      const int c = k * 64 + ln;
      unsigned off = 16u * c;
      if (valid < kTile) {   // rows past the sequence's end re-read the tile's first row: finite data, masked below
        const int row = c / kQ4Chunks;
        off = row < valid ? off : 16u * (c - row * kQ4Chunks);
      }
      if (k < kCopies - 1 || ln < 32) dma16(src, off, dst + k * 1024);
    }
  };
  // Copies run kAhead steps ahead: at step s the slot of step s - 1 is refilled.
  constexpr int kAhead = kSlots - 1;
  auto start_copies = [&]() {
    pages.fetch(p, sg, sg.t0 / 2);
    for (int s = 0; s < kAhead && s < n_steps; ++s) copy_step(s);
  };
  start_copies();

  // Queries through the slot that no copy has reached yet, 8 rows x 128 bytes a copy: as operands they would be
  // 32 rows x 32 bytes a load, four times over.
  static_assert(kSlots - 1 >= kAhead && 36 * 1024 <= kSlotBytes, "the last slot is free");
  bf16x8 q[kQ4Steps];
  {
    const unsigned stage = lds_addr(lds.ring) + (kSlots - 1) * kSlotBytes;
    const int ln = fresh_lane_id();
    const int head = min(head0 + 8 * wave + (ln >> 3), p.H - 1);
    const bf16* src = p.q + sg.b * p.q_sb + head * p.q_sh + 8 * ((ln & 7) ^ (ln >> 3));
#pragma unroll
    for (int d = 0; d < 9; ++d) dma16_addr(src + 64 * d, stage + (9 * wave + d) * 1024);
    wait_vm<0>();
    __syncthreads();
    const unsigned row = stage + 9 * 1024 * (l32 >> 3) + 128 * (l32 & 7);
#pragma unroll
    for (int c = 0; c < kQ4Steps; ++c) {
      const int u = q4_operand_unit(hl, c);
      q[c] = *lds_ptr<const bf16x8>(row + (c / 4) * 1024 + 16 * ((u & 7) ^ (l32 & 7)));
    }
    wait_lds();
    __syncthreads();
  }

  f32x16 acc[16];           // O^T of 32 heads and 32 columns: row m is column 16 m + j
  float mref = kNegInf, mtrue = kNegInf, lsum = 0.f;   // reference, largest score seen, sum
  bf16x8 pv[2];             // P, 16 keys each
  u16x2 vtop = {0, 0};      // largest scales seen, in the upper bytes

  // S^T[key 8 (i / 4) + 4 hl + i % 4][head l32] of a tile.
  auto scores = [&](int s, int t) -> f32x16 {
    const unsigned tile = tile_addr(s);
    const DMLA_LDS char* codes = lds_at(l32 * kQ4RowBytes + 16 * hl, tile);
    const DMLA_LDS char* rope = lds_at(l32 * kQ4RowBytes + kQ4RopeOff + 16 * hl, tile);
    // Blocks of four steps: codes are read two blocks ahead and converted one block ahead, a quarter of
    // the next block's beside each MFMA.
    constexpr int kBlocks = kQ4LatentSteps / 4;
    f32x16 x;
    u32x4 w[3];
    bf16x8 k[2][4];
    const u32x4 scales = q4_key_scales(lds_at(l32 * kQ4RowBytes, tile), hl);
    auto codes_of = [&](int a) { return *reinterpret_cast<const DMLA_LDS u32x4*>(codes + 32 * a); };
    w[0] = codes_of(0);
    w[1] = codes_of(1);
    {
      const float sc = q4_key_scale<0>(scales);
#pragma unroll
      for (int j = 0; j < 4; ++j) k[0][j] = q4_octet(w[0][j], sc);
    }
    in_order();
    auto block = [&](auto a_tag) {
      constexpr int a = decltype(a_tag)::value;
      if constexpr (a + 2 < kBlocks) w[(a + 2) % 3] = codes_of(a + 2);
      if constexpr (a < 4) vtop = __builtin_elementwise_max(vtop, __builtin_bit_cast(u16x2, scales[a] << 8));   // bytes 0 and 2
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
        if (a == 0 && j == 0) score_step<true>(x, k[0][0], q[0]);
        else score_step<false>(x, k[a & 1][j], q[4 * a + j]);
        if constexpr (a + 1 < kBlocks) k[(a + 1) & 1][j] = q4_octet(w[(a + 1) % 3][j], sc);
        in_order();
      }
    };
    static_for<kBlocks>(block);
#pragma unroll
    for (int j = 0; j < 4; ++j) score_step<false>(x, k[kBlocks & 1][j], q[4 * kBlocks + j]);
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
  auto softmax = [&](const f32x16& x) {
    mtrue = fmaxf(mtrue, tile_max(x));
    const float ms = mref == kNegInf ? 0.f : mref;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float v = fast_exp2(__builtin_fmaf(x[i], p.scale_log2, -ms));
      lsum += v;
      pv[i >> 3][i & 7] = (bf16)v;   // the sum above takes it unrounded
    }
  };

  // O^T += V^T P of step s's tile, in groups of a column pair: while a group's MFMAs run, the next group's
  // codes are converted.
  constexpr int kPairs = 8;   // groups per 16 keys
  u32x2 codes[2][8];
  float scales[2][8];
  // Codes and scales of the keys from 16 u on.
  auto read_codes = [&](int s, int u) {
    const unsigned tile = tile_addr(s);
    const DMLA_LDS char* from = lds_at(4 * hl * kQ4RowBytes + 8 * l32, tile);
    const DMLA_LDS char* sfrom = lds_at(4 * hl * kQ4RowBytes + kQ4ScaleOff + l32 / 2, tile);
#pragma unroll
    for (int j = 0; j < 8; ++j) {   // the keys of the lane's scores
      const int row = (16 * u + 8 * (j >> 2) + (j & 3)) * kQ4RowBytes;
      codes[u][j] = *reinterpret_cast<const DMLA_LDS u32x2*>(from + row);
      scales[u][j] = q4_scale(*reinterpret_cast<const DMLA_LDS uint8_t*>(sfrom + row));
    }
  };
  u32x4 even[2], odd[2];   // operands of two groups
  // Keys 2 r and 2 r + 1 of group gi's operands.
  auto convert = [&](auto g_tag, int r) {
    constexpr int gi = decltype(g_tag)::value, u = gi / kPairs, cp = gi % kPairs;
    const unsigned a = __builtin_bit_cast(unsigned, q4_pair<cp % 4>(codes[u][2 * r][cp / 4], scales[u][2 * r]));
    const unsigned b = __builtin_bit_cast(unsigned, q4_pair<cp % 4>(codes[u][2 * r + 1][cp / 4], scales[u][2 * r + 1]));
    even[gi & 1][r] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    odd[gi & 1][r] = __builtin_amdgcn_perm(b, a, 0x07060302u);
  };
  auto values = [&](int s) {
    read_codes(s, 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) convert(std::integral_constant<int, 0>{}, r);
    read_codes(s, 1);
    in_order();
    static_for<2 * kPairs>([&](auto g_tag) {
      constexpr int gi = decltype(g_tag)::value, u = gi / kPairs, cp = gi % kPairs;
      static_for<2>([&](auto i_tag) {
        constexpr int i = decltype(i_tag)::value;
        acc[2 * cp + i] = mfma32_bf16(__builtin_bit_cast(bf16x8, i ? odd[gi & 1] : even[gi & 1]), pv[u], acc[2 * cp + i]);
        if constexpr (gi + 1 < 2 * kPairs) {   // half of the next group's
          convert(std::integral_constant<int, gi + 1>{}, 2 * i);
          convert(std::integral_constant<int, gi + 1>{}, 2 * i + 1);
        }
        in_order();
      });
    });
  };

  auto arrive = [&](int s, bool copy) {
    // The copies of step s have landed; those of the next step stay in flight, where there is one.
    if (s + kAhead - 1 >= n_steps) wait_vm<0>();
    else wait_vm<(kAhead - 1) * kCopies>();
    wait_lds();   // the reads of the slot that is refilled below are done
    if (copy && s + kAhead < n_steps) copy_step(s + kAhead);
  };
  // The reference of a head is its first tile's largest score.  Where scores have climbed more than
  // kHeadroom above it, the segment starts over from the largest that was seen: rare, and the loop holds
  // no rescaling of the outputs.
  for (bool again = false;; again = true) {
    arrive(0, true);
    const f32x16 x0 = scores(0, sg.t0 + wave);
    mref = again ? mtrue : tile_max(x0);
    lsum = 0.f;
    // Zeros by the matrix core, a whole accumulator at a time: element by element the compiler would
    // assemble them elsewhere and move them.
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = mfma32_bf16(bf16x8{}, bf16x8{}, f32x16{});
    wait_vm<0>();   // whatever the compiler has in flight, so that it does not wait for it in the loop
    // The first tile's scores are computed again: kept across the loop's start, they cost spills in the loop
    // (64 sequences x 16 heads 79 us).
#pragma nounroll
    for (int s = 0; s < n_steps; ++s) {
      arrive(s, s > 0);
      softmax(scores(s, sg.t0 + s * kWaves + wave));
      values(s);
    }
    const int climb = q4_climb(mtrue, mref, max(vtop[0], vtop[1]) >> 8 >= kQ4BigScale + 127);
    if (lane == 0) lds.flag[wave] = climb;
    wait_vm<0>();
    wait_lds();
    __syncthreads();   // flags posted; the ring is free
    const bool repeat = q4_repeat(lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]);
    __syncthreads();   // flags read
    if (again || !repeat) break;
    start_copies();
  }

  // ---- the segment's output ----
  lsum = half_sum(lsum);
  agpr_settle();
  if (hl == 0) {
    lds.stat[(wave * kHeads + l32) * 2] = mref;
    lds.stat[(wave * kHeads + l32) * 2 + 1] = lsum;
  }
  if (lane == 0) lds.flag[wave] = pages.bad ? 1 : 0;
  __syncthreads();
  const float nanv = __builtin_nanf("");
  const bool poison = (lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]) != 0;
  // Reference and sum of a head of the workgroup over the tile groups.
  auto joined = [&](int hd, float& top, float& sum) {
    top = kNegInf;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) top = fmaxf(top, lds.stat[(k * kHeads + hd) * 2]);
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      const float m = lds.stat[(k * kHeads + hd) * 2], l = lds.stat[(k * kHeads + hd) * 2 + 1];
      sum += m == kNegInf ? l : l * fast_exp2(m - top);   // no finite reference: 0, or NaN
    }
    if (poison) sum = nanv;
  };
  auto put_lse = [&](int head, float top, float sum) {
    const float lse = sum == 0.f ? kNegInf : (top + __log2f(sum)) * kLn2;
    if (sg.nsplit > 1) p.part_lse[(int64_t)sg.slot * p.H + head] = lse;
    else if (p.lse != nullptr) p.lse[sg.b * p.H + head] = lse;
  };
  // The waves' outputs meet in LDS, a quarter of the columns a round, each at the common reference.  In round
  // q4 a lane holds the 64 neighbouring columns from 16 (8 q4 + 4 hl) on: column 16 x + j is accumulator j,
  // register 4 q4 + x.
  DMLA_LDS float* merge = reinterpret_cast<DMLA_LDS float*>(lds.ring);
  float top, sum;
  joined(l32, top, sum);
  const float fac = mref == kNegInf ? 0.f : fast_exp2(mref - top);
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4) {
    DMLA_LDS float* at = merge + (wave * kHeads + l32) * kMergeRow + 64 * hl;
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      f32x4 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = agpr_read(acc[(4 * d + j) % 16][4 * q4 + d / 4]) * fac;
      *reinterpret_cast<DMLA_LDS f32x4*>(at + 4 * d) = v;
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < kHeads * 16 / kThreads; ++it) {
      const int item = it * kThreads + threadIdx.x;
      const int hd = item >> 4, cc = (item & 15) * 8;   // head, and 8 of the round's 128 columns
      const int head = head0 + hd;
      joined(hd, top, sum);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      f32x4 v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const DMLA_LDS float* from = merge + (k * kHeads + hd) * kMergeRow + cc;
        v0 += *reinterpret_cast<const DMLA_LDS f32x4*>(from);
        v1 += *reinterpret_cast<const DMLA_LDS f32x4*>(from + 4);
      }
      if (head < p.H) {
        if (sg.nsplit > 1) {   // parts stay in fp32
          float* to = p.part_o + ((int64_t)sg.slot * p.H + head) * kDv + 128 * q4 + cc;
          *reinterpret_cast<f32x4*>(to) = v0 * inv;
          *reinterpret_cast<f32x4*>(to + 4) = v1 * inv;
        } else {
          bf16x8 v;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[j] = (bf16)(v0[j] * inv);
            v[4 + j] = (bf16)(v1[j] * inv);
          }
          *reinterpret_cast<bf16x8*>(p.o + sg.b * p.o_sb + head * p.o_sh + 128 * q4 + cc) = v;
        }
        if (q4 == 0 && cc == 0) put_lse(head, top, sum);
      }
    }
    __syncthreads();   // read out before the next round writes
  }
}

// One workgroup per range (dmla_ranges.h) and head group.
__global__ __launch_bounds__(kThreads, 1) void q4_decode_kernel(Q4DecodeParams p) {
  __shared__ __attribute__((aligned(1024))) char ring[kRingBytes];
  __shared__ __attribute__((aligned(16))) float stat[2 * kWaves * kHeads];
  __shared__ __attribute__((aligned(16))) int flag[kWaves];
  __shared__ __attribute__((aligned(16))) RangeLds ranges;
  const Lds lds = {(DMLA_LDS char*)ring, (DMLA_LDS float*)stat, (DMLA_LDS int*)flag};
  // The head groups of a range run 8 ids apart, on one XCD: the second read of its pages hits that L2.
  const int id = blockIdx.x;
  const int hg = (id / 8) % p.head_groups;
  const int r = (id / (8 * p.head_groups)) * 8 + id % 8;
  if (r >= p.n_ranges) return;
  for_each_segment<kTile, kQ4Cost>(
      p.seqlens, p.B, p.max_pages * kPage, p.n_ranges, p.min_width, r, ranges,
      [&](int b, int t0, int t1, int ctx, int nsplit) {
        run_segment(p, Q4Segment{b, t0, t1, ctx, nsplit, r + b}, lds, hg * kHeads);
      },
      [&](int b, int first_range, int nsplit) {
        if (hg != 0) return;
        p.num_splits[b] = nsplit;
        p.split_base[b] = first_range + b;
      });
}

// Up to 64 heads, workgroups of 32 (two groups of them read a tile twice, the second time from the L2); above, of 128.
// 64 sequences of 8192 tokens, this kernel against the wide one: 71 : 149 us with 16 heads, 76 : 143 with 32, 114 : 143
// with 64, 268 : 147 with 96; 4 sequences 26 : 36, 30 : 37, 35 : 36 and 37 : 37 us.
// Where the block tables hold up to four tiles a CU, latency counts, and more and smaller workgroups win for any
// number of heads: one sequence of 5000 tokens x 128 heads 27 : 31 us, of 16384 36 : 40, 4 of 8192 38.5 : 39.7; one of
// 65536 x 96 heads (eight tiles a CU) 71 : 55.
int wg_heads(int64_t H, int64_t tiles) { return H <= 2 * kHeads || tiles <= 4 * (int64_t)device_cu_count() ? kHeads : 128; }
// Ranges of a call, given the heads of a workgroup.
int64_t q4_ranges(int64_t H, int64_t heads) {
  const int64_t hg = (H + heads - 1) / heads;
  return std::max<int64_t>(1, device_cu_count() / hg);
}

}  // namespace
}  // namespace dmla

using namespace dmla;

static int64_t q4_plan_bytes(int64_t B) { return (B * 8 + 255) / 256 * 256; }

extern "C" int64_t dmla_decode_q4_workspace_bytes(int64_t B, int64_t H) {
  if (B <= 0 || H <= 0 || B > ((int64_t)1 << 20) || H > ((int64_t)1 << 16)) return 0;
  const int64_t most = std::max(q4_ranges(H, wg_heads(H, 0)), q4_ranges(H, wg_heads(H, INT64_MAX)));
  return q4_plan_bytes(B) + (most + B) * H * (int64_t)(kDv * 4 + 4);
}

extern "C" int dmla_decode_paged_q4(const void* q, const void* kv_pool, const int32_t* block_table,
                                    const int32_t* cache_seqlens, void* o, float* lse, int64_t B, int64_t H,
                                    int64_t d_qk, int64_t d_v, int64_t num_pages, int64_t max_pages_per_seq,
                                    int64_t q_sb, int64_t q_sh, int64_t kv_sp, int64_t bt_sb, int64_t o_sb, int64_t o_sh,
                                    float softmax_scale, void* workspace, int64_t workspace_bytes, dmla_stream_t stream) {
  clear_error();
  // (Of an empty call any address does: empty tensors have none.)
  if (B != 0 && H != 0 && (!q || !kv_pool || !block_table || !cache_seqlens || !o))
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
  if (H > ((int64_t)1 << 16) || B > ((int64_t)1 << 20) || max_pages_per_seq > ((int64_t)1 << 24) || num_pages > 0x7fffffff)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_decode_paged_q4: size too large");
  if (B == 0 || H == 0) return DMLA_OK;
  if (num_pages == 0 || max_pages_per_seq == 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: empty page pool or block table");
  const int64_t tiles = max_pages_per_seq * (kPage / kTile);   // of a sequence, at most
  const int heads = wg_heads(H, B * tiles);
  const int64_t R = q4_ranges(H, heads), slots = R + B;
  if (!ranges_fit(B, tiles, heads == kHeads ? kQ4Cost : kQ4WideCost, R))
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_decode_paged_q4: size too large");
  const int64_t need = dmla_decode_q4_workspace_bytes(B, H);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DMLA_ERR_WORKSPACE, "dmla_decode_paged_q4: workspace of %lld bytes needed (got %lld)", (long long)need,
                (long long)workspace_bytes);
  if (!aligned16(workspace)) return fail(DMLA_ERR_INVALID_ARG, "dmla_decode_paged_q4: workspace must be 16-byte aligned");
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
  p.part_o = reinterpret_cast<float*>(ws + q4_plan_bytes(B));
  p.part_lse = p.part_o + slots * H * kDv;
  p.q_sb = q_sb; p.q_sh = q_sh; p.kv_sp = kv_sp; p.bt_sb = bt_sb; p.o_sb = o_sb; p.o_sh = o_sh;
  p.B = (int)B; p.H = (int)H; p.num_pages = (int)num_pages; p.max_pages = (int)max_pages_per_seq;
  p.head_groups = (int)((H + heads - 1) / heads);
  p.n_ranges = (int)R;
  p.scale_log2 = softmax_scale * kLog2e;
  const int grid = (int)((R + 7) / 8 * 8 * p.head_groups);
  // The least work of a workgroup, in tiles: two for each wave.  4 sequences of 8192 tokens x 16 heads, and one of 5000:
  // 6 tiles 27.7 and 23.3 us, 8 tiles 25.8 and 23.5, 10 tiles 26.5 and 25.9, 16 tiles 27.9 and 27.8.  The wide kernel at
  // one of 5000: 3 to 6 tiles 29.6 to 30.2, 8 tiles 41.8.
  if (heads == kHeads) {
    p.min_width = 8;
    hipLaunchKernelGGL(q4_decode_kernel, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, p);
  } else {
    p.min_width = 4;
    launch_q4_wide(p, grid, (hipStream_t)stream);
  }
  const int rc = check_launch("dmla_decode_paged_q4");
  if (rc != DMLA_OK) return rc;
  // Sequences in one part were written above; the others, and the empty ones, come from the combine.
  CombineArgs c = {};
  c.part_o = p.part_o;
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
