// Paged decode over the 4-bit latent cache for more than 64 heads (up to 64, and small batches: dmla_q4_decode.hip,
// which states what is computed).
//
// MI355X design:
//  * One wave per SIMD: the fp32 outputs of 128 heads x 512 columns fill the AGPRs of the four waves, so
//    every wave issues one instruction in 4 to 5 cycles whatever its kind, and a step of 68 MFMAs (32 cycles
//    each) has room for some 480.  Converting the codes in the operands' registers takes 800: 32 heads' scores
//    need every code of the tile in every wave.  Here a tile becomes bf16 once, in LDS, a quarter by each
//    wave (32 conversions and 8 writes a lane), and both products read plain operands: 440 instructions.
//  * Keys lie in LDS as rows of 1024 bytes (latent dims) whose 16-byte units are permuted by key: unit u of
//    row r at u ^ key_swz(r).  The score product reads a unit of 32 rows (ds_read_b128), the value product
//    32 columns of 8 rows transposed (ds_read_b64_tr_b16), the conversion writes two units of 8 rows.  Bank
//    conflicts are a fifth of the LDS cycles, most of them the writes'; without those the time stayed.
//  * Codes and scales are copied global -> LDS by the wave that converts them, four tiles ahead, the rope
//    values straight to where the score product reads them: they are bf16 in the cache.
//  * A wave computes the scores and the softmax of 32 heads (their queries: 144 registers) and the outputs
//    of all 128 heads for 128 columns; probabilities go through LDS.
//  * Step s multiplies scores of tile s and values of tile s - 1 and converts tiles s + 1 and s + 2, with two barriers
//    that stand among MFMAs whose operands are there.
//    (Barriers that also wait for what follows them, and the copies of a whole tile in one place between the two
//    products, had cost 500 of a step's 4000 cycles.)
//  * The softmax reference of a head is its largest score in the segment's first tile; P may grow to 2^32
//    past it (bf16 keeps its relative precision whatever the size, sums stay in fp32), and a segment
//    whose scores climb further, or at all over latents of 2^60 and more, starts over from their exact maximum.
//
// Bound: the matrix units at the clock that they leave.  A tile takes 1.9 us with all CUs at work: 128 heads x 32 keys
// x 1088 x 2 flops, 1.18 PFLOP/s over the chip, what an 8192^3 bf16 library product reaches here (1.2 PFLOP/s); it
// took 2.1 us converted in registers.  Measured: 64 sequences of 1024 to 8192 tokens x 128 heads 104 us, the combine's
// 15 in it (800 TFLOP/s); a segment's start (queries, first pages, first tiles) takes 9 us and its end 5.
#include "dmla_host.h"
#include "dmla_q4_decode.h"

namespace dmla {
namespace {

constexpr int kTile = kQ4Tile, kWaves = kQ4Waves, kThreads = kQ4Threads;
constexpr int kHeads = 128, kHeadBlocks = 4;   // of a workgroup
constexpr int kColBlocks = 4;                  // 32 columns each, of a wave
constexpr int kKeyRow = 1024, kKeyBytes = kTile * kKeyRow, kKeyTiles = 3;
constexpr int kWaveBytes = kKeyTiles * kKeyBytes / kWaves;   // of the keys' memory, before and after the tiles
static_assert(kWaveBytes >= 24 * 1024, "two rounds of queries");
constexpr int kCodeWave = 8 * (256 + 16);      // codes and scales of a wave's 8 rows
constexpr int kCodeBytes = kWaves * kCodeWave, kCodeSlots = 4;
constexpr int kRopeBytes = kTile * 128, kRopeSlots = 4;
constexpr int kProbBytes = kWaves * 2048;      // P of a step
constexpr int kAhead = 4;                      // tiles between a copy's start and its step
constexpr int kCopies = 4;                     // copies of a wave and step

// Unit permutation of row r: 16 consecutive rows differ, and rows r .. r + 3 differ in the upper two bits.
__device__ __forceinline__ int key_swz(int r) { return (r & 3) << 2 | (r >> 2 & 3); }

struct Lds {
  unsigned keys, codes, rope, prob;   // addresses
  DMLA_LDS float* stat;               // [kHeads]: sums
  DMLA_LDS int* flag;                 // [kWaves]
};

__device__ __forceinline__ void run_segment(const Q4DecodeParams& p, const Q4Segment& sg, const Lds& lds, int head0) {
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int n_steps = sg.t1 - sg.t0;

  // ---- copies ----
  // Lane l copies 16 bytes of row 8 wave + l / 8 into place l of each kilobyte.  Which of the row's eight
  // pieces is permuted by row, against bank conflicts of the readers below.
  Q4Pages pages;
  const char* copy_src = nullptr;
  int copy_last = 0;   // last row of the tile that the sequence holds
  auto copy_begin = [&](int s) {
    const int t = min(sg.t0 + s, sg.t1 - 1);   // past the end: the last tile, which nobody counts
    copy_src = pages.tile(p, sg, t);
    copy_last = uniform(min(sg.ctx - t * kTile, kTile) - 1);
  };
  // Rows past the sequence's end are its last row again: finite data, masked below.
  auto copy_codes = [&](int s) {
    const int ln = fresh_lane_id();
    const unsigned off = min(8 * wave + (ln >> 3), copy_last) * kQ4RowBytes + 16 * ((ln & 7) ^ (ln >> 3));
    const unsigned dst = lds.codes + (s % kCodeSlots) * kCodeBytes + wave * kCodeWave;
    dma16(copy_src, off, dst);
    dma16(copy_src + 128, off, dst + 1024);
  };
  auto copy_rest = [&](int s) {
    const int ln = fresh_lane_id();
    const unsigned off = min(8 * wave + (ln >> 3), copy_last) * kQ4RowBytes + 16 * ((ln & 7) ^ (ln >> 3));
    dma16(copy_src + kQ4RopeOff, off, lds.rope + (s % kRopeSlots) * kRopeBytes + wave * 1024);
    const unsigned soff = min(8 * wave + (ln & 7), copy_last) * kQ4RowBytes;
    dma16_first8(copy_src + kQ4ScaleOff, soff, lds.codes + (s % kCodeSlots) * kCodeBytes + wave * kCodeWave + 2048);
  };
  auto copy_step = [&](int s) {
    copy_begin(s);
    copy_codes(s);
    copy_rest(s);
  };
  auto start_copies = [&]() {
    pages.fetch(p, sg, sg.t0 / 2);
    for (int s = 0; s < kAhead; ++s) copy_step(s);
  };

  // ---- queries: 36 operands of 16 dims; operand c holds dims 16 c + 8 hl .. of head l32 ----
  // Read straight into the operands, a load would touch 32 rows for 32 bytes each (3.9 us of a segment).
  // Instead the wave copies 8 rows x 128 bytes at a time into its part of the keys' memory, in two rounds
  // that fit there.
  bf16x8 q[kQ4Steps];
  const unsigned mine = lds.keys + wave * kWaveBytes;
  auto read_queries = [&](auto first_tag, auto n_tag) {
    constexpr int kFirst = decltype(first_tag)::value, kN = decltype(n_tag)::value;   // blocks of 64 dims
    const int ln = fresh_lane_id();
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int head = min(head0 + wave * 32 + 8 * g + (ln >> 3), p.H - 1);
      const bf16* src = p.q + sg.b * p.q_sb + head * p.q_sh + 64 * kFirst + 8 * ((ln & 7) ^ (ln >> 3));
#pragma unroll
      for (int i = 0; i < kN; ++i) dma16_addr(src + 64 * i, mine + (kN * g + i) * 1024);
    }
  };
  auto take_queries = [&](auto first_tag, auto n_tag) {
    constexpr int kFirst = decltype(first_tag)::value, kN = decltype(n_tag)::value;
    const unsigned a = lds_sum(kN * 1024 * (l32 >> 3) + 128 * (l32 & 7) + 16 * (hl ^ (l32 & 7)), mine);
#pragma unroll
    for (int c = 0; c < 4 * kN; ++c) q[4 * kFirst + c] = *lds_ptr<const bf16x8>((a ^ (32 * (c & 3))) + 1024 * (c >> 2));
  };
  using std::integral_constant;
  read_queries(integral_constant<int, 0>{}, integral_constant<int, 6>{});
  start_copies();
  wait_vm<kAhead * kCopies>();
  take_queries(integral_constant<int, 0>{}, integral_constant<int, 6>{});
  wait_lds();
  read_queries(integral_constant<int, 6>{}, integral_constant<int, 3>{});
  wait_vm<0>();
  take_queries(integral_constant<int, 6>{}, integral_constant<int, 3>{});
  wait_lds();
  __syncthreads();   // the keys' memory is free

  f32x16 acc[kHeadBlocks][kColBlocks];   // O^T: register i is column 128 wave + 32 j + 16 hl + i of head l32
  float mref = kNegInf, mtrue = kNegInf, lsum = 0.f;   // reference, largest score seen, sum
  bf16x8 pv[2];             // P of the wave's own heads, 16 keys each

  // A barrier that waits for nothing else: what it orders has been waited for.
  auto barrier = [] {
    in_order();
    asm volatile("s_barrier" ::: "memory");
    in_order();
  };
  auto opaque = [](unsigned a) {
    asm("" : "+s"(a));
    return a;
  };

  // ---- conversion of a tile, this wave's rows: lane l has row 8 wave + l % 8 and the scale blocks l / 8 and
  // 8 + l / 8 of it ----
  struct {
    u32x4 w[2];
    float sc[2];
    unsigned to;
  } cv;
  float vtop = 0.f;   // largest scale of the converted rows
  auto convert_begin = [&](int s, unsigned tile) {
    const int r = lane & 7, c = lane >> 3, row = 8 * wave + r;
    const unsigned from = opaque(lds.codes + (unsigned)(s % kCodeSlots) * kCodeBytes + wave * kCodeWave);
    const unsigned a = lds_sum(128 * r + 16 * (c ^ r), from), b = lds_sum(2048 + 16 * r + c, from);
    cv.w[0] = *lds_ptr<const u32x4>(a);
    cv.w[1] = *lds_ptr<const u32x4>(a + 1024);
    cv.sc[0] = q4_scale(*lds_ptr<const uint8_t>(b));
    cv.sc[1] = q4_scale(*lds_ptr<const uint8_t>(b + 8));
    cv.to = lds_sum(kKeyRow * row + 16 * ((4 * c) ^ key_swz(row)), opaque(tile));
  };
  auto convert_octet = [&](int i) {   // i = 0 .. 7
    *lds_ptr<bf16x8>((cv.to ^ (16 * (i & 3))) + 512 * (i >> 2)) = q4_octet(cv.w[i >> 2][i & 3], cv.sc[i >> 2]);
  };

  // ---- scores: S^T[key 8 (i / 4) + 4 hl + i % 4][head l32] of step s's tile ----
  bf16x8 rope[4];
  auto read_rope = [&](int s) {
    const unsigned a = lds_sum(128 * l32 + 16 * (hl ^ (l32 & 7)), opaque(lds.rope + (unsigned)(s % kRopeSlots) * kRopeBytes));
#pragma unroll
    for (int c = 0; c < 4; ++c) rope[c] = *lds_ptr<const bf16x8>(a ^ (32 * c));
  };
  constexpr int kDepth = 6;   // operands in flight
  unsigned key_addr = 0;
  bf16x8 k[kDepth];
  auto read_key = [&](int c) { k[c % kDepth] = *lds_ptr<const bf16x8>((key_addr ^ (32 * (c & 7))) + 256 * (c >> 3)); };
  auto scores_begin = [&](unsigned tile) { key_addr = lds_sum(kKeyRow * l32 + 16 * (hl ^ key_swz(l32)), opaque(tile)); };
  // After read_rope(s), scores_begin(tile) and the first kDepth reads; beside(m) runs after MFMA m = 0 .. 35.
  // The result may be read after score_done or two more MFMAs.
  auto scores = [&](auto beside) -> f32x16 {
    f32x16 x;
    static_for<kQ4Steps>([&](auto m_tag) {
      constexpr int m = decltype(m_tag)::value, c = m - 4;
      if constexpr (m < 4) score_step<m == 0>(x, rope[m], q[32 + m]);
      else score_step<false>(x, k[c % kDepth], q[c]);
      if constexpr (m >= 4 && c + kDepth < kQ4LatentSteps) read_key(c + kDepth);
      beside(m_tag);
      in_order();
    });
    return x;
  };
  auto mask = [&](f32x16& x, int s) {
    const int left = sg.ctx - (sg.t0 + s) * kTile;   // keys of the tile
    if (left < kTile) {
      asm volatile("" : "+v"(x));   // rare: a branch
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 8 * (i >> 2) + 4 * hl + (i & 3) < left ? x[i] : kNegInf;
    }
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
  // P through LDS, between the waves.
  auto post = [&] {
    const unsigned at = lds_sum(16 * lane, opaque(lds.prob + wave * 2048));
#pragma unroll
    for (int u = 0; u < 2; ++u) *lds_ptr<bf16x8>(at + 1024 * u) = pv[u];
  };

  // ---- values: O^T += V^T P of a tile, in groups g of 16 keys (u = g / 4) and 32 columns (j = g % 4) ----
  // Row m of the operand is column 4 (m / 8) + 16 (m / 4 % 2) + m % 4 of the block: a lane then ends with 16
  // neighbouring columns.
  bf16x8 prob[2][kHeadBlocks], val[3];
  unsigned val_addr = 0, prob_addr = 0;
  auto values_begin = [&](unsigned tile) {
    const int r = (lane & 15) >> 2, g = lane >> 4 & 1;
    val_addr = lds_sum(kKeyRow * (4 * hl + r) + 256 * wave + 16 * (4 * r | ((g + 2 * (lane & 1)) ^ hl)) + 8 * ((lane & 3) >> 1),
                       opaque(tile));
    prob_addr = lds_sum(16 * lane, lds.prob);
  };
  auto read_prob = [&](int u, int n) { prob[u][n] = *lds_ptr<const bf16x8>(prob_addr + 2048 * n + 1024 * u); };
  auto read_values = [&](int g) {
    const unsigned a = val_addr ^ (64 * (g % 4));
    const int rows = 16 * kKeyRow * (g / 4);
    val[g % 3] = concat(lds_read_tr16(lds_ptr<const bf16x4>(a + rows)),
                        lds_read_tr16(lds_ptr<const bf16x4>((a ^ 32) + rows + 8 * kKeyRow)));
  };
  // After values_begin(tile), the probabilities of the first 16 keys and the values of groups 0 and 1;
  // beside(i) runs after MFMA i = 0 .. 31.
  auto values = [&](auto beside) {
    static_for<32>([&](auto i_tag) {
      constexpr int i = decltype(i_tag)::value, g = i / 4, n = i % 4, u = g / 4;
      acc[n][g % 4] = mfma32_bf16(val[g % 3], prob[u][n], acc[n][g % 4]);
      if constexpr (n == 0 && g + 2 < 8) read_values(g + 2);
      if constexpr (n == 2 && g < 4) read_prob(1, g);
      beside(i_tag);
      in_order();
    });
  };

  // The reference of a head is its first tile's largest score.  Where scores have climbed more than
  // kQ4Headroom above it, the segment starts over from the largest that was seen: rare, and the loop holds
  // no rescaling of the outputs.
  for (bool again = false;; again = true) {
    wait_vm<0>();
    unsigned prev = lds.keys, cur = lds.keys + kKeyBytes, next = lds.keys + 2 * kKeyBytes;   // tiles s - 1, s, s + 1
    auto convert = [&](int s, unsigned tile) {
      convert_begin(s, tile);
#pragma unroll
      for (int i = 0; i < 8; ++i) convert_octet(i);
      vtop = fmaxf(vtop, fmaxf(cv.sc[0], cv.sc[1]));
    };
    convert(0, prev);
    convert(1, cur);
    wait_lds();
    __syncthreads();   // converted, and the rope values of tiles 0 to 3 landed
    read_rope(0);
    scores_begin(prev);
#pragma unroll
    for (int c = 0; c < kDepth; ++c) read_key(c);
    f32x16 x0 = scores([](auto) {});
    score_done(x0);
    mask(x0, 0);
    mref = again ? mtrue : tile_max(x0);
    lsum = 0.f;
    static_for<kPieces>([&](auto i) { softmax_piece(x0, i); });
    post();
    wait_lds();
    __syncthreads();   // everybody has read rope 0
    copy_step(kAhead);
    // Zeros by the matrix core, a whole accumulator at a time: element by element the compiler would
    // assemble them elsewhere and move them.
#pragma unroll
    for (int n = 0; n < kHeadBlocks; ++n)
#pragma unroll
      for (int j = 0; j < kColBlocks; ++j) acc[n][j] = mfma32_bf16(bf16x8{}, bf16x8{}, f32x16{});
    convert_begin(2, next);
    read_rope(1);
    scores_begin(cur);
#pragma unroll
    for (int c = 0; c < kDepth; ++c) read_key(c);
    // Step s: scores of tile s, with the rest of the conversion of tile s + 1; barrier A; values of tile s - 1,
    // with the softmax of tile s; barrier B; the start of both conversion and scores of the next step.  A
    // stands where tile s + 1 is written and P of step s - 1 posted, B where tile s - 1 has been read.  Both
    // stand among MFMAs whose operands are there, and what they guard is read a few MFMAs ahead of its use.
#pragma nounroll
    for (int s = 1; s < n_steps; ++s) {
      f32x16 x = scores([&](auto m_tag) {
        constexpr int m = decltype(m_tag)::value;
        if constexpr (m < 16 && m % 2 == 0) convert_octet(m / 2);
        if constexpr (m == 16) vtop = fmaxf(vtop, fmaxf(cv.sc[0], cv.sc[1]));
        if constexpr (m == 22) {
          wait_lds<5>();   // the octets are written; reads of later keys may be on their way
          barrier();           // A
        }
        if constexpr (m == 23) {
          values_begin(prev);
          copy_begin(s + kAhead);
        }
        if constexpr (m >= 24 && m < 28) read_prob(0, m - 24);
        if constexpr (m == 26) copy_codes(s + kAhead);
        if constexpr (m == 28) copy_rest(s + kAhead);
        if constexpr (m >= 30 && m % 2 == 0 && m < 34) read_values((m - 30) / 2);
      });
      values([&](auto i_tag) {
        constexpr int i = decltype(i_tag)::value;
        if constexpr (i == 2) {
          asm("s_nop 7" : "+v"(x));
          mask(x, s);
        } else if constexpr (i > 2 && i - 3 < kPieces) {
          softmax_piece(x, std::integral_constant<int, i - 3>{});
        } else if constexpr (i == 24) {
          wait_vm<2 * kCopies>();   // this wave's copies of tile s + 2; those of two tiles more may be on their way
          wait_lds();               // the values of tile s - 1
          barrier();                // B
        } else if constexpr (i == 25) {
          post();
        } else if constexpr (i == 26) {
          convert_begin(s + 2, prev);
        } else if constexpr (i == 27) {
          read_rope(s + 1);
        } else if constexpr (i == 28) {
          scores_begin(next);
        } else if constexpr (i > 28) {
          read_key(2 * (i - 29));
          read_key(2 * (i - 29) + 1);
        }
      });
      const unsigned t = prev;
      prev = cur;
      cur = next;
      next = t;
    }
    // The values of the last tile.
    wait_lds();
    __syncthreads();   // its P is posted
    values_begin(prev);
#pragma unroll
    for (int n = 0; n < kHeadBlocks; ++n) read_prob(0, n);
    read_values(0);
    read_values(1);
    values([](auto) {});
    const int climb = q4_climb(mtrue, mref, vtop >= q4_scale(kQ4BigScale + 127));
    if (lane == 0) lds.flag[wave] = climb;
    wait_vm<0>();
    wait_lds();
    __syncthreads();   // flags posted; all of the memory is free
    const bool repeat = q4_repeat(lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]);
    __syncthreads();   // flags read
    if (again || !repeat) break;
    start_copies();
  }

  // ---- the segment's output ----
  lsum = half_sum(lsum);
  agpr_settle();
  if (hl == 0) lds.stat[wave * 32 + l32] = lsum;
  if (lane == 0) lds.flag[wave] = pages.bad ? 1 : 0;
  __syncthreads();
  const bool poison = (lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]) != 0;
  if (hl == 0 && head0 + wave * 32 + l32 < p.H) {
    const int head = head0 + wave * 32 + l32;
    const float sum = poison ? __builtin_nanf("") : lsum;
    const float lse = sum == 0.f ? kNegInf : (mref + __log2f(sum)) * kLn2;
    if (sg.nsplit > 1) p.part_lse[(int64_t)sg.slot * p.H + head] = lse;
    else if (p.lse != nullptr) p.lse[sg.b * p.H + head] = lse;
  }
  // Through LDS, 32 heads at a time, so that a store covers whole lines: 256 bytes of each of 4 heads, or of a part 512
  // bytes of each of 2.  16-byte unit u of row r lies at u ^ r.
  const int g = lane >> 4, c = lane & 15;
  const unsigned put = lds_sum(512 * l32 + 16 * ((4 * hl) ^ l32), mine);
  const unsigned get16 = lds_sum(512 * g + 16 * ((2 * c) ^ g), mine);   // 8 columns of row g: this unit and the one beside it
  const unsigned get32 = lds_sum(512 * hl + 16 * (l32 ^ hl), mine);     // 4 columns of row hl
  bf16* out = p.o + sg.b * p.o_sb + (head0 + g) * p.o_sh + 128 * wave + 8 * c;
  float* part = p.part_o + ((int64_t)sg.slot * p.H + head0 + hl) * kQ4Dv + 128 * wave + 4 * l32;
  auto put16 = [&](int r, bf16* to) {   // row 4 r + g
    const f32x4 a = *lds_ptr<const f32x4>((get16 ^ (64 * r)) + 2048 * r), b = *lds_ptr<const f32x4>((get16 ^ (64 * r) ^ 16) + 2048 * r);
    bf16x8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = (bf16)a[i];
      v[4 + i] = (bf16)b[i];
    }
    *reinterpret_cast<bf16x8*>(to) = v;
  };
  auto put32 = [&](int r, float* to) {   // row 2 r + hl
    *reinterpret_cast<f32x4*>(to) = *lds_ptr<const f32x4>((get32 ^ (32 * r)) + 1024 * r);
  };
#pragma unroll
  for (int n = 0; n < kHeadBlocks; ++n) {
    const float sum = poison ? __builtin_nanf("") : lds.stat[32 * n + l32];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < kColBlocks; ++j)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        f32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = agpr_read(acc[n][j][4 * d + i]) * inv;
        *lds_ptr<f32x4>(put ^ (16 * (8 * j + d))) = v;
      }
    const int heads = p.H - head0 - 32 * n;
    if (heads >= 32) {
      if (sg.nsplit == 1) {
#pragma unroll
        for (int r = 0; r < 8; ++r) put16(r, out + (32 * n + 4 * r) * p.o_sh);
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) put32(r, part + (32 * n + 2 * r) * kQ4Dv);
      }
    } else {   // the last heads
#pragma nounroll
      for (int r = 0; r < 16; ++r) {
        if (sg.nsplit > 1 && 2 * r + hl < heads) put32(r, part + (32 * n + 2 * r) * kQ4Dv);
        if (sg.nsplit == 1 && r < 8 && 4 * r + g < heads) put16(r, out + (32 * n + 4 * r) * p.o_sh);
      }
    }
  }
}

// One workgroup per range (dmla_ranges.h) and head group.
__global__ __launch_bounds__(kThreads, 1) void q4_wide_kernel(Q4DecodeParams p) {
  __shared__ __attribute__((aligned(1024))) char keys[kKeyTiles * kKeyBytes];
  __shared__ __attribute__((aligned(1024))) char rope[kRopeSlots * kRopeBytes];
  __shared__ __attribute__((aligned(1024))) char prob[kProbBytes];
  __shared__ __attribute__((aligned(1024))) char codes[kCodeSlots * kCodeBytes];
  __shared__ __attribute__((aligned(16))) float stat[kHeads];
  __shared__ __attribute__((aligned(16))) int flag[kWaves];
  __shared__ __attribute__((aligned(16))) RangeLds ranges;
  const Lds lds = {lds_addr((DMLA_LDS char*)keys), lds_addr((DMLA_LDS char*)codes), lds_addr((DMLA_LDS char*)rope),
                   lds_addr((DMLA_LDS char*)prob), (DMLA_LDS float*)stat, (DMLA_LDS int*)flag};
  // The head groups of a range run 8 ids apart, on one XCD: the second read of its pages hits that L2.
  const int id = blockIdx.x;
  const int hg = (id / 8) % p.head_groups;
  const int r = (id / (8 * p.head_groups)) * 8 + id % 8;
  if (r >= p.n_ranges) return;
  for_each_segment<kTile, kQ4WideCost>(
      p.seqlens, p.B, p.max_pages * kQ4Page, p.n_ranges, p.min_width, r, ranges,
      [&](int b, int t0, int t1, int ctx, int nsplit) {
        run_segment(p, Q4Segment{b, t0, t1, ctx, nsplit, r + b}, lds, hg * kHeads);
      },
      [&](int b, int first_range, int nsplit) {
        if (hg != 0) return;
        p.num_splits[b] = nsplit;
        p.split_base[b] = first_range + b;
      });
}

}  // namespace

void launch_q4_wide(const Q4DecodeParams& p, int grid, hipStream_t stream) {
  hipLaunchKernelGGL(q4_wide_kernel, dim3((unsigned)grid), dim3(kThreads), 0, stream, p);
}

}  // namespace dmla
