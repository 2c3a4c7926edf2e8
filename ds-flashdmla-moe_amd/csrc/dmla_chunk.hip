// Attention of a chunk of new tokens over the paged bf16 latent cache: every sequence brings the queries of its
// newest tokens, one or many, packed one sequence after another.  No reference counterpart.
//
//   o[i, h] = softmax_j(scale q[i, h] . k[j]) . k[j][:512] over the tokens j of query i's sequence, with causal those
//   up to itself; lse[i, h] = log sum_j exp(scale q[i, h] . k[j]).
//
// MI355X design:
//  * A workgroup takes 128 rows (query, head), the head fastest: all heads read the same keys.  One wave per SIMD:
//    wave w computes the scores and the softmax of rows 32 w .. 32 w + 31 (their queries: 144 registers) and the
//    outputs of all 128 rows for the 128 columns from 128 w on (fp32, the 256 AGPRs); probabilities go through LDS.
//  * Keys lie in LDS as rows of 1024 bytes (latent dims) whose 16-byte units are permuted by key: unit u of
//    row r at u ^ key_swz(r), copied there directly, a row per copy.  The score product reads a unit of 32 rows
//    (ds_read_b128), the value product 32 columns of 8 rows transposed (ds_read_b64_tr_b16).  The rope dims have
//    rows of 128 bytes of their own, eight of them a copy.
//  * Step s multiplies scores of tile s and values of tile s - 1; copies run two tiles ahead, four tiles fit.
//  * Up to 32 rows (one token of 16 heads, say) would leave three waves without scores.  There every wave has all rows and
//    a quarter of the dims, and the partial scores of four waves are added through LDS in a fixed order (512 sequences of
//    2048 tokens x 16 heads: 264 -> 229 us).
//  * One workgroup per CU takes an equal share of all work, whatever the lengths ("cutting the work" below), and
//    a second kernel joins what was cut.
//
// Bound, by what a call is made of (MI355X, 1.2 PFLOP/s and 5 TB/s being what a large product and a large copy reach):
//  * Chunks and prompts by the matrix cores: a tile of 32 keys takes 128 rows 1.6 us, 1.4 PFLOP/s over all CUs; 1024
//    queries x 128 heads over 8192 tokens 1.69 ms (1.30 PFLOP/s, a large library product 1.36).  68 MFMAs are 2200 of a
//    tile's 3400 cycles; an MFMA hides about six other instructions, and what is more of them shows.
//  * Many single tokens by HBM: 512 sequences of 2048 tokens x 16 heads 227 us, 5.3 TB/s.
//  * Short rows of keys by what a piece costs beside its tiles, 9 us: 3 us of queries through LDS (their copies, the
//    first tile, the last tile's values) and 4 us of outputs, both at what a CU's vector memory path takes (some 27
//    bytes a cycle).  Four prompts of 200 to 2000 tokens x 128 heads: 837 us, 1.04 PFLOP/s.
//  * One token by latency: the cut, queries, tiles, the join: 26 us for 5000 tokens x 128 heads.
#include <algorithm>
#include <cmath>

#include "dmla_host.h"
#include "dmla_pipe.h"
#include "dmla_chunk_cut.h"

namespace dmla {
namespace {

constexpr int kDqk = 576, kDv = 512;
constexpr int kRowBlocks = kRows / 32;                     // of a workgroup
constexpr int kColBlocks = 4;                              // 32 columns each, of a wave
constexpr int kSteps = kDqk / 16, kLatSteps = kDv / 16;    // MFMAs of a tile's scores
constexpr int kKeyRow = 1024, kKeyBytes = kTile * kKeyRow, kSlots = 4;
constexpr int kRopeBytes = kTile * 128;
constexpr int kProbBytes = kWaves * 2048;                   // P of a step
constexpr int kNarrowRopes = 3, kShareBytes = 3 * kWaves * 1024;   // scores that the waves exchange, behind three ropes
constexpr int kLdsBytes = kSlots * kKeyBytes + std::max(kSlots * kRopeBytes + kProbBytes, kNarrowRopes * kRopeBytes + kShareBytes + 2048);
constexpr int kCopies = 9;                                 // of a wave and tile
// Queries come through that memory, in blocks of 64 dims (4 KB of a wave): the first six in the first three slots
// of keys, where they may land while the piece before puts out through the fourth, two in the fourth, and one
// in the third and fourth of the ropes and P.
constexpr int kQueryEarly = 6, kQueryBlock = 4096;
static_assert(kWaves * kQueryEarly * kQueryBlock == 3 * kKeyBytes && kWaves * 2 * kQueryBlock == kKeyBytes &&
              kWaves * kQueryBlock == 2 * kRopeBytes + kProbBytes, "where the queries lie");
constexpr float kHeadroom = 32.0f;                         // log2 headroom of P over a row's reference

__device__ __forceinline__ int key_swz(int r) { return (r & 3) << 2 | (r >> 2 & 3); }

// A copy of the kernel's arguments, read again: kept in scalar registers from piece to piece, or over a tile loop that
// needs a few of them, they would be spilled.
struct ArgumentWords {
  int w[sizeof(ChunkParams) / 4];
};
static_assert(sizeof(ArgumentWords) == sizeof(ChunkParams), "whole words");
__device__ __forceinline__ ChunkParams arguments() {
  auto a = (const __attribute__((address_space(4))) int*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  ArgumentWords words;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(ChunkParams) / 4); ++i) words.w[i] = a[i];
  return __builtin_bit_cast(ChunkParams, words);
}

struct Lds {
  unsigned keys, rope, prob;   // addresses
  DMLA_LDS float* stat;        // [kRows]: sums
  DMLA_LDS float* top;         // [kRows]: largest scores, log2 units
  DMLA_LDS int* flag;          // [kWaves]
};

// The pages of a piece, 64 at a time in a register (lane i: page first + i).
struct Pages {
  int first = 0, pages = 0;
  int bad = 0x7fffffff;   // the first page outside the pool that was met

  __device__ __forceinline__ void fetch(const ChunkParams& p, const Piece& pc, int from) {
    first = uniform(from);
    const int i = first + fresh_lane_id();
    pages = i < (pc.t1 + 1) / 2 ? p.block_table[pc.b * p.bt_sb + i] : 0;
    asm volatile("" : "+v"(pages));   // waited for here, in the rare branch, and not by every reader
  }
  // The page of index i; they come in ascending order.  A bad page reads page 0 instead.
  __device__ __forceinline__ void reach(const ChunkParams& p, const Piece& pc, int i) {
    if (i - first >= 64) fetch(p, pc, first + 64);
  }
  __device__ __forceinline__ int page(const ChunkParams& p, int i) {
    const int page = __builtin_amdgcn_readlane(pages, uniform((i - first) & 63));
    const bool off = (unsigned)page >= (unsigned)p.num_pages;
    bad = off ? min(bad, i) : bad;
    return off ? 0 : page;
  }
};

// The queries of 128 rows of a sequence from row0 on, this wave's 32: blocks [kFirst, kFirst + kN) of 64 dims.  Read
// straight into the operands, a load would touch 32 rows for 32 bytes each; a copy moves eight rows x 128 bytes.
__device__ __forceinline__ unsigned query_block(const Lds& lds, int wave, int i) {
  if (i < kQueryEarly) return lds.keys + (wave * kQueryEarly + i) * kQueryBlock;
  if (i < kQueryEarly + 2) return lds.keys + 3 * kKeyBytes + (wave * 2 + i - kQueryEarly) * kQueryBlock;
  return lds.rope + 2 * kRopeBytes + wave * kQueryBlock;
}
// Of up to kNarrowRows rows every wave has all of them, but only a quarter of the dims: two latent blocks, and of
// the rope block 16 dims.  They lie where the first three of the six would.
__device__ __forceinline__ bool narrow(int rows) { return rows <= kNarrowRows; }
__device__ __forceinline__ int query_dims(int wave, int rows, int i) {
  return 64 * (!narrow(rows) ? i : i < 2 ? 2 * wave + i : 8);
}
// This lane's place in rows 8 g .. 8 g + 7 of them.
__device__ __forceinline__ const bf16* query_rows(const ChunkParams& p, int wave, int q0, int row0, int rows, int g) {
  const int ln = fresh_lane_id();
  const int r = row0 + min((narrow(rows) ? 0 : 32 * wave) + 8 * g + (ln >> 3), rows - 1);
  const int token = fast_div(r, p.hdiv), head = r - token * p.H;
  return (const bf16*)(p.q + (q0 + token) * p.q_st + head * p.q_sh + 8 * ((ln & 7) ^ (ln >> 3)));
}
template <int kFirst, int kN>
__device__ __forceinline__ void copy_queries(const ChunkParams& p, const Lds& lds, int wave, int q0, int row0, int rows) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const bf16* src = query_rows(p, wave, q0, row0, rows, g);
#pragma unroll
    for (int i = kFirst; i < kFirst + kN; ++i)
      if (i < 3 || !narrow(rows)) dma16_addr(src + query_dims(wave, rows, i), query_block(lds, wave, i) + g * 1024);
  }
}

// Whether another pass has to follow.
// have: the queries are on their way.  After it, those of the next piece's rows are.
template <bool kNarrow>
__device__ __forceinline__ bool run_piece(const Piece& pc, const Lds& lds, const Pass& pass, bool have,
                                          const DMLA_LDS int* next) {
  const ChunkParams p = arguments();
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int rows = pc.rows;
  constexpr int kBlocks = kNarrow ? 1 : kRowBlocks;   // of 32 rows
  const int first_row = kNarrow ? 0 : 32 * wave;      // of the wave's 32
  // Rows past the last one are the last one again, and not written.
  auto limit_of = [&](int r) {   // last key of row r
    return p.causal ? pc.s.len - pc.s.n + fast_div(pc.row0 + min(r, rows - 1), p.hdiv) : pc.s.len - 1;
  };
  const int lim = limit_of(first_row + l32);
  const int lim0 = uniform(limit_of(first_row));   // the wave's smallest

  // ---- copies: lane l copies 16 bytes into place l of each kilobyte, nine of a wave and tile ----
  Pages pages;
  // Rows of a tile from key_end on are its last row before, again.
  const int key_end = uniform(min(limit_of(rows - 1) + 1, pass.to));
  const int t1 = max(pc.t0, min(pc.t1, (max(key_end, 0) + kTile - 1) / kTile));
  // (Few scalars between them: what the compiler keeps of a loop's scalars, it keeps in lanes of a register.)
  const char* copy_src = nullptr;   // the first of the wave's rows
  int copy_more = 0;                // rows behind it
  unsigned copy_keys = 0, copy_rope = 0, copy_lane = 0;
  const int row_step = uniform((int)p.kv_ss);
  // What the copies of a tile need, in kBegins parts for the gaps between MFMAs (an MFMA hides about six instructions).
  constexpr int kBegins = 4;
  int copy_t = 0, copy_row = 0;
  auto copy_begin = [&](int s, int part) {
    if (part == 0) {
      copy_t = min(pc.t0 + s, t1 - 1);   // past the end: the last tile, which nobody counts
      pages.reach(p, pc, copy_t >> 1);
    } else if (part == 1) {
      const int last = uniform(min(key_end - copy_t * kTile, kTile) - 1);
      copy_row = min(8 * wave, last);
      copy_more = last - copy_row;
      copy_row += (copy_t & 1) * kTile;   // of the page
    } else if (part == 2) {
      copy_src = (const char*)(p.kv + pages.page(p, copy_t >> 1) * p.kv_sp);
    } else {
      copy_src += copy_row * row_step;
      copy_lane = 16 * (fresh_lane_id() ^ key_swz(8 * wave));
      copy_keys = lds.keys + (unsigned)(s % kSlots) * kKeyBytes + wave * 8 * kKeyRow;
      copy_rope = lds.rope + (unsigned)(s % (kNarrow ? kNarrowRopes : kSlots)) * kRopeBytes + wave * 1024;
    }
  };
  auto copy = [&](int i) {
    if (i < 8) {   // key_swz(8 wave + i) is key_swz(8 wave) ^ key_swz(i)
      dma16(copy_src, (copy_lane ^ (16 * key_swz(i))) + min(i, copy_more) * row_step, copy_keys + i * kKeyRow);
    } else {
      const int ln = fresh_lane_id();
      const unsigned off = min(ln >> 3, copy_more) * row_step + 2 * kDv + 16 * ((ln & 7) ^ (ln >> 3));
      dma16(copy_src, off, copy_rope);
    }
  };
  auto copy_tile = [&](int s) {
#pragma unroll
    for (int i = 0; i < kBegins; ++i) copy_begin(s, i);
#pragma unroll
    for (int i = 0; i < kCopies; ++i) copy(i);
  };

  // ---- queries: 36 operands of 16 dims; operand c holds dims 16 c + 8 hl .. of row l32.  Narrow: those of dims
  // 128 wave .. + 127, and of rope dims 16 wave .. + 15 ----
  const int n_steps = t1 - pc.t0;
  constexpr int kOwnSteps = kNarrow ? kSteps / kWaves : kSteps;
  bf16x8 q[kOwnSteps];
  auto take_queries = [&](auto first_tag, auto n_tag) {
    constexpr int kFirst = decltype(first_tag)::value, kN = decltype(n_tag)::value;
#pragma unroll
    for (int i = kFirst; i < kFirst + kN; ++i) {
      const unsigned a = lds_sum(1024 * (l32 >> 3) + 128 * (l32 & 7) + 16 * (hl ^ (l32 & 7)), query_block(lds, wave, i));
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (4 * i + c < kOwnSteps) q[4 * i + c] = *lds_ptr<const bf16x8>(kNarrow && i == 2 ? a ^ (32 * wave) : a ^ (32 * c));
    }
  };
  if (!have) copy_queries<0, 9>(p, lds, wave, pc.s.q0, pc.row0, rows);
  pages.fetch(p, pc, pc.t0 / 2);
  wait_vm<0>();
  using std::integral_constant;
  take_queries(integral_constant<int, 0>{}, integral_constant<int, kNarrow ? 3 : 9>{});
  wait_lds();
  __syncthreads();   // the keys' memory is free
  if (n_steps > 0) copy_tile(0);

  f32x16 acc[kBlocks][kColBlocks];   // O^T: register i is column 128 wave + 32 j + 16 hl + i of row l32
  float mref = kNegInf, mtrue = kNegInf, lsum = 0.f;   // reference, largest score seen, sum
  bf16x8 pv[2];             // P of the wave's own rows, 16 keys each

  // A barrier that waits for nothing else: what it orders has been waited for.
  auto barrier = [] {
    in_order();
    asm volatile("s_barrier" ::: "memory");
    in_order();
  };
  auto opaque = [](unsigned a) {
    if constexpr (kNarrow) a = (unsigned)uniform((int)a);
    asm("" : "+s"(a));
    return a;
  };

  // ---- scores: S^T[key 8 (i / 4) + 4 hl + i % 4][row l32] of step s's tile ----
  bf16x8 rope[4];
  constexpr int kDepth = 6;   // operands in flight
  unsigned key_addr = 0;
  bf16x8 k[kDepth];
  auto read_rope = [&](int s) {
    const unsigned a = lds_sum(128 * l32 + 16 * (hl ^ (l32 & 7)), opaque(lds.rope + (unsigned)(s % kSlots) * kRopeBytes));
#pragma unroll
    for (int c = 0; c < 4; ++c) rope[c] = *lds_ptr<const bf16x8>(a ^ (32 * c));
  };
  auto read_key = [&](int c) { k[c % kDepth] = *lds_ptr<const bf16x8>((key_addr ^ (32 * (c & 7))) + 256 * (c >> 3)); };
  auto scores_begin = [&](int s) {
    key_addr = lds_sum(kKeyRow * l32 + 16 * (hl ^ key_swz(l32)), opaque(lds.keys + (unsigned)(s % kSlots) * kKeyBytes));
  };
  // After read_rope(s), scores_begin(s) and the first kDepth reads; beside(m) runs after MFMA m = 0 .. 35.
  // The result may be read after score_done or two more MFMAs.
  auto scores = [&](auto beside) -> f32x16 {
    f32x16 x;
    static_for<kSteps>([&](auto m_tag) {
      constexpr int m = decltype(m_tag)::value, c = m - 4;
      if constexpr (m < 4) score_step<m == 0>(x, rope[m], q[kLatSteps + m]);
      else score_step<false>(x, k[c % kDepth], q[c]);
      if constexpr (m >= 4 && c + kDepth < kLatSteps) read_key(c + kDepth);
      beside(m_tag);
      in_order();
    });
    return x;
  };
  auto mask = [&](f32x16& x, int s) {
    const int key = (pc.t0 + s) * kTile;
    if (key + kTile - 1 > lim0) {
      asm volatile("" : "+v"(x));   // the last tiles only: a branch
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = key + 8 * (i >> 2) + 4 * hl + (i & 3) <= lim ? x[i] : kNegInf;
    }
  };
  auto tile_max = [&](const f32x16& x) {
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
    return half_max(mx) * p.scale_log2;   // scale > 0
  };
  // (fmaxf would quiet each operand first, an instruction more for each.)
  auto max3 = [](float a, float b, float c) {
    float v;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(v) : "v"(a), "v"(b), "v"(c));
    return v;
  };
  // The softmax of a tile in kPieces pieces, which the value product of another tile takes between its
  // MFMAs: the maximum, then an element at a time.
  constexpr int kPieces = 21;
  float mx_part[4];
  float ms = 0.f;
  auto softmax_piece = [&](const f32x16& x, auto i_tag) {
    constexpr int i = decltype(i_tag)::value;
    if constexpr (i < 4) {
      mx_part[i] = max3(max3(x[4 * i], x[4 * i + 1], x[4 * i + 2]), x[4 * i + 3], x[4 * i + 3]);
    } else if constexpr (i == 4) {
      const float mx = half_max(max3(max3(mx_part[0], mx_part[1], mx_part[2]), mx_part[3], mx_part[3]));
      mtrue = fmaxf(mtrue, mx * p.scale_log2);   // scale > 0
      ms = mref == kNegInf ? 0.f : mref;
    } else if constexpr (i < kPieces) {
      constexpr int e = i - 5;
      const float v = fast_exp2(__builtin_fmaf(x[e], p.scale_log2, -ms));
      lsum += v;
      pv[e >> 3][e & 7] = (bf16)v;   // what the value product takes; the sum keeps fp32
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
  bf16x8 prob[kBlocks], val[3];
  unsigned val_addr = 0, prob_addr = 0;
  auto values_begin = [&](int s) {
    const int r = (lane & 15) >> 2, g = lane >> 4 & 1;
    val_addr = lds_sum(kKeyRow * (4 * hl + r) + 256 * wave + 16 * (4 * r | ((g + 2 * (lane & 1)) ^ hl)) + 8 * ((lane & 3) >> 1),
                       opaque(lds.keys + (unsigned)(s % kSlots) * kKeyBytes));
    prob_addr = lds_sum(16 * lane, lds.prob);
  };
  auto read_prob = [&](int u, int n) { prob[n] = *lds_ptr<const bf16x8>(prob_addr + 2048 * n + 1024 * u); };
  auto read_values = [&](int g) {
    const unsigned a = val_addr ^ (64 * (g % 4));
    const int at = 16 * kKeyRow * (g / 4);
    val[g % 3] = concat(lds_read_tr16(lds_ptr<const bf16x4>(a + at)),
                        lds_read_tr16(lds_ptr<const bf16x4>((a ^ 32) + at + 8 * kKeyRow)));
  };
  // After values_begin(s), the probabilities of the first 16 keys and the values of groups 0 and 1;
  // beside(i) runs after MFMA i = 0 .. 31.
  auto values = [&](auto beside) {
    static_for<32>([&](auto i_tag) {
      constexpr int i = decltype(i_tag)::value, g = i / 4, n = i % 4;
      acc[n][g % 4] = mfma32_bf16(val[g % 3], prob[n], acc[n][g % 4]);
      if constexpr (n == 0 && g + 2 < 8) read_values(g + 2);
      if constexpr (g == 3) read_prob(1, n);
      beside(i_tag);
      in_order();
    });
  };
  // ---- up to 32 rows.  Scores: wave w multiplies its quarter of the dims and finishes, from the four partial
  // products, keys 8 w .. 8 w + 7 of the tile (elements 4 w .. 4 w + 3); values: all keys for its 128 columns.  Two
  // barriers a tile: products of scores and values between them, the softmax of 4 elements behind the second.
  // A wave alone with 32 rows' scores takes 3400 cycles a tile.
  const unsigned share = lds.rope + kNarrowRopes * kRopeBytes, narrow_prob = share + kShareBytes;
  auto total_of = [&](float v, auto f) {   // of a row, over the waves
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
    __syncthreads();
    if (hl == 0) lds.stat[32 * wave + l32] = v;
    __syncthreads();
    v = f(f(lds.stat[l32], lds.stat[32 + l32]), f(lds.stat[64 + l32], lds.stat[96 + l32]));
    __syncthreads();   // read
    return v;
  };
  auto narrow_steps = [&] {
    f32x4 own;
    auto partial = [&](int s) {   // its quarter of tile s's scores, and the others' keys of it to them
      const unsigned kb = lds_sum(kKeyRow * l32 + 16 * (hl ^ key_swz(l32)), opaque(lds.keys + (unsigned)(s % kSlots) * kKeyBytes + 256 * wave));
      const unsigned rb = lds_sum(128 * l32 + 16 * (hl ^ (l32 & 7)), opaque(lds.rope + (unsigned)(s % kNarrowRopes) * kRopeBytes)) ^ (32 * wave);
      bf16x8 k[kOwnSteps];
#pragma unroll
      for (int c = 0; c < 8; ++c) k[c] = *lds_ptr<const bf16x8>(kb ^ (32 * c));
      k[8] = *lds_ptr<const bf16x8>(rb);
      f32x16 x;
      static_for<kOwnSteps>([&](auto c_tag) {
        constexpr int c = decltype(c_tag)::value;
        score_step<c == 0>(x, k[c], q[c]);
      });
      score_done(x);
      static_for<kWaves>([&](auto d_tag) {
        constexpr int d = decltype(d_tag)::value;
        const f32x4 v = {x[4 * d], x[4 * d + 1], x[4 * d + 2], x[4 * d + 3]};
        if (d == wave) own = v;
        else *lds_ptr<f32x4>(lds_sum(16 * lane, opaque(share + (3 * d + wave - (wave > d ? 1 : 0)) * 1024))) = v;
      });
    };
    // Scores of the wave's keys of tile s: what the others have of them (always in the waves' order), the mask.
    auto finish = [&](int s) {
      const unsigned at = lds_sum(16 * lane, opaque(share + 3 * wave * 1024));
      f32x4 part[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) part[i] = *lds_ptr<const f32x4>(at + 1024 * i);
      f32x4 sum = wave == 0 ? own : part[0];
      sum += wave == 1 ? own : part[wave > 1 ? 1 : 0];
      sum += wave == 2 ? own : part[wave > 2 ? 2 : 1];
      sum += wave == 3 ? own : part[2];
      const int key = (pc.t0 + s) * kTile + 8 * wave + 4 * hl;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = key + i <= lim ? sum[i] * p.scale_log2 : kNegInf;
      mtrue = fmaxf(mtrue, fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3])));
      return sum;
    };
    auto softmax = [&](const f32x4& x) {
      const float ms = mref == kNegInf ? 0.f : mref;
      bf16x4 pr;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = fast_exp2(x[i] - ms);
        lsum += v;
        pr[i] = (bf16)v;   // what the value product takes; the sum keeps fp32
      }
      *lds_ptr<bf16x4>(lds_sum(16 * lane, opaque(narrow_prob + 1024 * (wave >> 1) + 8 * (wave & 1)))) = pr;
    };
    copy_tile(1);
    copy_tile(2);
    wait_vm<2 * kCopies>();
    __syncthreads();   // tile 0 landed
    partial(0);
    __syncthreads();   // partial products posted
    const f32x4 x0 = finish(0);
    if (pass.careful) {
      mref = lds.top[l32];
    } else {
      mref = total_of(mtrue, [](float a, float b) { return fmaxf(a, b); });
    }
    softmax(x0);
    wait_vm<kCopies>();
    wait_lds();
    __syncthreads();   // P posted, tile 1 landed
#pragma nounroll
    for (int s = 0;; ++s) {
      copy_tile(s + 3);   // where tile s - 1 was
      {
        const int r = (lane & 15) >> 2, g = lane >> 4 & 1;
        const unsigned vb = lds_sum(kKeyRow * (4 * hl + r) + 256 * wave + 16 * (4 * r | ((g + 2 * (lane & 1)) ^ hl)) + 8 * ((lane & 3) >> 1),
                                    opaque(lds.keys + (unsigned)(s % kSlots) * kKeyBytes));
        const unsigned pb = lds_sum(16 * lane, opaque(narrow_prob));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 pr = *lds_ptr<const bf16x8>(pb + 1024 * u);
#pragma unroll
          for (int j = 0; j < kColBlocks; ++j) {
            const unsigned a = (vb ^ (64 * j));
            const bf16x8 v = concat(lds_read_tr16(lds_ptr<const bf16x4>(a + 16 * kKeyRow * u)),
                                    lds_read_tr16(lds_ptr<const bf16x4>((a ^ 32) + 16 * kKeyRow * u + 8 * kKeyRow)));
            acc[0][j] = mfma32_bf16(v, pr, acc[0][j]);
          }
        }
      }
      if (s + 1 == n_steps) break;
      partial(s + 1);
      wait_lds();
      barrier();   // partial products posted, P and tile s read
      softmax(finish(s + 1));
      wait_vm<kCopies>();   // tile s + 2; one tile more may be on its way
      wait_lds();
      barrier();   // P posted, tile s + 2 landed
    }
    mtrue = total_of(mtrue, [](float a, float b) { return fmaxf(a, b); });
  };

  {
    lsum = 0.f;
    // Zeros by the matrix core, a whole accumulator at a time: element by element the compiler would
    // assemble them elsewhere and move them.
#pragma unroll
    for (int n = 0; n < kBlocks; ++n)
#pragma unroll
      for (int j = 0; j < kColBlocks; ++j) acc[n][j] = mfma32_bf16(bf16x8{}, bf16x8{}, f32x16{});
    if constexpr (kNarrow) {
      if (n_steps > 0) narrow_steps();
    } else if (n_steps > 0) {
      wait_vm<0>();
      __syncthreads();   // tile 0 landed
      read_rope(0);
      scores_begin(0);
#pragma unroll
      for (int c = 0; c < kDepth; ++c) read_key(c);
      f32x16 x0 = scores([&](auto m_tag) {
        constexpr int m = decltype(m_tag)::value;
        if constexpr (m % 18 == 0)
          for (int i = 0; i < kBegins; ++i) copy_begin(1 + m / 18, i);
        if constexpr (m % 2 == 1) copy(m % 18 / 2);
      });
      score_done(x0);
      mask(x0, 0);
      const float top = tile_max(x0);
      mref = pass.careful ? lds.top[first_row + l32] : top;
      mtrue = top;
      static_for<kPieces>([&](auto i) { softmax_piece(x0, i); });
      post();
      wait_vm<kCopies>();
      wait_lds();
      __syncthreads();   // tile 1 landed
      read_rope(1);
      scores_begin(1);
#pragma unroll
      for (int c = 0; c < kDepth; ++c) read_key(c);
      // Step s: scores of tile s; barrier A; values of tile s - 1, with the softmax of tile s; barrier B; the start of
      // the next step's scores.  A stands where P of step s - 1 is posted, B where tile s - 1 has been read and tile
      // s + 1 has landed.  Both stand among MFMAs whose operands are there, and what they guard is read a few MFMAs
      // ahead of its use.  Copies start two tiles ahead.
#pragma nounroll
      for (int s = 1; s < n_steps; ++s) {
        f32x16 x = scores([&](auto m_tag) {
          constexpr int m = decltype(m_tag)::value;
          if constexpr (m >= 1 && m <= kBegins) copy_begin(s + 2, m - 1);
          // (A copy takes a CU some 90 cycles for four waves, three MFMAs; beside the softmax there is no room for them.)
          if constexpr (m >= 6 && m % 3 == 0 && m != 24) copy(m < 24 ? m / 3 - 2 : m / 3 - 3);
          if constexpr (m == 22) {
            wait_lds<7>();   // P is posted; reads of later keys may be on their way
            barrier();       // A
          }
          if constexpr (m == 23) values_begin(s - 1);
          if constexpr (m >= 24 && m < 28) read_prob(0, m - 24);
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
            wait_vm<kCopies>();   // this wave's copies of tile s + 1; those of one tile more may be on their way
            wait_lds();           // the values of tile s - 1
            barrier();            // B
          } else if constexpr (i == 25) {
            post();
          } else if constexpr (i == 26) {
            read_rope(s + 1);
            scores_begin(s + 1);
          } else if constexpr (i > 26 && i <= 26 + kDepth / 2) {
            read_key(2 * (i - 27));
            read_key(2 * (i - 27) + 1);
          }
        });
      }
      // The values of the last tile.
      wait_lds();
      __syncthreads();   // its P is posted
      values_begin(n_steps - 1);
#pragma unroll
      for (int n = 0; n < kRowBlocks; ++n) read_prob(0, n);
      read_values(0);
      read_values(1);
      values([](auto) {});
    }
  }
  if constexpr (kNarrow) lsum = total_of(lsum, [](float a, float b) { return a + b; });

  // ---- output ----
  const ChunkParams out = arguments();
  if constexpr (!kNarrow) lsum = half_sum(lsum);
  if (hl == 0 && (!kNarrow || wave == 0)) {
    if (!pass.careful) lds.top[first_row + l32] = mtrue;
    lds.stat[first_row + l32] = (int64_t)lim >= pages.bad * (int64_t)kPage ? __builtin_nanf("") : lsum;
  }
  bool wrong = !pass.careful && mtrue > mref + kHeadroom;
  agpr_settle();
  wait_vm<0>();
  wait_lds();
  __syncthreads();   // the keys' memory is free, the sums are posted
  auto written = [&](int row) {
    bool w = row < rows;
    if (pass.careful) {
      const int l = out.causal ? pc.s.len - pc.s.n + fast_div(pc.row0 + min(row, rows - 1), out.hdiv) : pc.s.len - 1;
      w = w && l >= pass.from && l < pass.to;
    }
    return w;
  };
  auto place = [&](int row, int64_t st, int64_t sh) {   // of a row in o
    const int r = pc.row0 + row, token = fast_div(r, out.hdiv);
    return (pc.s.q0 + token) * st + (r - token * out.H) * sh;
  };
  if (hl == 0 && (!kNarrow || wave == 0) && written(first_row + l32)) {
    const float sum = lds.stat[first_row + l32];
    const float lse2 = sum == 0.f ? kNegInf : mref + __log2f(sum);
    if (pc.slot >= 0) out.part_lse[(int64_t)pc.slot * kRows + first_row + l32] = lse2;
    else if (out.lse != nullptr) out.lse[place(first_row + l32, out.H, 1)] = lse2 * kLn2;
  }
  // Through LDS, so that a store covers whole lines: 256 bytes of each of 4 rows, or of a part 512 bytes of each of 2.
  // A wave has its own memory there.
  float check = 0.f;   // the largest output
  auto look = [&](float a, float b) { asm("v_maximum3_f32 %0, |%1|, |%2|, %0" : "+v"(check) : "v"(a), "v"(b)); };
  auto inverse = [&](int n) {
    const float sum = lds.stat[32 * n + l32];
    return sum == 0.f ? 0.f : 1.f / sum;
  };
  if (pc.slot < 0) {
    // The next piece's queries are asked for between the conversions, a copy every other 16 values: in one go they
    // would wait for each other (24 of them 3600 cycles).
    const int next_q0 = uniform(next[0]), next_row0 = uniform(next[1]), next_rows = uniform(next[2]);
    // Rows of 256 bytes, 16-byte unit u of row r at u ^ (r % 16), 32 rows at a time in the last slot.
    const unsigned mine = lds.keys + 3 * kKeyBytes + wave * 8192;
    const unsigned put = lds_sum(256 * l32 + 16 * ((2 * hl) ^ (l32 & 15)), mine);
    const int g = lane >> 4, c = lane & 15;
    const unsigned get = lds_sum(256 * g + 16 * (c ^ g), mine);   // 8 columns of row g
    // Where rows follow each other evenly (contiguous outputs), offsets from the first one need no division.
    const bool even = out.o_st == out.H * out.o_sh && out.o_sh < (1 << 20);
    const int out_step = (int)out.o_sh;
    Global<bf16> first = out.o + pc.s.q0 * out.o_st + pc.row0 * out.o_sh + 128 * wave + (g * out_step + 8 * c);
    const bool plain = even && !pass.careful;
#pragma unroll
    for (int n = 0; n < kRowBlocks; ++n) {
      const bf16* src = nullptr;
      if (next_rows > 0) src = query_rows(out, wave, next_q0, next_row0, next_rows, n);
      auto ask = [&](int i) {
        if (next_rows > 0 && i < (narrow(next_rows) ? 3 : kQueryEarly))
          dma16_addr(src + query_dims(wave, next_rows, i), query_block(lds, wave, i) + n * 1024);
      };
      if (n >= kBlocks || 32 * n >= rows) {   // no rows there
#pragma unroll
        for (int i = 0; i < kQueryEarly; ++i) ask(i);
        continue;
      }
      const float inv = inverse(n);
#pragma unroll
      for (int j = 0; j < kColBlocks; ++j)
#pragma unroll
        for (int d = 0; d < 2; ++d) {
          ask(2 * j + d);
          bf16x8 v;
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const float a = agpr_read(acc[n % kBlocks][j][8 * d + i]) * inv, b = agpr_read(acc[n % kBlocks][j][8 * d + i + 1]) * inv;
            look(a, b);
            v[i] = (bf16)a;
            v[i + 1] = (bf16)b;
          }
          *lds_ptr<bf16x8>(put ^ (16 * (4 * j + d))) = v;
        }
      bf16x8 v[8];   // row 4 r + g
#pragma unroll
      for (int r = 0; r < 8; ++r) v[r] = *lds_ptr<const bf16x8>((get ^ (64 * (r & 3))) + 1024 * r);
      if (plain) {
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (32 * n + 4 * r + g < rows) *reinterpret_cast<Global<bf16x8>>(first + (32 * n + 4 * r) * out_step) = v[r];
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int row = 32 * n + 4 * r + g;
          if (written(row)) *reinterpret_cast<Global<bf16x8>>(out.o + place(row, out.o_st, out.o_sh) + 128 * wave + 8 * c) = v[r];
        }
      }
    }
  } else {
    // Rows of 512 bytes, 16-byte unit u of row r at u ^ r.
    const unsigned mine = lds.keys + wave * kKeyBytes;
    const unsigned put = lds_sum(512 * l32 + 16 * ((4 * hl) ^ l32), mine);
    const unsigned get = lds_sum(512 * hl + 16 * (l32 ^ hl), mine);     // 4 columns of row hl
    Global<float> part = out.part_o + (int64_t)pc.slot * kRows * kDv + 128 * wave;
#pragma unroll
    for (int n = 0; n < kBlocks; ++n) {
      if (32 * n >= rows) break;
      const float inv = inverse(n);
#pragma unroll
      for (int j = 0; j < kColBlocks; ++j)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          f32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = agpr_read(acc[n][j][4 * d + i]) * inv;
          look(v[0], v[1]);
          look(v[2], v[3]);
          *lds_ptr<f32x4>(put ^ (16 * (8 * j + d))) = v;
        }
#pragma unroll
      for (int r = 0; r < 16; ++r) {   // row 2 r + hl
        const f32x4 v = *lds_ptr<const f32x4>((get ^ (32 * r)) + 1024 * r);
        const int row = 32 * n + 2 * r + hl;
        if (written(row)) *reinterpret_cast<Global<f32x4>>(part + row * kDv + 4 * l32) = v;
      }
    }
  }
  wrong = wrong || !(check < __builtin_inff());
  wait_lds();
  if (lane == 0) lds.flag[wave] = 0;
  if (__any(wrong)) lds.flag[wave] = 1;
  __syncthreads();   // the keys' memory is free
  // The rest of the next queries, while the piece after that is worked out.
  const int next_q0 = uniform(next[0]), next_row0 = uniform(next[1]), next_rows = uniform(next[2]);
  if (next_rows > 0) {
    if (pc.slot >= 0) copy_queries<0, kQueryEarly>(out, lds, wave, next_q0, next_row0, next_rows);
    copy_queries<kQueryEarly, 3>(out, lds, wave, next_q0, next_row0, next_rows);
  }
  return uniform(lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]) != 0;
}

__global__ __launch_bounds__(kThreads, 1) void chunk_kernel(ChunkParams) {
  __shared__ __attribute__((aligned(1024))) char mem[kLdsBytes];
  __shared__ __attribute__((aligned(16))) float stat[kRows], top[kRows];
  __shared__ __attribute__((aligned(16))) int flag[kWaves];
  __shared__ __attribute__((aligned(16))) Window window;
  DMLA_LDS Window* win = (DMLA_LDS Window*)&window;
  DMLA_LDS i32x4* pieces = (DMLA_LDS i32x4*)window.piece;
  const unsigned base = lds_addr((DMLA_LDS char*)mem);
  const Lds lds = {base, base + kSlots * kKeyBytes, base + kSlots * (kKeyBytes + kRopeBytes), (DMLA_LDS float*)stat, (DMLA_LDS float*)top,
                   (DMLA_LDS int*)flag};
  // Ranges that follow each other run on one XCD: they read the same keys.
  auto my_range = [&] {
    const int per_xcd = (arguments().n_ranges + 7) / 8;
    return (int)(blockIdx.x % 8) * per_xcd + (int)(blockIdx.x / 8);
  };
  if (my_range() >= arguments().n_ranges) return;
  if (!cut(arguments(), win, my_range())) return;
  next_piece(arguments(), win, pieces, my_range());
  bool have = false;
  for (int turn = 0;; turn ^= 1) {
    DMLA_LDS i32x4* now = pieces + 3 * turn;
    DMLA_LDS i32x4* other = pieces + 3 * (turn ^ 1);
    __syncthreads();   // this piece is known, the one before it is read
    const i32x4 a = now[0], b = now[1];
    if (uniform(a[2]) == 0) break;
    next_piece(arguments(), win, other, my_range());
    const Piece pc = {Sequence{uniform(a[0]), uniform(a[3]), uniform(b[0])}, uniform(b[1]), uniform(a[1]), uniform(a[2]), uniform(b[2]), uniform(b[3]),
                      uniform(now[2][0])};
    const DMLA_LDS int* next = (const DMLA_LDS int*)other;
    Pass pass = {false, (int)0x80000000, 0x7fffffff};
    const bool few = narrow(pc.rows);
    for (;;) {
      const bool again = few ? run_piece<true>(pc, lds, pass, have, next) : run_piece<false>(pc, lds, pass, have, next);
      have = true;
      if (pass.careful ? pass.to == 0x7fffffff : !again) break;
      const ChunkParams p = arguments();
      const int base = pc.s.len - pc.s.n, last = pc.row0 + pc.rows - 1;
      const int first_lim = p.causal ? base + fast_div(pc.row0, p.hdiv) : pc.s.len - 1;
      const int last_lim = p.causal ? base + fast_div(last, p.hdiv) : pc.s.len - 1;
      pass = careful_pass(p, pc, lds.flag, pass.careful ? pass.to : first_lim, last_lim);
      wait_vm<0>();   // the next piece's queries, which are copied once more
      __syncthreads();
      have = false;
    }
  }
}

// ---- joining parts ------------------------------------------------------------------------------------
// Row tiles that span ranges: o = sum_j w_j o_j / sum_j w_j with w_j = 2^(lse_j - max); and the queries behind the last
// sequence.  p.groups workgroups per range.  Those of the range that a row tile begins in join it, a wave several
// rows at a time, so that eight parts are in flight whether a row has two of them or more; those of the ranges that it
// fills whole (which begin no row tile) help.  With kManyParts and more a workgroup takes kSpan columns of a row, and
// its 16-lane groups every sixteenth part (one sequence of 100000 tokens x 16 heads, 256 parts: 7 us, row by row 16), unless
// the workgroups are so few that each would take many in turn (128 rows of 17 parts: 34 us, row by row 17).
constexpr int kManyParts = 16, kSpan = 64, kSpanTurns = 3;
constexpr int kInFlight = 8;
struct Joined {   // the parts of a row tile: of its first range, then those that the next ranges begin with
  int rows, q0, row0, range, parts;
  __device__ __forceinline__ int64_t place(int j, int row) const {
    return (int64_t)(j == 0 ? 2 * range + 1 : 2 * (range + j)) * kRows + row;
  }
};

// Where a row's output goes, and its lse.
__device__ __forceinline__ int64_t token_head(const ChunkParams& p, const Joined& t, int row, int& head) {
  const int r = t.row0 + row, token = fast_div(r, p.hdiv);
  head = r - token * p.H;
  return t.q0 + token;
}
__device__ __forceinline__ float joined_lse(float top, float sum, bool odd) {
  return odd ? __builtin_nanf("") : sum > 0.f ? (top + __log2f(sum)) * kLn2 : kNegInf;
}
__device__ __forceinline__ float joined_scale(float sum, bool odd) {
  return odd ? __builtin_nanf("") : sum > 0.f ? 1.f / sum : 0.f;
}

// Rows first, first + step, .. of a wave, kAt of them at a time, kInFlight / kAt parts each; with kAt 1 any number.
template <int kAt>
__device__ __forceinline__ void join_rows(const ChunkParams& p, const Joined& t, int first, int step) {
  constexpr int kParts = kInFlight / kAt;
  const int lane = threadIdx.x & 63;
  for (int row = first; row < t.rows; row += kAt * step) {
    float top[kAt], sum[kAt];
    bool odd[kAt];   // not a number among them
    f32x4 a0[kAt], a1[kAt];
#pragma unroll
    for (int r = 0; r < kAt; ++r) {
      top[r] = kNegInf;
      sum[r] = 0.f;
      odd[r] = false;
      a0[r] = a1[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int j0 = 0; j0 < (kAt == 1 ? t.parts : 1); j0 += kParts) {
      f32x4 v0[kAt][kParts], v1[kAt][kParts];
      float l[kAt][kParts];
#pragma unroll
      for (int r = 0; r < kAt; ++r)
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          const int64_t at = t.place(min(j0 + j, t.parts - 1), min(row + r * step, t.rows - 1));
          l[r][j] = p.part_lse[at];
          v0[r][j] = *reinterpret_cast<Global<const f32x4>>(p.part_o + at * kDv + 8 * lane);
          v1[r][j] = *reinterpret_cast<Global<const f32x4>>(p.part_o + at * kDv + 8 * lane + 4);
        }
#pragma unroll
      for (int r = 0; r < kAt; ++r) {
        float high = top[r];
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          high = fmaxf(high, l[r][j]);
          odd[r] = odd[r] || l[r][j] != l[r][j];
        }
        if (kAt == 1 && j0 > 0) {
          const float less = top[r] == kNegInf ? 0.f : fast_exp2(top[r] - high);
          sum[r] *= less;
          a0[r] *= less;
          a1[r] *= less;
        }
        top[r] = high;
#pragma unroll
        for (int j = 0; j < kParts; ++j) {
          const float w = j0 + j >= t.parts || high == kNegInf ? 0.f : fast_exp2(l[r][j] - high);
          if (w == 0.f) continue;   // a part without a weight adds nothing, whatever it holds
          sum[r] += w;
          a0[r] += w * v0[r][j];
          a1[r] += w * v1[r][j];
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kAt; ++r) {
      if (row + r * step >= t.rows) break;
      const float scale = joined_scale(sum[r], odd[r]);
      bf16x8 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = (bf16)(a0[r][i] * scale);
        v[4 + i] = (bf16)(a1[r][i] * scale);
      }
      int head;
      const int64_t token = token_head(p, t, row + r * step, head);
      *reinterpret_cast<Global<bf16x8>>(p.o + token * p.o_st + head * p.o_sh + 8 * lane) = v;
      if (lane == 0 && p.lse != nullptr) p.lse[token * p.H + head] = joined_lse(top[r], sum[r], odd[r]);
    }
  }
}

struct JoinLds {
  f32x4 sums[4][kSpan / 4];
  float sum[4];
};
// kSpan columns of a row, by a workgroup.
__device__ __forceinline__ void join_span(const ChunkParams& p, const Joined& t, JoinLds& lds, int row, int span) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int column = span * kSpan + 4 * (lane & 15), group = 4 * wave + (lane >> 4);   // of 16
  float top = kNegInf;
  bool odd = false;
  for (int j0 = 0; j0 < t.parts; j0 += 64) {
    const float l = j0 + lane < t.parts ? p.part_lse[t.place(j0 + lane, row)] : kNegInf;
    top = fmaxf(top, l);
    odd = odd || l != l;
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  odd = __any(odd);
  float sum = 0.f;
  f32x4 a = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = group; j0 < t.parts; j0 += 16 * kInFlight) {
    f32x4 v[kInFlight];
    float l[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int64_t at = t.place(min(j0 + 16 * i, t.parts - 1), row);
      l[i] = p.part_lse[at];
      v[i] = *reinterpret_cast<Global<const f32x4>>(p.part_o + at * kDv + column);
    }
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const float w = j0 + 16 * i >= t.parts || top == kNegInf ? 0.f : fast_exp2(l[i] - top);
      sum += w;
      if (w != 0.f) a += w * v[i];
    }
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    sum += __shfl_xor(sum, o, 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] += __shfl_xor(a[i], o, 64);
  }
  __syncthreads();   // the span before this one is read
  if (lane < 16) lds.sums[wave][lane] = a;
  if (lane == 0) lds.sum[wave] = sum;
  __syncthreads();
  if (threadIdx.x < 16) {
    sum = lds.sum[0] + lds.sum[1] + lds.sum[2] + lds.sum[3];
    a = lds.sums[0][lane] + lds.sums[1][lane] + lds.sums[2][lane] + lds.sums[3][lane];
    const float scale = joined_scale(sum, odd);
    bf16x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (bf16)(a[i] * scale);
    int head;
    const int64_t token = token_head(p, t, row, head);
    *reinterpret_cast<Global<bf16x4>>(p.o + token * p.o_st + head * p.o_sh + column) = v;
    if (column == 0 && p.lse != nullptr) p.lse[token * p.H + head] = joined_lse(top, sum, odd);
  }
}

__global__ __launch_bounds__(256) void chunk_combine_kernel(ChunkParams p) {
  __shared__ JoinLds lds;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int mine = (int)blockIdx.x / p.groups, index = (int)blockIdx.x % p.groups;
  if (mine < p.n_ranges) {
    constexpr int kWords = kMaxRanges / 64;
    i32x4 link[kWords];   // lane i: of ranges i, 64 + i, ..
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const i32x4 v = p.links[min(64 * k + lane, p.n_ranges - 1)];
      link[k] = 64 * k + lane < p.n_ranges ? v : i32x4{0, 0, 0, 0};
    }
    // The last range up to this one in which a row tile begins, if the ranges since are whole within it, and the first
    // one behind it that is not.
    int range = -1, rows = 0, q0 = 0, row0 = 0, other = 0, end = p.n_ranges;
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const unsigned long long upto = mine >= 64 * k + 63 ? ~0ull : mine < 64 * k ? 0 : (2ull << (mine - 64 * k)) - 1;
      const unsigned long long begins = __ballot(link[k][0] > 0) & upto, odd = __ballot(link[k][3] != 2 && link[k][0] == 0) & upto;
      if (begins != 0) {
        const int at = 63 - __builtin_clzll(begins);
        range = 64 * k + at;
        rows = __builtin_amdgcn_readlane(link[k][0], at);
        q0 = __builtin_amdgcn_readlane(link[k][1], at);
        row0 = __builtin_amdgcn_readlane(link[k][2], at);
      }
      if (odd != 0) other = 64 * k + 63 - __builtin_clzll(odd) + 1;
    }
#pragma unroll
    for (int k = kWords - 1; k >= 0; --k) {
      const unsigned long long upto = range >= 64 * k + 63 ? ~0ull : range < 64 * k ? 0 : (2ull << (range - 64 * k)) - 1;
      const unsigned long long ends = __ballot(link[k][3] != 2) & ~upto;
      if (ends != 0) end = 64 * k + __builtin_ctzll(ends);
    }
    if (range >= other) {
      const Joined t = {rows, q0, row0, range, end - range + 1};
      const int workgroup = (mine - range) * p.groups + index, workgroups = (end - range) * p.groups;
      const int spans = t.rows * (kDv / kSpan);
      if (t.parts >= kManyParts && spans <= kSpanTurns * workgroups) {
        for (int u = workgroup; u < spans; u += workgroups)
          join_span(p, t, lds, u / (kDv / kSpan), u % (kDv / kSpan));
      } else if (t.parts <= 2) {
        join_rows<4>(p, t, 4 * workgroup + wave, 4 * workgroups);
      } else if (t.parts <= 4) {
        join_rows<2>(p, t, 4 * workgroup + wave, 4 * workgroups);
      } else {
        join_rows<1>(p, t, 4 * workgroup + wave, 4 * workgroups);
      }
    }
  }
  const int behind = p.cu == nullptr ? p.T : p.B == 0 ? 0 : min(max(p.cu[p.B], 0), p.T);
  const int64_t total = (int64_t)(p.T - behind) * p.H;
  for (int64_t u = (int64_t)blockIdx.x * 4 + wave; u < total; u += (int64_t)gridDim.x * 4) {
    const int token = behind + (int)(u / p.H), head = (int)(u % p.H);
    *reinterpret_cast<Global<bf16x8>>(p.o + token * p.o_st + head * p.o_sh + 8 * lane) = bf16x8{};
    if (lane == 0 && p.lse != nullptr) p.lse[(int64_t)token * p.H + head] = kNegInf;
  }
}

// Ranges of a call: one per CU, as many as its work can fill at most.
int64_t chunk_ranges(int64_t T, int64_t B, int64_t H, int64_t max_pages) {
  const int64_t most = chunk_weight(T, B, H, max_pages, kNarrowRows);
  return std::max<int64_t>(1, std::min<int64_t>(std::min(device_cu_count(), kMaxRanges), (most + kMinWidth - 1) / kMinWidth));
}
int64_t chunk_bytes(int64_t ranges) { return ranges * (2 * kRows * (int64_t)(kDv + 1) * 4 + (int64_t)sizeof(RangeLink)); }

}  // namespace
}  // namespace dmla

using namespace dmla;

extern "C" int64_t dmla_chunk_paged_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t max_pages_per_seq) {
  if (T <= 0 || B <= 0 || H <= 0 || max_pages_per_seq <= 0 || T > ((int64_t)1 << 30) || H > ((int64_t)1 << 16) ||
      B > ((int64_t)1 << 20) || T * H > ((int64_t)1 << 30) || max_pages_per_seq > ((int64_t)1 << 20))
    return 0;
  return chunk_bytes(chunk_ranges(T, B, H, max_pages_per_seq));
}

extern "C" int dmla_chunk_paged(const void* q, const void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                                const int32_t* cu_seqlens_q, void* o, float* lse, int64_t T, int64_t B, int64_t H,
                                int64_t d_qk, int64_t d_v, int64_t num_pages, int64_t max_pages_per_seq, int64_t q_st,
                                int64_t q_sh, int64_t kv_sp, int64_t kv_ss, int64_t bt_sb, int64_t o_st, int64_t o_sh,
                                float softmax_scale, int causal, void* workspace, int64_t workspace_bytes,
                                dmla_stream_t stream) {
  clear_error();
  const char* what = "dmla_chunk_paged";
  if (T < 0 || B < 0 || H < 0 || num_pages < 0 || max_pages_per_seq < 0)
    return fail(DMLA_ERR_INVALID_ARG, "%s: negative size", what);
  if (cu_seqlens_q == nullptr && T != B)
    return fail(DMLA_ERR_INVALID_ARG, "%s: without cu_seqlens_q there is one query per sequence", what);
  if (d_qk != kDqk || d_v != kDv)
    return fail(DMLA_ERR_UNSUPPORTED, "%s: only d_qk=576, d_v=512 is compiled (got %lld, %lld)", what, (long long)d_qk,
                (long long)d_v);
  if (!(softmax_scale > 0.f) || !__builtin_isfinite(softmax_scale))
    return fail(DMLA_ERR_INVALID_ARG, "%s: softmax_scale must be finite and > 0", what);
  if (!aligned16(q) || !aligned16(kv_pool) || !aligned16(o))
    return fail(DMLA_ERR_INVALID_ARG, "%s: q, kv_pool and o must be 16-byte aligned", what);
  if (!mult8(q_st) || !mult8(q_sh) || !mult8(kv_sp) || !mult8(kv_ss) || !mult8(o_st) || !mult8(o_sh))
    return fail(DMLA_ERR_INVALID_ARG, "%s: strides must be multiples of 8 elements", what);
  if (kv_ss < kDqk || kv_sp < kv_ss * kPage || kv_ss * 2 * kPage >= ((int64_t)1 << 31))
    return fail(DMLA_ERR_INVALID_ARG, "%s: kv_pool strides out of range", what);
  if (bt_sb < max_pages_per_seq) return fail(DMLA_ERR_INVALID_ARG, "%s: block_table row stride < max_pages_per_seq", what);
  if (H > ((int64_t)1 << 16) || B > ((int64_t)1 << 20) || T > ((int64_t)1 << 30) || T * H > ((int64_t)1 << 30) ||
      max_pages_per_seq > ((int64_t)1 << 20) || num_pages > 0x7fffffff)
    return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  if (T == 0 || H == 0) return DMLA_OK;
  if (!q || !o || (B > 0 && !cache_seqlens) || (B > 0 && max_pages_per_seq > 0 && !block_table) || (num_pages > 0 && !kv_pool))
    return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  if (B > 0 && (num_pages == 0 || max_pages_per_seq == 0))
    return fail(DMLA_ERR_INVALID_ARG, "%s: empty page pool or block table", what);
  ChunkParams p = {};
  p.q = (Global<const bf16>)q;
  p.kv = (Global<const char>)kv_pool;
  p.block_table = (Global<const int32_t>)block_table;
  p.seqlens = (Global<const int32_t>)cache_seqlens;
  p.cu = (Global<const int32_t>)cu_seqlens_q;
  p.o = (Global<bf16>)o;
  p.lse = (Global<float>)lse;
  p.q_st = q_st; p.q_sh = q_sh; p.kv_sp = 2 * kv_sp; p.kv_ss = 2 * kv_ss; p.bt_sb = bt_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.T = (int)T; p.B = (int)B; p.H = (int)H; p.num_pages = (int)num_pages; p.max_pages = (int)max_pages_per_seq;
  p.causal = causal ? 1 : 0;
  p.hdiv = make_fastdiv((unsigned)H);
  p.scale_log2 = softmax_scale * kLog2e;
  p.n_ranges = (int)chunk_ranges(T, B, H, max_pages_per_seq);
  p.two_by_h = 2.0f / (float)H;
  p.weight_shift = chunk_weight_shift(T, B, H, max_pages_per_seq);
  p.weight_scale = std::ldexp(1.0f, -p.weight_shift);
  // A combine workgroup holds 110 registers a lane, so 4 per CU run at once; a call of few row tiles takes 8 (one of
  // 100000 tokens x 128 heads 17.8 -> 15.3 us), more would only queue (64 sequences x 16 heads 6.9 with 4, 10.9 with 8).
  p.groups = (T * H / kRows + std::min(B, T)) * 8 <= p.n_ranges ? 8 : 4;
  if (B == 0) {   // nothing but queries behind the last sequence
    p.n_ranges = 0;
    hipLaunchKernelGGL(chunk_combine_kernel, dim3(256), dim3(256), 0, (hipStream_t)stream, p);
    return check_launch(what);
  }
  const int64_t need = chunk_bytes(p.n_ranges);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DMLA_ERR_WORKSPACE, "%s: workspace of %lld bytes needed (got %lld)", what, (long long)need,
                (long long)workspace_bytes);
  if (!aligned16(workspace)) return fail(DMLA_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", what);
  p.part_o = (Global<float>)workspace;
  p.part_lse = p.part_o + (int64_t)p.n_ranges * 2 * kRows * kDv;
  p.links = (Global<RangeLink>)(p.part_lse + (int64_t)p.n_ranges * 2 * kRows);
  hipLaunchKernelGGL(chunk_kernel, dim3((unsigned)((p.n_ranges + 7) / 8 * 8)), dim3(kThreads), 0, (hipStream_t)stream, p);
  hipLaunchKernelGGL(chunk_combine_kernel, dim3((unsigned)(p.n_ranges * p.groups)), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch(what);
}
