// The account of attention weight: mass[b, t] += sum_h exp(scale q_h . k_t - lse_h), the weight that the
// heads of a decode step gave each cached token, from the step's queries and log-sum-exps, over bf16 or
// 4-bit pages (dmla_q4.h).  What the eviction ranks tokens by.  No reference counterpart.
//
// A second pass over the keys is what the sum needs: a token's weight is known only once its heads'
// sums over the whole context are.  Per token it reads the row and does 2 x 576 flops per head, so up to
// 128 heads the rows' bytes bound it (1152 bytes at 6.2 TB/s 0.19 ns, 147 kflop at 2.1 PFLOP/s 0.07 ns).
//
// MI355X design:
//  * One workgroup of eight waves per CU streams key tiles through LDS, in steps of kKP blocks of 32 tokens.  Eight
//    waves take kHW blocks of 32 heads x kKP blocks of keys: two waves per SIMD, so that one's LDS reads and
//    exponentials run beside the other's MFMAs.
//  * A wave holds its heads' queries in registers (144) as the MFMA's row operand, keys are its columns, so a
//    lane ends with one key's scores of 16 heads and the sum over heads is in-lane adds and a lane swap.
//  * Every token belongs to one workgroup and its sum to one thread: no atomics, the same bits every time.
//    Measured: 64 sequences of 1024 to 8192 tokens x 128 heads on bf16 pages 76 us, 4.7 TB/s (four waves, each with
//    half the registers idle, 115); one of 5000 tokens 10.1 us; 16 sequences x 16 heads on 4-bit pages 13.2 us.
//    The sums of kChunk tokens wait in LDS, beside the account's old values, which are copied there like keys:
//    a load into registers would wait for every copy before it.
#include <algorithm>
#include <type_traits>

#include "dmla_host.h"
#include "dmla_q4.h"
#include "dmla_ranges.h"

namespace dmla {
namespace {

constexpr int kDqk = 576, kPage = 64;
constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kChunk = 512;   // tokens whose sums wait in LDS
static_assert(kChunk == kThreads, "a token per thread");

struct MassParams {
  const bf16* q;
  const char* kv;
  const int32_t* block_table;
  const int32_t* seqlens;
  const float* lse;      // [B, H]
  float* mass;
  int64_t q_sb, q_sh, kv_sp, kv_ss, bt_sb, m_sb;   // kv strides in bytes
  int B, H, num_pages, max_pages;
  int n_ranges, min_width;
  float scale_log2;
};

// kQ4: 4-bit pages, else bf16 pages (the tile layout of dmla_common.h).  kPages pages of 64 tokens a step.
template <bool kQ4, int kPages>
struct Tile {
  static constexpr int kTokens = kPage * kPages;
  static constexpr int kKP = 2 * kPages, kHW = kWaves / kKP;             // key and head blocks
  static constexpr int kBlockBytes = kQ4 ? 32 * kQ4RowBytes : 9 * kGroupBytes;
  static constexpr int kBytes = kKP * kBlockBytes;
  static constexpr int kSlots = kQ4 ? (kPages == 1 ? 5 : 3) : 2;
  static constexpr int kCopies = kQ4 ? kBytes / 1024 : 9 * kWaves;       // of a step, all waves
  static constexpr int kMost = (kCopies + kWaves - 1) / kWaves, kLeast = kCopies / kWaves;   // of a wave
  static constexpr int kCost = kQ4 ? 4 / kPages : 4;                     // a segment's start and end, in steps
  static constexpr bool kOneRound = kHW * 36 * 1024 <= kSlots * kBytes;   // all queries fit the ring at once
  static constexpr int kQBytes = (kOneRound ? 36 : 24) * 1024;           // queries of a head block in a round
  static_assert(kHW * kQBytes <= kSlots * kBytes, "the queries pass through the ring");
};

// Scores of a wave's 32 heads (rows: head 8 (i / 4) + 4 hl + i % 4) with the 32 keys of a tile (lane l: key l % 32).
template <bool kQ4>
__device__ __forceinline__ f32x16 scores(const bf16x8 (&q)[kQ4Steps], unsigned tile, int lane) {
  const int l32 = lane & 31, hl = lane >> 5;
  f32x16 s = {};
  if constexpr (kQ4) {
    const DMLA_LDS char* row = lds_ptr<const char>(lds_sum(l32 * kQ4RowBytes, tile));
    const u32x4 scales = q4_key_scales(row, hl);
    static_for<8>([&](auto a_tag) {
      constexpr int a = decltype(a_tag)::value;
      const u32x4 w = q4_key_codes(row, hl, a);
      const float sc = q4_key_scale<a>(scales);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = mfma32_bf16(q[4 * a + j], q4_octet(w[j], sc), s);
    });
#pragma unroll
    for (int c = 0; c < 4; ++c) s = mfma32_bf16(q[kQ4LatentSteps + c], q4_key_rope(row, hl, c), s);
  } else {
    constexpr int kDepth = 5;   // operands read ahead
    const unsigned at = lds_sum(tile_chunk_off(l32, hl), tile);
    bf16x8 k[kDepth];
    auto read = [&](int c) {
      k[c % kDepth] = *lds_ptr<const bf16x8>((at ^ (32 * (c & 3))) + (c >> 2) * kGroupBytes);   // tile_chunk_off(l32, 2 c + hl)
    };
#pragma unroll
    for (int c = 0; c < kDepth; ++c) read(c);
    static_for<kQ4Steps>([&](auto c_tag) {
      constexpr int c = decltype(c_tag)::value;
      in_order();
      s = mfma32_bf16(q[c], k[c % kDepth], s);
      if constexpr (c + kDepth < kQ4Steps) read(c + kDepth);
    });
  }
  return s;
}

struct Lds {
  unsigned ring;
  DMLA_LDS float* sums;   // [kHW][kChunk]
  DMLA_LDS float* old;    // [kChunk]
};

template <bool kQ4, int kPages>
__device__ __forceinline__ void mass_segment(const MassParams& p, int b, int t0, int t1, int ctx, const Lds& lds) {
  using T = Tile<kQ4, kPages>;
  constexpr int kKP = T::kKP, kHW = T::kHW, kSlots = T::kSlots;
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int hw = wave / kKP, kp = wave % kKP;   // with few heads, the waves at work sit on different SIMDs
  int page0 = 0, pages = 0;   // lane i: page page0 + i of the sequence
  auto fetch_pages = [&](int from) {
    page0 = uniform(from);
    const int i = page0 + fresh_lane_id();
    pages = i * kPage < ctx ? p.block_table[b * p.bt_sb + i] : 0;
    asm volatile("" : "+v"(pages));   // waited for here, in the rare branch, and not by every reader
  };
  unsigned bad_bits = 0;   // bit kPages (slot) + j: page j of the step in the slot lies outside the pool
  // This wave's share of a step's copies.  Rows past the end re-read a row of the sequence.
  auto copy_step = [&](int t) {
    const int slot = (t - t0) % kSlots;
    const unsigned dst = lds.ring + (unsigned)(slot * T::kBytes);
    const int ln = fresh_lane_id();
    const char* src[kPages];
    int valid[kPages];
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      int at = t * kPages + j;
      valid[j] = ctx - at * kPage;
      if (valid[j] <= 0) {   // a second page that the sequence does not reach: the first one's first row
        at = t * kPages;
        valid[j] = 1;
      }
      if (at - page0 >= 64) fetch_pages(page0 + 64);
      int page = __builtin_amdgcn_readlane(pages, uniform((at - page0) & 63));
      const bool bad = page < 0 || page >= p.num_pages;
      const unsigned bit = 1u << (kPages * slot + j);
      bad_bits = bad ? bad_bits | bit : bad_bits & ~bit;   // its tokens are left out below
      src[j] = p.kv + (bad ? 0 : page) * p.kv_sp;
    }
    if constexpr (kQ4) {
      constexpr int kPageCopies = kPage * kQ4RowBytes / 1024;
#pragma unroll
      for (int i = 0; i < T::kMost; ++i) {
        const int k = i * kWaves + wave;
        if (k >= T::kCopies) continue;
        const int j = kPages > 1 && k >= kPageCopies ? kPages - 1 : 0;
        const int c = (k - j * kPageCopies) * 64 + ln;
        unsigned off = 16u * c;
        if (valid[j] < kPage) {
          const int row = c / kQ4Chunks;
          off = row < valid[j] ? off : 16u * (c - row * kQ4Chunks);
        }
        dma16(src[j], off, dst + k * 1024);
      }
    } else {
      const int row = 8 * wave + (ln >> 3);
      const unsigned off = 16u * ((ln & 7) ^ swz(row & 15)) + (row < valid[0] ? (unsigned)(row * (int)p.kv_ss) : 0u);
#pragma unroll
      for (int cg = 0; cg < 9; ++cg)
        dma16(src[0] + cg * 128, off, dst + (wave / 4) * T::kBlockBytes + cg * kGroupBytes + (wave & 3) * 1024);
    }
  };
  // The copies of step t have landed; those of the kSlots - 1 steps after it may be on their way.
  auto await_copies = [&](int t) {
    constexpr int kFlight = kSlots - 1;
    if (t + kFlight >= t1) wait_vm<0>();   // the last steps have fewer behind them
    else if (wave < T::kCopies % kWaves || T::kCopies % kWaves == 0) wait_vm<kFlight * T::kMost>();
    else wait_vm<kFlight * T::kLeast>();
  };

  for (int h0 = 0; h0 < p.H; h0 += 32 * kHW) {
    const int hb = h0 + 32 * hw;
    const bool idle = hb >= p.H;   // no heads for this wave: it copies
    // Queries through the ring, 8 rows x 128 bytes a copy (as operands they would be 32 rows x 32 bytes a load),
    // in one round or two of 64-dim blocks; the waves of a head block share the copies.
    bf16x8 q[kQ4Steps];
    const unsigned stage = lds.ring + hw * T::kQBytes;
    auto queries = [&](auto first_tag, auto n_tag) {
      constexpr int kFirst = decltype(first_tag)::value, kN = decltype(n_tag)::value;
      const int ln = fresh_lane_id();
#pragma unroll
      for (int i = 0; i < 4 * kN / kKP; ++i) {
        const int k = i * kKP + kp, g = k / kN, d = k - g * kN;
        const int head = min(hb + 8 * g + (ln >> 3), p.H - 1);
        const bf16* src = p.q + b * p.q_sb + head * p.q_sh + 64 * (kFirst + d) + 8 * ((ln & 7) ^ (ln >> 3));
        if (!idle) dma16_addr(src, stage + k * 1024);
      }
      wait_vm<0>();
      __syncthreads();
      const unsigned row = stage + kN * 1024 * (l32 >> 3) + 128 * (l32 & 7);
#pragma unroll
      for (int c = 4 * kFirst; c < 4 * (kFirst + kN); ++c) {
        const int u = kQ4 ? q4_operand_unit(hl, c) : 2 * c + hl;
        q[c] = lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(
            static_cast<uintptr_t>(row + (c / 4 - kFirst) * 1024 + 16 * ((u & 7) ^ (l32 & 7)))));
      }
      wait_lds();
      __syncthreads();
    };
    if constexpr (T::kOneRound) {
      queries(std::integral_constant<int, 0>{}, std::integral_constant<int, 9>{});
    } else {
      queries(std::integral_constant<int, 0>{}, std::integral_constant<int, 6>{});
      queries(std::integral_constant<int, 6>{}, std::integral_constant<int, 3>{});
    }
    fetch_pages(t0 * kPages);
    for (int t = t0; t < t0 + kSlots && t < t1; ++t) copy_step(t);
    float lse2[16];   // of the lane's rows, in log2 units
    bool on[16];      // a head with lse = -inf, or none at all, adds nothing, whatever its score (a lane mask in SGPRs)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int head = hb + 8 * (i >> 2) + 4 * hl + (i & 3);
      const float v = head < p.H ? p.lse[(int64_t)b * p.H + head] : kNegInf;
      lse2[i] = v * kLog2e;
      on[i] = v != kNegInf;
    }
    const int n_hw = min(kHW, (p.H - h0 + 31) / 32);
    float* mass = p.mass + b * p.m_sb;
    int chunk0 = t0;
    for (int t = t0; t < t1; ++t) {
      await_copies(t);
      __syncthreads();   // step t has landed; the sums of the chunk before have been read
      const int slot = (t - t0) % kSlots;
      if (t == chunk0) {   // one value of the account for each thread of the workgroup
        const int at = min(t * T::kTokens + (int)threadIdx.x, ctx - 1);
        dma4(mass, 4u * at, lds_addr(lds.old) + wave * 256);
      }
      if (!idle) {
        const unsigned tile = lds.ring + (unsigned)(slot * T::kBytes + kp * T::kBlockBytes);
        const f32x16 s = scores<kQ4>(q, tile, lane);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float w = fast_exp2(__builtin_fmaf(s[i], p.scale_log2, -lse2[i]));
          sum += on[i] ? w : 0.f;
        }
        sum = half_sum(sum);
        const bool bad = (bad_bits >> (kPages * slot + kp / 2) & 1) != 0;
        if (hl == 0) lds.sums[hw * kChunk + (t - chunk0) * T::kTokens + 32 * kp + l32] = bad ? 0.f : sum;
      }
      const bool last = t + 1 == t1 || (t + 1 - chunk0) * T::kTokens == kChunk;
      // The account's values: they are older than the copies of step chunk0 + kSlots, which landed above if that is
      // step t or before it.
      if (last && t - chunk0 < kSlots) wait_vm<0>();
      __syncthreads();          // the slot has been read, the sums are written
      if (last) {
        const int i = threadIdx.x, at = chunk0 * T::kTokens + i;
        if (at < min((t + 1) * T::kTokens, ctx)) {
          float add = 0.f;
          for (int w = 0; w < n_hw; ++w) add += lds.sums[w * kChunk + i];
          mass[at] = lds.old[i] + add;
        }
        chunk0 = t + 1;
      }
      if (t + kSlots < t1) copy_step(t + kSlots);
    }
    wait_vm<0>();      // the account is written before the next heads read it
    __syncthreads();
  }
}

template <bool kQ4, int kPages>
__global__ __launch_bounds__(kThreads, 1) void mass_kernel(MassParams p) {
  using T = Tile<kQ4, kPages>;
  __shared__ __attribute__((aligned(1024))) char ring[T::kSlots * T::kBytes];
  __shared__ __attribute__((aligned(16))) float sums[T::kHW * kChunk];
  __shared__ __attribute__((aligned(16))) float old[kChunk];
  __shared__ __attribute__((aligned(16))) RangeLds ranges;
  const Lds lds = {lds_addr((DMLA_LDS char*)ring), (DMLA_LDS float*)sums, (DMLA_LDS float*)old};
  for_each_segment<T::kTokens, T::kCost>(
      p.seqlens, p.B, p.max_pages * kPage, p.n_ranges, p.min_width, blockIdx.x, ranges,
      [&](int b, int t0, int t1, int ctx, int) { mass_segment<kQ4, kPages>(p, b, t0, t1, ctx, lds); }, [](int, int, int) {});
}

}  // namespace
}  // namespace dmla

using namespace dmla;

extern "C" int dmla_attn_mass(const void* q, const void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                              const float* lse, float* mass, int64_t B, int64_t H, int64_t d_qk, int64_t num_pages,
                              int64_t max_pages_per_seq, int64_t mass_len, int64_t q_sb, int64_t q_sh, int64_t kv_sp,
                              int64_t kv_ss, int64_t bt_sb, int64_t m_sb, int q4, float softmax_scale,
                              dmla_stream_t stream) {
  clear_error();
  // (Of an empty call any address does: empty tensors have none.)
  if (B != 0 && H != 0 && (!q || !kv_pool || !block_table || !cache_seqlens || !lse || !mass))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: null pointer argument");
  if (B < 0 || H < 0 || num_pages < 0 || max_pages_per_seq < 0 || mass_len < 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: negative size");
  if (d_qk != kDqk) return fail(DMLA_ERR_UNSUPPORTED, "dmla_attn_mass: only d_qk=576 is compiled (got %lld)", (long long)d_qk);
  if (!(softmax_scale > 0.f) || !__builtin_isfinite(softmax_scale))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: softmax_scale must be finite and > 0");
  if (!aligned16(q) || !aligned16(kv_pool))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: q and kv_pool must be 16-byte aligned");
  if (!mult8(q_sb) || !mult8(q_sh)) return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: q strides must be multiples of 8 elements");
  if (kv_sp % 16 != 0 || kv_ss % 16 != 0 || kv_ss < (q4 ? kQ4RowBytes : 2 * kDqk) || kv_sp < kPage * kv_ss ||
      kv_ss * kPage >= ((int64_t)1 << 31))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: kv_pool strides must be multiples of 16 bytes and cover a row / page");
  if (q4 && kv_ss != kQ4RowBytes)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_attn_mass: rows of a 4-bit page must follow each other");
  if (bt_sb < max_pages_per_seq)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: block_table row stride < max_pages_per_seq");
  if (H > ((int64_t)1 << 16) || B > ((int64_t)1 << 20) || max_pages_per_seq > ((int64_t)1 << 24) || num_pages > 0x7fffffff ||
      B * (max_pages_per_seq * 2 + 16) >= ((int64_t)1 << 31))
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_attn_mass: size too large");
  if (mass_len < max_pages_per_seq * kPage || m_sb < mass_len)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: mass rows must cover the block table's tokens");
  if (B == 0 || H == 0) return DMLA_OK;
  if (num_pages == 0 || max_pages_per_seq == 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_attn_mass: empty page pool or block table");
  MassParams p = {};
  p.q = static_cast<const bf16*>(q);
  p.kv = static_cast<const char*>(kv_pool);
  p.block_table = block_table;
  p.seqlens = cache_seqlens;
  p.lse = lse;
  p.mass = mass;
  p.q_sb = q_sb; p.q_sh = q_sh; p.kv_sp = kv_sp; p.kv_ss = kv_ss; p.bt_sb = bt_sb; p.m_sb = m_sb;
  p.B = (int)B; p.H = (int)H; p.num_pages = (int)num_pages; p.max_pages = (int)max_pages_per_seq;
  p.n_ranges = device_cu_count();
  p.min_width = 1;   // one sequence of 5000 tokens: 10.1 us, 15.5 with 2 steps a workgroup at least, 20 with 4
  p.scale_log2 = softmax_scale * kLog2e;
  const dim3 grid((unsigned)p.n_ranges);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, (hipStream_t)stream, p); };
  // bf16 rows bound the pass whatever the heads.  Of 4-bit rows, up to 64 heads, four blocks of keys at once keep
  // more waves busy: 64 sequences of 8192 tokens 44 us with 16 heads, 56 with 64 (two blocks: 60 and 63); 128 heads
  // take 102 (86).
  if (!q4) launch(mass_kernel<false, 1>);
  else if (H > 64) launch(mass_kernel<true, 1>);
  else launch(mass_kernel<true, 2>);
  return check_launch("dmla_attn_mass");
}
