// The account of attention weight: mass[b, t] += sum_h exp(scale q_h . k_t - lse_h), the weight that the
// heads of a decode step gave each cached token, from the step's queries and log-sum-exps, over bf16 or
// 4-bit pages (dmla_q4.h).  What the eviction ranks tokens by.  No reference counterpart.
//
// A second pass over the keys is what the sum needs: a token's weight is known only once its heads'
// sums over the whole context are.  Per token it reads the row and does 2 x 576 flops per head, so up to
// 128 heads the rows' bytes bound it (1152 bytes at 6.2 TB/s 0.19 ns, 147 kflop at 2.1 PFLOP/s 0.07 ns).
// One workgroup of four waves per CU streams key tiles through LDS; a wave holds up to 32 heads' queries
// in registers as the MFMA's row operand, keys are its columns, so a lane ends with one key's scores of
// 16 heads and the sum over heads is in-lane adds and a lane swap.  Every token belongs to
// one workgroup and its sum to one thread: no atomics, the same bits every time.
#include <algorithm>
#include <type_traits>

#include "dmla_host.h"
#include "dmla_q4.h"
#include "dmla_ranges.h"

namespace dmla {
namespace {

constexpr int kDqk = 576, kPage = 64;
constexpr int kWaves = 4, kThreads = 64 * kWaves;
static_assert(kThreads == kRangeThreads, "one workgroup cuts the ranges");
constexpr int kChunk = 1024;   // tokens whose sums wait in LDS

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

// kQ4: 4-bit pages, tiles of 64 tokens; else bf16 pages, tiles of 32 (the layout of dmla_common.h).
template <bool kQ4>
struct Tile {
  static constexpr int kTokens = kQ4 ? 64 : 32;
  static constexpr int kBytes = kQ4 ? kTokens * kQ4RowBytes : 9 * kGroupBytes;
  static constexpr int kBlocks = kTokens / 32;
  static constexpr int kSlots = kQ4 ? 5 : 3;
  static constexpr int kCost = kQ4 ? 3 : 4;   // a segment's start and end, in tiles
};

// One step of the score product of 32 heads (rows) with 32 keys: the query operand, and the keys' from
// the tile's rows 32 kb .. +31.
__device__ __forceinline__ bf16x8 query_operand_bf16(const bf16* q, int hl, int c) {
  return *reinterpret_cast<const bf16x8*>(q + 16 * c + 8 * hl);
}
template <bool kQ4>
__device__ __forceinline__ f32x16 scores(const bf16x8 (&q)[kQ4Steps], const DMLA_LDS char* tile, int kb, int lane) {
  const int l32 = lane & 31, hl = lane >> 5;
  f32x16 s;
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = 0.f;
  if constexpr (kQ4) {
    const DMLA_LDS char* row = tile + (32 * kb + l32) * kQ4RowBytes;
    const u32x2 scales = q4_key_scales(row, hl);
    auto block = [&](auto a_tag) {
      constexpr int kA = decltype(a_tag)::value;
      const u32x4 w = q4_key_codes(row, hl, kA);
      const float sc = q4_key_scale<kA>(scales);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = mfma32_bf16(q[4 * kA + j], q4_octet(w[j], sc), s);
    };
    block(std::integral_constant<int, 0>{});
    block(std::integral_constant<int, 1>{});
    block(std::integral_constant<int, 2>{});
    block(std::integral_constant<int, 3>{});
    block(std::integral_constant<int, 4>{});
    block(std::integral_constant<int, 5>{});
    block(std::integral_constant<int, 6>{});
    block(std::integral_constant<int, 7>{});
#pragma unroll
    for (int c = 0; c < 4; ++c) s = mfma32_bf16(q[kQ4LatentSteps + c], q4_key_rope(row, hl, c), s);
  } else {
#pragma unroll
    for (int c = 0; c < kQ4Steps; ++c)
      s = mfma32_bf16(q[c], lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(tile + tile_chunk_off(l32, 2 * c + hl))), s);
  }
  return s;
}

template <bool kQ4, int kHW>
__device__ __forceinline__ void mass_segment(const MassParams& p, int b, int t0, int t1, int ctx, DMLA_LDS char* ring,
                                             DMLA_LDS float* sums) {
  using T = Tile<kQ4>;
  constexpr int kKP = kWaves / kHW;
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int hw = wave % kHW, kp = wave / kHW;
  const unsigned ring_addr = lds_addr(ring);
  constexpr int kPerPage = kPage / T::kTokens;
  int page0, pages;
  auto fetch_pages = [&](int from) {
    page0 = from;
    const int i = page0 + lane;
    pages = i < (t1 + kPerPage - 1) / kPerPage ? p.block_table[b * p.bt_sb + i] : 0;
  };
  auto page_of = [&](int t) {
    if (t / kPerPage - page0 >= 64) fetch_pages(page0 + 64);
    return __builtin_amdgcn_readlane(pages, (t / kPerPage - page0) & 63);
  };
  // This wave's share of a tile's copies.  Rows past the end re-read the tile's first row.
  const int dma_row = 8 * wave + (lane >> 3);                            // bf16 tiles: rows 8 wave ..
  const unsigned dma_col = 16u * ((lane & 7) ^ swz(dma_row & 15));
  auto copy_tile = [&](int t) {
    int page = page_of(t);
    page = page < 0 || page >= p.num_pages ? 0 : page;   // its tokens are left out below
    const unsigned dst = ring_addr + (unsigned)(((t - t0) % T::kSlots) * T::kBytes);
    const int valid = ctx - t * T::kTokens;
    const char* src = p.kv + page * p.kv_sp + (int64_t)(t % kPerPage) * T::kTokens * p.kv_ss;
    if constexpr (kQ4) {
#pragma unroll
      for (int k = 0; k < T::kBytes / 1024; ++k) {
        if (k % kWaves != wave) continue;
        if (valid >= T::kTokens) {
          dma16(src + k * 1024, 16u * lane, dst + k * 1024);
        } else {
          const int i = k * 64 + lane, row = i / kQ4Chunks, col = i - row * kQ4Chunks;
          dma16(src, 16u * (row < valid ? i : col), dst + k * 1024);
        }
      }
    } else {
      const unsigned off = dma_col + (dma_row < valid ? (unsigned)(dma_row * (int)p.kv_ss) : 0u);
#pragma unroll
      for (int cg = 0; cg < 9; ++cg) dma16(src + cg * 128, off, dst + cg * kGroupBytes + wave * 1024);
    }
  };
  constexpr int kFlight = T::kSlots - 2;
  constexpr int kTotal = kQ4 ? T::kBytes / 1024 : 9 * kWaves;   // copies of a tile, all waves

  for (int h0 = 0; h0 < p.H; h0 += 32 * kHW) {
    const int hb = h0 + 32 * hw;
    const bf16* q_row = p.q + b * p.q_sb + min(hb + l32, p.H - 1) * p.q_sh;
    bf16x8 q[kQ4Steps];
#pragma unroll
    for (int c = 0; c < kQ4Steps; ++c) q[c] = kQ4 ? q4_query_operand(q_row, hl, c) : query_operand_bf16(q_row, hl, c);
    float lse2[16];   // of the lane's rows, in log2 units; a head with no keys, or none at all, has weight 0
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int head = hb + 8 * (i >> 2) + 4 * hl + (i & 3);
      const float v = head < p.H ? p.lse[(int64_t)b * p.H + head] : kNegInf;
      lse2[i] = v == kNegInf ? -kNegInf : v * kLog2e;
    }
    fetch_pages(t0 / kPerPage);
    for (int t = t0; t < t0 + T::kSlots - 1 && t < t1; ++t) copy_tile(t);
    int use_page0 = t0 / kPerPage - 64, use_pages = 0;   // the pages of the tiles in work (validity)
    int chunk0 = t0;
    for (int t = t0; t < t1; ++t) {
      if (t + kFlight >= t1 - 1) wait_vm<0>();
      else if (wave < kTotal % kWaves || kTotal % kWaves == 0) wait_vm<kFlight*((kTotal + kWaves - 1) / kWaves)>();
      else wait_vm<kFlight*(kTotal / kWaves)>();
      wait_lds();
      __syncthreads();   // tile t has landed, and nobody reads the slot refilled next
      if (t + T::kSlots - 1 < t1) copy_tile(t + T::kSlots - 1);
      if (t / kPerPage - use_page0 >= 64) {
        use_page0 = t / kPerPage;
        const int i = use_page0 + lane;
        use_pages = i < (t1 + kPerPage - 1) / kPerPage ? p.block_table[b * p.bt_sb + i] : 0;
      }
      const int page = __builtin_amdgcn_readlane(use_pages, (t / kPerPage - use_page0) & 63);
      const bool bad = page < 0 || page >= p.num_pages;
      const DMLA_LDS char* tile = ring + ((t - t0) % T::kSlots) * T::kBytes;
#pragma unroll
      for (int kb = 0; kb < T::kBlocks; ++kb) {
        if ((t * T::kBlocks + kb) % kKP != kp) continue;   // the waves with the same heads take turns
        const f32x16 s = scores<kQ4>(q, tile, kb, lane);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += fast_exp2(__builtin_fmaf(s[i], p.scale_log2, -lse2[i]));
        sum = half_sum(sum);
        if (hl == 0) sums[hw * kChunk + (t - chunk0) * T::kTokens + 32 * kb + l32] = bad ? 0.f : sum;
      }
      if (t + 1 == t1 || (t + 1 - chunk0) * T::kTokens == kChunk) {
        __syncthreads();
        const int base = chunk0 * T::kTokens, n = min((t + 1) * T::kTokens, ctx) - base;
        for (int i = threadIdx.x; i < n; i += kThreads) {
          float add = 0.f;
#pragma unroll
          for (int w = 0; w < kHW; ++w) add += sums[w * kChunk + i];
          p.mass[b * p.m_sb + base + i] += add;
        }
        __syncthreads();   // read out before the next chunk's sums, and no copy waits behind these stores
        chunk0 = t + 1;
      }
    }
  }
}

template <bool kQ4, int kHW>
__global__ __launch_bounds__(kThreads, 1) void mass_kernel(MassParams p) {
  using T = Tile<kQ4>;
  __shared__ __attribute__((aligned(1024))) char smem[T::kSlots * T::kBytes];
  __shared__ __attribute__((aligned(16))) float sum_mem[kHW * kChunk];
  __shared__ __attribute__((aligned(16))) RangeLds ranges;
  for_each_segment<T::kTokens, T::kCost>(
      p.seqlens, p.B, p.max_pages * kPage, p.n_ranges, p.min_width, blockIdx.x, ranges,
      [&](int b, int t0, int t1, int ctx, int) {
        mass_segment<kQ4, kHW>(p, b, t0, t1, ctx, (DMLA_LDS char*)smem, (DMLA_LDS float*)sum_mem);
      },
      [](int, int, int) {});
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
  if (!q || !kv_pool || !block_table || !cache_seqlens || !lse || !mass)
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
  p.min_width = 8;
  p.scale_log2 = softmax_scale * kLog2e;
  const dim3 grid((unsigned)p.n_ranges);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, (hipStream_t)stream, p); };
  if (q4) {
    if (H <= 32) launch(mass_kernel<true, 1>);
    else if (H <= 64) launch(mass_kernel<true, 2>);
    else launch(mass_kernel<true, 4>);
  } else {
    if (H <= 32) launch(mass_kernel<false, 1>);
    else if (H <= 64) launch(mass_kernel<false, 2>);
    else launch(mass_kernel<false, 4>);
  }
  return check_launch("dmla_attn_mass");
}
