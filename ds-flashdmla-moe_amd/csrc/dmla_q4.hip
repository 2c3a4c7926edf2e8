// The writer and the reader of the 4-bit paged latent cache (row format: dmla_q4.h):
//   * the append quantises new bf16 rows into pages through the block table;
//   * the gather reads a window of each sequence back as dense bf16 rows (what a chunked prefill over
//     cached context takes as k_lat, one length a call).
// No reference counterpart: the reference has no paged cache.
#include <algorithm>

#include "dmla_host.h"
#include "dmla_q4.h"

namespace dmla {
namespace {

constexpr int kD = 576, kLat = 512, kPage = 64;
constexpr int kWavesPerWG = 4;
constexpr int kBatch = 4;   // rows in flight per wave

struct Q4RowArgs {
  uint8_t* pool;
  const int32_t* block_table;
  const int32_t* seqlens;
  const int32_t* lens;     // append: new_lens; gather: starts (both nullable)
  bf16* rows;              // append: new_kv (read); gather: out
  int32_t* bad;            // append only; nullable
  int64_t kv_sp, bt_sb, r_sb, r_ss;
  int B, n;                // rows per sequence in `rows`
  int num_pages, max_pages;
  int each;                // rows of a wave at a time, at most kBatch
  FastDiv ndiv;            // division by n
};

// Page and row of position pos, -1 where the table has no valid page for it.
__device__ __forceinline__ int page_of(const Q4RowArgs& a, int b, int64_t pos) {
  const int64_t slot = pos / kPage;
  const int page = slot < a.max_pages ? a.block_table[b * a.bt_sb + slot] : -1;
  return page >= 0 && page < a.num_pages ? page : -1;
}

// (By value: a bit cast of a vector's element takes the vector's first.)
__device__ __forceinline__ bf16x2 as_bf16x2(unsigned w) { return __builtin_bit_cast(bf16x2, w); }

// A row at a time of a wave's kBatch: lane l holds values 8l .. 8l+7 (one 16-byte load, one 4-byte store of codes), four
// lanes share a block of 32, whose largest value meets in two quad swaps; lanes 0..7 move the rope.
// Bound: HBM (1152 bytes in, 400 out per row), and below some 20000 rows launch and latency: 8 x 2048 rows in 6.6 us,
// 64 x 8192 rows in 192 us, 4.2 TB/s.  kBatch rows per wave keep enough loads in flight (eight measured 13 % slower).
// Rows built in LDS and stored in 16-byte pieces instead of 256 + 16 x 1 + 128 bytes a row took the same time.
__global__ void __launch_bounds__(64 * kWavesPerWG) q4_append_kernel(Q4RowArgs a) {
  const int lane = lane_id();
  const int wave = uniform(threadIdx.x >> 6);
  const int64_t total = (int64_t)a.B * a.n;
  const int step = gridDim.x * kWavesPerWG;
  for (int64_t r0 = (int64_t)(blockIdx.x * kWavesPerWG + wave) * a.each; r0 < total; r0 += (int64_t)a.each * step) {
    bf16x8 x[kBatch], rope[kBatch];
    int64_t dst[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      dst[i] = -1;
      const int64_t r = r0 + i;
      if (i >= a.each || r >= total) continue;
      const int b = fast_div((int)r, a.ndiv), t = (int)r - b * a.n;
      if (a.lens != nullptr && t >= a.lens[b]) continue;
      const int64_t pos = (int64_t)max(a.seqlens[b], 0) + t;
      const int page = page_of(a, b, pos);
      if (page < 0) {
        if (a.bad != nullptr && lane == 0) a.bad[0] = 1;
        continue;
      }
      dst[i] = page * a.kv_sp + (pos % kPage) * kQ4RowBytes;
      const bf16* src = a.rows + b * a.r_sb + t * a.r_ss;
      x[i] = *reinterpret_cast<const bf16x8*>(src + 8 * lane);
      if (lane < 8) rope[i] = *reinterpret_cast<const bf16x8*>(src + kLat + 8 * lane);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (dst[i] < 0) continue;
      const u32x4 w = __builtin_bit_cast(u32x4, x[i]);
      unsigned top = 0;   // |value| as an integer: bf16 bits order like the values
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, max(w[j] << 16 & 0x7fffffffu, w[j] & 0x7fff0000u));
      top = max(top, (unsigned)__builtin_amdgcn_mov_dpp((int)top, 0xb1, 0xf, 0xf, true));   // quad_perm 1,0,3,2
      top = max(top, (unsigned)__builtin_amdgcn_mov_dpp((int)top, 0x4e, 0xf, 0xf, true));   // quad_perm 2,3,0,1
      const int sb = q4_scale_byte(top);
      const float scale = q4_scale(sb);
      unsigned codes = 0;
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, as_bf16x2(w[0]), scale, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, as_bf16x2(w[1]), scale, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, as_bf16x2(w[2]), scale, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, as_bf16x2(w[3]), scale, 3);
      if (sb == 255) codes = 0;
      uint8_t* row = a.pool + dst[i];
      *reinterpret_cast<unsigned*>(row + 4 * lane) = codes;
      if ((lane & 3) == 0) row[kQ4ScaleOff + (lane >> 2)] = (uint8_t)sb;
      if (lane < 8) *reinterpret_cast<bf16x8*>(row + kQ4RopeOff + 16 * lane) = rope[i];
    }
  }
}

// One wave per row, kBatch neighbouring rows at a time: lane l turns the codes of values 8l .. 8l+7 into 16 bytes of
// bf16; lanes 0..7 move the rope.  Rows at or past the sequence's length are zeros, rows on an invalid page are NaN.
// Bound: HBM (400 bytes in, 1152 out per row): 32 x 5000 rows, half of them cached, in 32 us, 6.8 TB/s.
// kStream: stores that do not stay in the caches, for outputs of kStreamBytes and more.  The 256 MiB of the last
// cache hold a smaller output until it is read, and a larger one only gets in the way there: 144 MiB of rows took
// 34 us (31.9 streamed) and 64 with a reader right behind (78), 162 MiB 40 (34) and 68 (85), 180 MiB 58 (39) and
// 77 (94), 198 MiB 80 (41) and 117 (103), 252 MiB 105 (53) and 173 (144).  What reads it is mostly attention,
// which the matrix units bound, so the gather's own time decides.
constexpr int64_t kStreamBytes = (int64_t)160 << 20;
template <bool kStream>
__global__ void __launch_bounds__(64 * kWavesPerWG) q4_gather_kernel(Q4RowArgs a) {
  const int lane = lane_id();
  const int wave = uniform(threadIdx.x >> 6);
  const int64_t total = (int64_t)a.B * a.n;
  const int step = gridDim.x * kWavesPerWG;
  const u32x4 nan4 = {0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  for (int64_t r0 = (int64_t)(blockIdx.x * kWavesPerWG + wave) * a.each; r0 < total; r0 += (int64_t)a.each * step) {
    unsigned codes[kBatch];
    int sb[kBatch], kind[kBatch];   // kind: 0 nothing to do, 1 a row, 2 zeros, 3 an invalid page
    u32x4 rope[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      kind[i] = 0;
      const int64_t r = r0 + i;
      if (i >= a.each || r >= total) continue;
      const int b = fast_div((int)r, a.ndiv), t = (int)r - b * a.n;
      const int64_t pos = (int64_t)(a.lens != nullptr ? max(a.lens[b], 0) : 0) + t;
      kind[i] = 2;
      if (pos >= min((int64_t)a.seqlens[b], (int64_t)a.max_pages * kPage)) continue;
      const int page = page_of(a, b, pos);
      kind[i] = 3;
      if (page < 0) continue;
      kind[i] = 1;
      const uint8_t* row = a.pool + page * a.kv_sp + (pos % kPage) * kQ4RowBytes;
      codes[i] = *reinterpret_cast<const unsigned*>(row + 4 * lane);
      sb[i] = row[kQ4ScaleOff + (lane >> 2)];
      if (lane < 8) rope[i] = *reinterpret_cast<const u32x4*>(row + kQ4RopeOff + 16 * lane);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (kind[i] == 0) continue;
      const int64_t r = r0 + i;
      const int b = fast_div((int)r, a.ndiv), t = (int)r - b * a.n;
      bf16* out = a.rows + b * a.r_sb + t * a.r_ss;
      u32x4 v = {0u, 0u, 0u, 0u}, p = v;
      if (kind[i] == 1) {
        const float s = q4_scale(sb[i]);
        v[0] = __builtin_bit_cast(unsigned, q4_pair<0>(codes[i], s));
        v[1] = __builtin_bit_cast(unsigned, q4_pair<1>(codes[i], s));
        v[2] = __builtin_bit_cast(unsigned, q4_pair<2>(codes[i], s));
        v[3] = __builtin_bit_cast(unsigned, q4_pair<3>(codes[i], s));
        p = rope[i];
      } else if (kind[i] == 3) {
        v = p = nan4;
      }
      u32x4* to = reinterpret_cast<u32x4*>(out + 8 * lane);
      if constexpr (kStream) {
        __builtin_nontemporal_store(v, to);
        if (lane < 8) __builtin_nontemporal_store(p, to + kLat / 8);
      } else {
        *to = v;
        if (lane < 8) to[kLat / 8] = p;
      }
    }
  }
}

// Checks shared by both entry points.
int q4_rows_validate(const char* what, const void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                     const void* rows, int64_t B, int64_t n, int64_t num_pages, int64_t max_pages_per_seq,
                     int64_t kv_sp, int64_t bt_sb, int64_t r_sb, int64_t r_ss) {
  // (Of an empty call any address does: empty tensors have none.)
  if (B != 0 && n != 0 && (!kv_pool || !block_table || !cache_seqlens || !rows))
    return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  if (B < 0 || n < 0 || num_pages < 0 || max_pages_per_seq < 0)
    return fail(DMLA_ERR_INVALID_ARG, "%s: negative size", what);
  if (!aligned16(kv_pool) || !aligned16(rows))
    return fail(DMLA_ERR_INVALID_ARG, "%s: the pool and the rows must be 16-byte aligned", what);
  if (kv_sp % 16 != 0 || kv_sp < kPage * kQ4RowBytes)
    return fail(DMLA_ERR_INVALID_ARG, "%s: page stride must be a multiple of 16 bytes and cover a page (got %lld)", what,
                (long long)kv_sp);
  if (!mult8(r_sb) || !mult8(r_ss) || r_ss < kD)
    return fail(DMLA_ERR_INVALID_ARG, "%s: row strides must be multiples of 8 and cover a row", what);
  if (bt_sb < max_pages_per_seq)
    return fail(DMLA_ERR_INVALID_ARG, "%s: block_table row stride < max_pages_per_seq", what);
  if (B > ((int64_t)1 << 24) || n > ((int64_t)1 << 24) || B * n >= ((int64_t)1 << 31) || num_pages > 0x7fffffff ||
      max_pages_per_seq > ((int64_t)1 << 24))
    return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  return DMLA_OK;
}

// A wave takes neighbouring rows, as many as leave every SIMD eight waves, up to kBatch; a CU gets up to 64 workgroups,
// eight times what fits (64 x 8192 rows appended in 193 us, 248 with the eight that fit; a gather of 32 x 5000 rows
// 31.7 and 35.7 us).
dim3 q4_rows_grid(int64_t rows, int& each) {
  const int64_t cus = device_cu_count();
  each = (int)std::min<int64_t>(kBatch, (rows + 32 * cus - 1) / (32 * cus));
  const int64_t per_wg = (int64_t)kWavesPerWG * each;
  return dim3((unsigned)std::min<int64_t>((rows + per_wg - 1) / per_wg, cus * 64));
}

}  // namespace
}  // namespace dmla

using namespace dmla;

extern "C" int dmla_kv_append_q4(void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                                 const int32_t* new_lens, const void* new_kv, int32_t* bad_index_flag, int64_t B,
                                 int64_t n_new, int64_t num_pages, int64_t max_pages_per_seq, int64_t kv_sp,
                                 int64_t bt_sb, int64_t nk_sb, int64_t nk_ss, dmla_stream_t stream) {
  clear_error();
  const int rc = q4_rows_validate("dmla_kv_append_q4", kv_pool, block_table, cache_seqlens, new_kv, B, n_new, num_pages,
                                  max_pages_per_seq, kv_sp, bt_sb, nk_sb, nk_ss);
  if (rc != DMLA_OK || B == 0 || n_new == 0) return rc;
  Q4RowArgs a = {};
  a.pool = static_cast<uint8_t*>(kv_pool);
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.lens = new_lens;
  a.rows = static_cast<bf16*>(const_cast<void*>(new_kv));
  a.bad = bad_index_flag;
  a.kv_sp = kv_sp; a.bt_sb = bt_sb; a.r_sb = nk_sb; a.r_ss = nk_ss;
  a.B = (int)B; a.n = (int)n_new;
  a.num_pages = (int)num_pages; a.max_pages = (int)max_pages_per_seq;
  a.ndiv = make_fastdiv((unsigned)n_new);
  const dim3 grid = q4_rows_grid(B * n_new, a.each);
  hipLaunchKernelGGL(q4_append_kernel, grid, dim3(64 * kWavesPerWG), 0, (hipStream_t)stream, a);
  return check_launch("dmla_kv_append_q4");
}

extern "C" int dmla_kv_gather_q4(const void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                                 const int32_t* starts, void* out, int64_t B, int64_t n_out, int64_t num_pages,
                                 int64_t max_pages_per_seq, int64_t kv_sp, int64_t bt_sb, int64_t o_sb, int64_t o_ss,
                                 dmla_stream_t stream) {
  clear_error();
  const int rc = q4_rows_validate("dmla_kv_gather_q4", kv_pool, block_table, cache_seqlens, out, B, n_out, num_pages,
                                  max_pages_per_seq, kv_sp, bt_sb, o_sb, o_ss);
  if (rc != DMLA_OK || B == 0 || n_out == 0) return rc;
  Q4RowArgs a = {};
  a.pool = static_cast<uint8_t*>(const_cast<void*>(kv_pool));
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.lens = starts;
  a.rows = static_cast<bf16*>(out);
  a.kv_sp = kv_sp; a.bt_sb = bt_sb; a.r_sb = o_sb; a.r_ss = o_ss;
  a.B = (int)B; a.n = (int)n_out;
  a.num_pages = (int)num_pages; a.max_pages = (int)max_pages_per_seq;
  a.ndiv = make_fastdiv((unsigned)n_out);
  const dim3 grid = q4_rows_grid(B * n_out, a.each);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kWavesPerWG), 0, (hipStream_t)stream, a);
  };
  if (B * n_out * kD * 2 >= kStreamBytes) launch(q4_gather_kernel<true>);
  else launch(q4_gather_kernel<false>);
  return check_launch("dmla_kv_gather_q4");
}
