// Eviction from the paged latent cache by accumulated attention weight.
//
// A sequence of N tokens above the budget K keeps its first S tokens (sinks), its newest R, and of the
// middle ones the K - S - R with the largest accounts (the lower index first among equals; NaN counts as
// the largest).  Attention does not depend on the order of the rows, since a row carries its position,
// so the pages are compacted with as few copies as possible:
//   * sinks, and kept middle rows below K - R, stay where they are;
//   * the other kept middle rows, in order, fill the freed places below K - R, in order;
//   * the newest R rows move down to [K - R, K), in order.
// Cutting 4096 + 64 tokens back to 4096 with R = 256 then moves at most 64 + 256 rows, where closing every
// gap would move nearly all.  No reference counterpart.
//
// Three launches: the selection (one workgroup per sequence), the middle moves together with a copy of
// the newest rows into the workspace where their old and new places overlap (N - K < R), and the newest
// rows' move.  A middle move's destination is a freed place and its source lies at or past K - R, so those moves
// depend on nothing; the newest rows overwrite such sources and therefore come last.
#include <algorithm>

#include "dmla_common.h"
#include "dmla_host.h"

namespace dmla {
namespace {

constexpr int kPage = 64;
constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kDigitBits = 11, kBins = 1 << kDigitBits;   // radix digits of 11, 11 and 10 bits
constexpr int kPerThread = 16;   // consecutive tokens of a thread in the ordered pass

struct EvictArgs {
  char* pool;
  const int32_t* block_table;
  const int32_t* seqlens;
  const float* mass;
  int32_t* new_lens;
  int32_t* src;
  float* mass_out;
  int32_t* bad;          // nullable
  int64_t kv_sp, kv_ss;  // bytes
  int64_t bt_sb, m_sb, mo_sb, src_sb;
  int B, mass_len, num_pages, max_pages, width;   // width: entries of a row of src
  int budget, recent, sink;
  int row_chunks;        // 16-byte pieces of a row
  int32_t* info;         // [B][2]: tokens cut from the sequence (0: untouched), middle rows to move
  int32_t* free_at;      // [B][budget - recent - sink] freed places, and the rows that fill them
  int32_t* late_at;
  char* stage;           // [B][recent] rows
};

// An integer that orders like the account: larger is better, -0 equals 0, NaN above everything.
__device__ __forceinline__ unsigned rank_key(float f) {
  unsigned u = __float_as_uint(f);
  if (f != f) return 0xffffffffu;
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix of v over the workgroup; total gets the sum.  tmp: kSelWaves ints.
__device__ __forceinline__ int scan_exclusive(int v, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();   // tmp is free
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  int before = 0, sum = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) {
    const int t = tmp[w];
    before += w < wave ? t : 0;
    sum += t;
  }
  total = sum;
  return before + x - v;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(EvictArgs a) {
  __shared__ int hist[kBins];
  __shared__ int tmp[kSelWaves];
  __shared__ int pick[2];   // the digit that holds the last kept key, and how many keys lie above it
  const int tid = threadIdx.x;
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int n = min(max(a.seqlens[b], 0), a.max_pages * kPage);
    const float* mass = a.mass + b * a.m_sb;
    float* mass_out = a.mass_out + b * a.mo_sb;
    int32_t* src = a.src + b * a.src_sb;
    int bad = 0;
    if (n > a.budget)
      for (int i = tid; i < (n + kPage - 1) / kPage; i += kSelThreads) {
        const int page = a.block_table[b * a.bt_sb + i];
        bad |= page < 0 || page >= a.num_pages;
      }
    bad = __syncthreads_or(bad);
    if (bad && a.bad != nullptr && tid == 0) a.bad[0] = 1;
    const bool cut = n > a.budget && !bad;
    const int new_len = cut ? a.budget : n;
    if (!cut) {
      if (tid == 0) {
        a.new_lens[b] = n;
        a.info[2 * b] = 0;
        a.info[2 * b + 1] = 0;
      }
      for (int i = tid; i < a.width; i += kSelThreads) src[i] = i < n ? i : -1;
      for (int i = tid; i < a.mass_len; i += kSelThreads) mass_out[i] = i < n ? mass[i] : 0.f;
      continue;
    }
    const int lo = a.sink, hi = n - a.recent;      // the middle tokens
    const int low_end = a.budget - a.recent;       // places of the kept ones: [lo, low_end)
    const int want = low_end - lo;
    // Radix select: the key of the last kept middle token, digit by digit, and how many tokens with
    // exactly that key are kept.
    unsigned prefix = 0, mask = 0;
    int left = want;   // how many are still to be taken from the tokens whose key matches prefix
    for (int d = 0; d < 3 && want > 0; ++d) {
      const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
      const int bins = d == 2 ? 1 << 10 : kBins;
      for (int i = tid; i < bins; i += kSelThreads) hist[i] = 0;
      __syncthreads();
      for (int i = lo + tid; i < hi; i += kSelThreads) {
        const unsigned key = rank_key(mass[i]);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1);
      }
      __syncthreads();
      // bins from the top: thread t holds the bins - 1 - 2t and the one below
      const int top = bins - 1 - 2 * tid;
      const int c0 = top >= 0 ? hist[top] : 0, c1 = top >= 1 ? hist[top - 1] : 0;
      int total;
      const int above = scan_exclusive(c0 + c1, tmp, total);
      if (above < left && left <= above + c0) {
        pick[0] = top;
        pick[1] = above;
      } else if (above + c0 < left && left <= above + c0 + c1) {
        pick[0] = top - 1;
        pick[1] = above + c0;
      }
      __syncthreads();
      prefix |= (unsigned)pick[0] << shift;
      mask |= (unsigned)(bins - 1) << shift;
      left -= pick[1];
      __syncthreads();
    }
    // In index order: which tokens stay, which places below low_end are freed, which rows fill them.
    int32_t* free_at = a.free_at + (int64_t)b * want;
    int32_t* late_at = a.late_at + (int64_t)b * want;
    int eq_seen = 0, n_free = 0, n_late = 0;
    for (int base = 0; base < hi && want > 0; base += kSelThreads * kPerThread) {
      const int i0 = base + tid * kPerThread;
      unsigned above = 0, equal = 0;   // one bit per token
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        const int i = i0 + j;
        if (i < lo || i >= hi) continue;
        const unsigned key = rank_key(mass[i]);
        above |= (key > prefix ? 1u : 0u) << j;
        equal |= (key == prefix ? 1u : 0u) << j;
      }
      int total;
      int rank = eq_seen + scan_exclusive(__popc(equal), tmp, total);
      eq_seen += total;
      unsigned kept = above;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j)
        if ((equal >> j) & 1) kept |= (rank++ < left ? 1u : 0u) << j;
      unsigned below = 0, middle = 0;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        below |= (i0 + j < low_end ? 1u : 0u) << j;
        middle |= (i0 + j >= lo && i0 + j < hi ? 1u : 0u) << j;
      }
      const unsigned freed = middle & below & ~kept, late = kept & ~below;
      // both ranks in one scan: a batch of 16384 tokens keeps either sum below 16 bits
      const int before = scan_exclusive(__popc(freed) | __popc(late) << 16, tmp, total);
      int fr = n_free + (before & 0xffff), lr = n_late + (before >> 16);
      n_free += total & 0xffff;
      n_late += total >> 16;
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        if ((freed >> j) & 1) free_at[fr++] = i0 + j;
        if ((late >> j) & 1) late_at[lr++] = i0 + j;
        if ((kept & below) >> j & 1) src[i0 + j] = i0 + j;
      }
    }
    if (tid == 0) {
      a.new_lens[b] = new_len;
      a.info[2 * b] = n - a.budget;
      a.info[2 * b + 1] = n_late;
    }
    __threadfence_block();
    __syncthreads();   // the lists are complete
    for (int i = tid; i < n_late; i += kSelThreads) src[free_at[i]] = late_at[i];
    for (int i = tid; i < a.sink; i += kSelThreads) src[i] = i;
    for (int i = tid; i < a.recent; i += kSelThreads) src[low_end + i] = hi + i;
    __threadfence_block();
    __syncthreads();   // src is complete
    for (int i = tid; i < a.mass_len; i += kSelThreads) mass_out[i] = i < new_len ? mass[src[i]] : 0.f;
  }
}

__device__ __forceinline__ char* row_at(const EvictArgs& a, int b, int pos) {
  return a.pool + a.block_table[b * a.bt_sb + pos / kPage] * a.kv_sp + (int64_t)(pos % kPage) * a.kv_ss;
}

// Phase 0: the middle moves, and the newest rows into the workspace where they overlap their new places.
// Phase 1: the newest rows to their places.  Grid: x over the 16-byte pieces of a sequence, y over sequences.
template <int kPhase>
__global__ void __launch_bounds__(256) evict_move_kernel(EvictArgs a) {
  const int want = a.budget - a.recent - a.sink;
  const int step = gridDim.x * 256;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int cut = a.info[2 * b], moves = a.info[2 * b + 1];
    if (cut == 0) continue;
    const int low_end = a.budget - a.recent;
    const bool staged = cut < a.recent;
    char* stage = a.stage + (int64_t)b * a.recent * a.row_chunks * 16;
    const int rows = kPhase == 0 ? moves + (staged ? a.recent : 0) : a.recent;
    for (int64_t p = blockIdx.x * 256 + threadIdx.x; p < (int64_t)rows * a.row_chunks; p += step) {
      const int r = (int)(p / a.row_chunks), c = (int)(p - (int64_t)r * a.row_chunks);
      const char* from;
      char* to;
      if constexpr (kPhase == 0) {
        if (r < moves) {
          from = row_at(a, b, a.late_at[(int64_t)b * want + r]);
          to = row_at(a, b, a.free_at[(int64_t)b * want + r]);
        } else {
          from = row_at(a, b, low_end + cut + (r - moves));
          to = stage + (int64_t)(r - moves) * a.row_chunks * 16;
        }
      } else {
        from = staged ? stage + (int64_t)r * a.row_chunks * 16 : row_at(a, b, low_end + cut + r);
        to = row_at(a, b, low_end + r);
      }
      *reinterpret_cast<i32x4*>(to + 16 * c) = *reinterpret_cast<const i32x4*>(from + 16 * c);
    }
  }
}

struct EvictLayout {
  int64_t info, lists, stage, total;   // byte offsets
};
// free_at and late_at hold the same number of entries; every part starts at a multiple of 16 bytes.
EvictLayout evict_layout(int64_t B, int64_t budget, int64_t recent, int64_t sink, int64_t row_bytes) {
  auto up = [](int64_t x) { return (x + 15) / 16 * 16; };
  const int64_t list = up(B * (budget - recent - sink) * 4);
  EvictLayout l;
  l.info = 0;
  l.lists = up(B * 8);
  l.stage = l.lists + 2 * list;
  l.total = l.stage + B * recent * row_bytes;
  return l;
}

}  // namespace
}  // namespace dmla

using namespace dmla;

static bool evict_sizes_ok(int64_t B, int64_t row_bytes, int64_t max_pages, int64_t budget, int64_t recent, int64_t sink) {
  return B > 0 && B <= ((int64_t)1 << 20) && row_bytes > 0 && row_bytes % 16 == 0 && row_bytes <= 65536 && max_pages > 0 &&
         max_pages <= ((int64_t)1 << 20) && budget > 0 && recent >= 0 && sink >= 0 && recent <= budget && sink <= budget - recent;
}

extern "C" int64_t dmla_kv_evict_workspace_bytes(int64_t B, int64_t row_bytes, int64_t max_pages_per_seq, int64_t budget,
                                                 int64_t recent, int64_t sink) {
  if (!evict_sizes_ok(B, row_bytes, max_pages_per_seq, budget, recent, sink)) return 0;
  if (budget >= max_pages_per_seq * kPage) return evict_layout(B, 0, 0, 0, row_bytes).total;   // nothing is ever cut
  return evict_layout(B, budget, recent, sink, row_bytes).total;
}

extern "C" int dmla_kv_evict(void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens, const float* mass,
                             int32_t* new_lens, int32_t* src, float* mass_out, int32_t* bad_index_flag, int64_t B,
                             int64_t row_bytes, int64_t num_pages, int64_t max_pages_per_seq, int64_t mass_len,
                             int64_t kv_sp, int64_t kv_ss, int64_t bt_sb, int64_t m_sb, int64_t mo_sb, int64_t src_sb,
                             int64_t budget, int64_t recent, int64_t sink, void* workspace, int64_t workspace_bytes,
                             dmla_stream_t stream) {
  clear_error();
  if (!kv_pool || !block_table || !cache_seqlens || !mass || !new_lens || !src || !mass_out)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: null pointer argument");
  if (B < 0 || num_pages < 0 || max_pages_per_seq < 0 || mass_len < 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: negative size");
  if (budget <= 0 || recent < 0 || sink < 0 || recent > budget || sink > budget - recent)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: budget must be positive and cover recent + sink");
  if (row_bytes <= 0 || row_bytes % 16 != 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: row_bytes must be a positive multiple of 16");
  if (!aligned16(kv_pool)) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: kv_pool must be 16-byte aligned");
  if (kv_sp % 16 != 0 || kv_ss % 16 != 0 || kv_ss < row_bytes || kv_ss > ((int64_t)1 << 31) || kv_sp < kPage * kv_ss)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: strides must be multiples of 16 bytes and cover a row / page");
  if (bt_sb < max_pages_per_seq)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: block_table row stride < max_pages_per_seq");
  if (B == 0) return DMLA_OK;
  if (num_pages == 0 || max_pages_per_seq == 0)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: empty page pool or block table");
  if (max_pages_per_seq > ((int64_t)1 << 20) || B > ((int64_t)1 << 20) || num_pages > 0x7fffffff || row_bytes > 65536)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_kv_evict: size too large");
  const int64_t cap = max_pages_per_seq * kPage;
  if (mass_len < cap || m_sb < mass_len || mo_sb < mass_len || mass_len > ((int64_t)1 << 30))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: mass rows must cover the block table's tokens");
  const int64_t width = std::min(budget, cap);
  if (src_sb < width) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: src rows must hold min(budget, tokens) entries");
  if (mass == mass_out) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: mass_out must not be mass");
  const int64_t need = dmla_kv_evict_workspace_bytes(B, row_bytes, max_pages_per_seq, budget, recent, sink);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(DMLA_ERR_WORKSPACE, "dmla_kv_evict: workspace of %lld bytes needed (got %lld)", (long long)need,
                (long long)workspace_bytes);
  if (!aligned16(workspace)) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_evict: workspace must be 16-byte aligned");
  const bool can_cut = budget < cap;
  const EvictLayout l = can_cut ? evict_layout(B, budget, recent, sink, row_bytes) : evict_layout(B, 0, 0, 0, row_bytes);
  char* ws = static_cast<char*>(workspace);
  EvictArgs a = {};
  a.pool = static_cast<char*>(kv_pool);
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.mass = mass;
  a.new_lens = new_lens; a.src = src; a.mass_out = mass_out; a.bad = bad_index_flag;
  a.kv_sp = kv_sp; a.kv_ss = kv_ss; a.bt_sb = bt_sb; a.m_sb = m_sb; a.mo_sb = mo_sb; a.src_sb = src_sb;
  a.B = (int)B; a.mass_len = (int)mass_len; a.num_pages = (int)num_pages; a.max_pages = (int)max_pages_per_seq;
  a.width = (int)width;
  a.budget = (int)std::min<int64_t>(budget, 0x7fffffff); a.recent = can_cut ? (int)recent : 0; a.sink = can_cut ? (int)sink : 0;
  a.row_chunks = (int)(row_bytes / 16);
  a.info = reinterpret_cast<int32_t*>(ws + l.info);
  a.free_at = reinterpret_cast<int32_t*>(ws + l.lists);
  a.late_at = reinterpret_cast<int32_t*>(ws + l.lists + (l.stage - l.lists) / 2);
  a.stage = ws + l.stage;
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)std::min<int64_t>(B, 65535)), dim3(kSelThreads), 0,
                     (hipStream_t)stream, a);
  int rc = check_launch("dmla_kv_evict");
  if (rc != DMLA_OK || !can_cut) return rc;
  // About eight workgroups per CU over all sequences, no more than a sequence has pieces to move.
  const int64_t gy = std::min<int64_t>(B, 65535);
  const int64_t share = std::max<int64_t>(1, (int64_t)device_cu_count() * 8 / gy);
  auto launch = [&](auto kernel, int64_t rows) {
    if (rows == 0) return;
    const int64_t gx = std::min(share, (rows * a.row_chunks + 255) / 256);
    hipLaunchKernelGGL(kernel, dim3((unsigned)gx, (unsigned)gy), dim3(256), 0, (hipStream_t)stream, a);
  };
  launch(evict_move_kernel<0>, std::min(budget - recent - sink, cap - budget) + recent);
  launch(evict_move_kernel<1>, recent);
  return check_launch("dmla_kv_evict(move)");
}
