// Pages by request lengths: the bookkeeping of a scheduler's step on the device, next to the paged cache.
// No reference counterpart: the reference has no paged cache.
//
// Free pages are a stack: free_pages[0 .. count) are free, the top is taken first.
//   release: the pages between a sequence's old and its new length go on top, sequence after sequence.
//   reserve: with need_b = ceil((len_b + new_b) / 64) - ceil(len_b / 64) and P_b = need_0 + .. + need_b, the i-th
//     page of sequence b's need is entry count - 1 - (P_b - need_b + i); row t of b (packed row cu_b + t) has
//     slot page * 64 + (len_b + t) % 64.
//   append by slot: a row goes where its slot says.
//
// Bound: release and reserve read and write some words per sequence, page and row, so they take a launch and the
// latency of what each workgroup reads before it knows its rows: lengths, one prefix sum, free pages.  Every
// workgroup of reserve works out the same prefix sums (256 sequences at a time) instead of waiting for a kernel that
// does; new entries of the table and the count left are written by one thread each and read by none.
#include <algorithm>

#include "dmla_host.h"
#include "dmla_common.h"

namespace dmla {
namespace {

constexpr int kPage = 64;
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kCap = 1 << 30;   // prefix sums stop here: sizes are below it, and a sum past it fits nowhere

// Inclusive sum over the workgroup's threads, at most kCap (0 <= v <= kCap); sum: over all.  Saturation is
// associative, so the order of the steps does not matter.
template <int kW>
__device__ __forceinline__ int capped_scan(int v, int* tmp, int& sum) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  auto add = [](int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)kCap); };
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x = add(x, y);
  }
  __syncthreads();   // tmp is free
  if (lane == 63) tmp[wave] = x;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    if (w < wave) x = add(x, tmp[w]);
    sum = add(sum, tmp[w]);
  }
  return x;
}

// The first i of n ascending values with v[i] > x (n where there is none).
__device__ __forceinline__ int first_above(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (v[mid] > x) hi = mid; else lo = mid + 1;
  }
  return lo;
}

struct ReserveArgs {
  int32_t* block_table;
  const int32_t* seqlens;
  const int32_t* new_lens;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* total_lens;
  int32_t* cu;
  int32_t* slots;
  int32_t* new_count;
  int32_t* bad;   // nullable
  int64_t bt_sb;
  int B, rows, max_pages, num_pages, capacity, each;   // each: rows of a workgroup
};

__global__ void __launch_bounds__(kThreads) kv_reserve_kernel(ReserveArgs a) {
  __shared__ int tmp[kWaves];
  __shared__ int s_end[kThreads], s_new[kThreads], s_len[kThreads], s_first[kThreads];   // s_first: -1: not served
  const int tid = threadIdx.x;
  const int r0 = min((int64_t)blockIdx.x * a.each, (int64_t)a.rows), r1 = min((int64_t)r0 + a.each, (int64_t)a.rows);
  const int avail = min(max(a.free_count[0], 0), a.capacity);
  const int64_t room = (int64_t)a.max_pages * kPage;
  int rows_before = 0, pages_before = 0, taken = 0;
  bool refused = false;
  for (int c0 = 0; c0 < a.B; c0 += kThreads) {
    const int b = c0 + tid, count = min(kThreads, a.B - c0);
    const bool in = b < a.B;
    const int len = in ? max(a.seqlens[b], 0) : 0;
    const int n = in ? min(max(a.new_lens[b], 0), kCap) : 0;
    int chunk_rows, chunk_pages;
    const int end = (int)min((unsigned)rows_before + (unsigned)capped_scan<kWaves>(n, tmp, chunk_rows), (unsigned)kCap);
    const int have = (int)(((int64_t)len + kPage - 1) / kPage);
    const bool fits = end <= a.rows && (int64_t)len + n <= room;
    const int need = fits && n > 0 ? (int)(((int64_t)len + n + kPage - 1) / kPage) - have : 0;
    const int upto = (int)min((unsigned)pages_before + (unsigned)capped_scan<kWaves>(need, tmp, chunk_pages), (unsigned)kCap);
    const bool served = n == 0 || (fits && (need == 0 || upto <= avail));
    if (in && !served) refused = true;
    s_end[tid] = end;
    s_new[tid] = n;
    s_len[tid] = len;
    s_first[tid] = served ? upto - need : -1;
    if (blockIdx.x == 0) {
      if (in) {
        a.total_lens[b] = served ? (int)min((int64_t)len + n, (int64_t)0x7fffffff) : len;
        a.cu[b + 1] = min(end, a.rows);
      }
      // The served ones that need pages come first, so the largest of their sums is what was taken.
      int m = served && need > 0 ? upto : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) m = max(m, __shfl_xor(m, o, 64));
      taken = max(taken, m);
    }
    __syncthreads();
    const int lo = max(r0, min(rows_before, a.rows)), hi = min(r1, (int)min((unsigned)rows_before + (unsigned)chunk_rows, (unsigned)kCap));
    for (int r = lo + tid; r < hi; r += kThreads) {
      const int i = first_above(s_end, count, r);
      int slot = -1;
      if (s_first[i] >= 0) {
        const int t = r - (s_end[i] - s_new[i]);
        const int pos = s_len[i] + t;   // within the table: s_len + s_new is at most max_pages * 64
        const int old = (s_len[i] + kPage - 1) / kPage, p = pos / kPage;
        int32_t* entry = a.block_table + (c0 + i) * a.bt_sb + p;
        int page;
        if (p >= old) {
          page = a.free_pages[avail - 1 - (s_first[i] + p - old)];
          if (pos % kPage == 0) *entry = page;   // the page's first row is new, too
        } else {
          page = *entry;
        }
        if (page >= 0 && page < a.num_pages) slot = page * kPage + pos % kPage;
        else refused = true;
      }
      a.slots[r] = slot;
    }
    rows_before = (int)min((unsigned)rows_before + (unsigned)chunk_rows, (unsigned)kCap);
    pages_before = (int)min((unsigned)pages_before + (unsigned)chunk_pages, (unsigned)kCap);
    __syncthreads();   // the sequences' values are read
  }
  for (int r = max(r0, min(rows_before, a.rows)) + tid; r < r1; r += kThreads) a.slots[r] = -1;   // past the last sequence
  if (blockIdx.x == 0) {
    if ((tid & 63) == 0) tmp[tid >> 6] = taken;
    __syncthreads();
    if (tid == 0) {
      int m = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) m = max(m, tmp[w]);
      a.new_count[0] = avail - m;
      a.cu[0] = 0;
    }
  }
  if (refused && a.bad != nullptr) a.bad[0] = 1;
}

struct ReleaseArgs {
  const int32_t* block_table;
  const int32_t* old_lens;
  const int32_t* new_lens;
  int32_t* free_pages;
  const int32_t* free_count;
  int32_t* new_count;
  int32_t* bad;   // nullable
  int64_t bt_sb;
  int B, max_pages, num_pages, capacity;
};

// One workgroup: the pages of a step are few.  The entries that go, in order, kReleaseThreads at a time: a
// thread finds its entry's sequence in the prefix sums, and valid entries close up by ranks from ballots.
constexpr int kReleaseThreads = 1024, kReleaseWaves = kReleaseThreads / 64;
__global__ void __launch_bounds__(kReleaseThreads) kv_release_kernel(ReleaseArgs a) {
  __shared__ int tmp[kReleaseWaves];
  __shared__ int s_end[kReleaseThreads], s_keep[kReleaseThreads], s_count[kReleaseThreads];
  __shared__ int s_valid[2][kReleaseWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  int count = min(max(a.free_count[0], 0), a.capacity);
  bool refused = false;
  for (int c0 = 0; c0 < a.B; c0 += kReleaseThreads) {
    const int b = c0 + tid;
    const bool in = b < a.B;
    const int held = in ? (int)min(((int64_t)max(a.old_lens[b], 0) + kPage - 1) / kPage, (int64_t)a.max_pages) : 0;
    const int keep = in ? (int)min(((int64_t)max(a.new_lens[b], 0) + kPage - 1) / kPage, (int64_t)held) : 0;
    int entries;
    const int end = capped_scan<kReleaseWaves>(held - keep, tmp, entries);
    s_end[tid] = end;
    s_keep[tid] = keep;
    s_count[tid] = held - keep;
    __syncthreads();
    int turn = 0;
    for (int e0 = 0; e0 < entries; e0 += kReleaseThreads, turn ^= 1) {
      const int e = e0 + tid;
      int page = -1;
      if (e < entries) {
        const int i = first_above(s_end, kReleaseThreads, e);
        page = a.block_table[(c0 + i) * a.bt_sb + s_keep[i] + e - (s_end[i] - s_count[i])];
      }
      const bool valid = page >= 0 && page < a.num_pages;
      refused = refused || (e < entries && !valid);
      const uint64_t mask = __ballot(valid);
      if (lane == 0) s_valid[turn][wave] = __popcll(mask);
      __syncthreads();   // (the other turn's counts are read before the next of this turn's are written)
      int before = 0, all = 0;
#pragma unroll
      for (int w = 0; w < kReleaseWaves; ++w) {
        before += w < wave ? s_valid[turn][w] : 0;
        all += s_valid[turn][w];
      }
      const int64_t at = (int64_t)count + before + __popcll(mask & ((1ull << lane) - 1));
      if (valid) {
        if (at < a.capacity) a.free_pages[at] = page;
        else refused = true;
      }
      count = (int)min((int64_t)count + all, (int64_t)a.capacity);
    }
    __syncthreads();   // the sequences' values are read
  }
  if (tid == 0) a.new_count[0] = count;
  if (refused && a.bad != nullptr) a.bad[0] = 1;
}

struct AppendRowsArgs {
  bf16* pool;
  const int32_t* slots;
  const bf16* rows;
  int32_t* bad;   // nullable
  int64_t kv_sp, kv_ss, r_ss;
  int T, chunks, num_pages;   // chunks: 16-byte pieces of a row
  FastDiv cdiv;               // division by chunks
};

// A 16-byte piece per thread and step, consecutive threads on consecutive pieces of a row.
__global__ void __launch_bounds__(256) kv_append_rows_kernel(AppendRowsArgs a) {
  const int64_t total = (int64_t)a.T * a.chunks;
  for (int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; u < total; u += (int64_t)gridDim.x * blockDim.x) {
    const int r = fast_div((int)u, a.cdiv), c = (int)u - r * a.chunks;
    const int slot = a.slots[r];
    if (slot < 0) continue;
    if (slot / kPage >= a.num_pages) {
      if (a.bad != nullptr) a.bad[0] = 1;
      continue;
    }
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(a.rows + r * a.r_ss + 8 * c);
    *reinterpret_cast<bf16x8*>(a.pool + slot / kPage * a.kv_sp + slot % kPage * a.kv_ss + 8 * c) = v;
  }
}

}  // namespace
}  // namespace dmla

using namespace dmla;

namespace {

// Sizes that both calls take.
int pages_validate(const char* what, int64_t B, int64_t num_pages, int64_t max_pages, int64_t capacity, int64_t bt_sb) {
  if (B < 0 || num_pages < 0 || max_pages < 0 || capacity < 0) return fail(DMLA_ERR_INVALID_ARG, "%s: negative size", what);
  if (bt_sb < max_pages) return fail(DMLA_ERR_INVALID_ARG, "%s: block_table row stride < max_pages_per_seq", what);
  if (B > ((int64_t)1 << 24) || num_pages > ((int64_t)1 << 25) || max_pages > ((int64_t)1 << 24) || capacity >= kCap)
    return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  return DMLA_OK;
}

}  // namespace

extern "C" int dmla_kv_reserve(int32_t* block_table, const int32_t* cache_seqlens, const int32_t* new_lens,
                               const int32_t* free_pages, const int32_t* free_count, int32_t* total_lens,
                               int32_t* cu_seqlens, int32_t* slots, int32_t* new_count, int32_t* bad_index_flag, int64_t B,
                               int64_t num_rows, int64_t num_pages, int64_t max_pages_per_seq, int64_t capacity,
                               int64_t bt_sb, dmla_stream_t stream) {
  clear_error();
  const int rc = pages_validate("dmla_kv_reserve", B, num_pages, max_pages_per_seq, capacity, bt_sb);
  if (rc != DMLA_OK) return rc;
  if (num_rows < 0) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_reserve: negative size");
  if (num_rows >= kCap) return fail(DMLA_ERR_UNSUPPORTED, "dmla_kv_reserve: size too large");
  // (Where a size is 0 its arrays are empty and any address does.)
  if (!free_count || !cu_seqlens || !new_count || (B > 0 && (!cache_seqlens || !new_lens || !total_lens)) ||
      (B > 0 && max_pages_per_seq > 0 && !block_table) || (capacity > 0 && !free_pages) || (num_rows > 0 && !slots))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_reserve: null pointer argument");
  ReserveArgs a = {};
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.new_lens = new_lens;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.total_lens = total_lens;
  a.cu = cu_seqlens;
  a.slots = slots;
  a.new_count = new_count;
  a.bad = bad_index_flag;
  a.bt_sb = bt_sb;
  a.B = (int)B; a.rows = (int)num_rows; a.max_pages = (int)max_pages_per_seq; a.num_pages = (int)num_pages;
  a.capacity = (int)capacity;
  const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>((num_rows + kThreads - 1) / kThreads, 2 * device_cu_count()));
  a.each = (int)((num_rows + wgs - 1) / wgs);
  hipLaunchKernelGGL(kv_reserve_kernel, dim3((unsigned)wgs), dim3(kThreads), 0, (hipStream_t)stream, a);
  return check_launch("dmla_kv_reserve");
}

extern "C" int dmla_kv_release(const int32_t* block_table, const int32_t* old_lens, const int32_t* new_lens,
                               int32_t* free_pages, const int32_t* free_count, int32_t* new_count,
                               int32_t* bad_index_flag, int64_t B, int64_t num_pages, int64_t max_pages_per_seq,
                               int64_t capacity, int64_t bt_sb, dmla_stream_t stream) {
  clear_error();
  const int rc = pages_validate("dmla_kv_release", B, num_pages, max_pages_per_seq, capacity, bt_sb);
  if (rc != DMLA_OK) return rc;
  if (!free_count || !new_count || (B > 0 && (!old_lens || !new_lens)) || (B > 0 && max_pages_per_seq > 0 && !block_table) ||
      (capacity > 0 && !free_pages))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_release: null pointer argument");
  ReleaseArgs a = {};
  a.block_table = block_table;
  a.old_lens = old_lens;
  a.new_lens = new_lens;
  a.free_pages = free_pages;
  a.free_count = free_count;
  a.new_count = new_count;
  a.bad = bad_index_flag;
  a.bt_sb = bt_sb;
  a.B = (int)B; a.max_pages = (int)max_pages_per_seq; a.num_pages = (int)num_pages; a.capacity = (int)capacity;
  // A thousand sequences' entries are counted in 32 bits.
  if (std::min<int64_t>(B, kReleaseThreads) * max_pages_per_seq >= kCap)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_kv_release: size too large");
  hipLaunchKernelGGL(kv_release_kernel, dim3(1), dim3(kReleaseThreads), 0, (hipStream_t)stream, a);
  return check_launch("dmla_kv_release");
}

extern "C" int dmla_kv_append_rows(void* kv_pool, const int32_t* slots, const void* rows, int32_t* bad_index_flag,
                                   int64_t T, int64_t d, int64_t num_pages, int64_t kv_sp, int64_t kv_ss, int64_t r_ss,
                                   dmla_stream_t stream) {
  clear_error();
  if (T < 0 || d <= 0 || num_pages < 0) return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_append_rows: negative or zero size");
  // (Of an empty call any address does: empty tensors have none.)
  if (T > 0 && (!slots || !rows || (num_pages > 0 && !kv_pool)))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_append_rows: null pointer argument");
  if (d % 8 != 0) return fail(DMLA_ERR_UNSUPPORTED, "dmla_kv_append_rows: d must be a multiple of 8 (got %lld)", (long long)d);
  if (!aligned16(kv_pool) || !aligned16(rows))
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_append_rows: kv_pool and rows must be 16-byte aligned");
  if (!mult8(kv_sp) || !mult8(kv_ss) || !mult8(r_ss) || kv_ss < d || kv_sp < kPage * kv_ss || r_ss < d)
    return fail(DMLA_ERR_INVALID_ARG, "dmla_kv_append_rows: strides must be multiples of 8 and cover a row / page");
  if (num_pages > ((int64_t)1 << 25) || d / 8 > 0x7fffffff || T > 0x7fffffff || T * (d / 8) > 0x7fffffff)
    return fail(DMLA_ERR_UNSUPPORTED, "dmla_kv_append_rows: size too large");
  if (T == 0) return DMLA_OK;
  AppendRowsArgs a = {};
  a.pool = static_cast<bf16*>(kv_pool);
  a.slots = slots;
  a.rows = static_cast<const bf16*>(rows);
  a.bad = bad_index_flag;
  a.kv_sp = kv_sp; a.kv_ss = kv_ss; a.r_ss = r_ss;
  a.T = (int)T; a.chunks = (int)(d / 8); a.num_pages = (int)num_pages;
  a.cdiv = make_fastdiv((unsigned)(d / 8));
  const int64_t blocks = std::min<int64_t>((T * (d / 8) + 255) / 256, (int64_t)device_cu_count() * 16);
  hipLaunchKernelGGL(kv_append_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("dmla_kv_append_rows");
}
