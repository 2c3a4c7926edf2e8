// Which pages of a long context a query attends: the mean row of every full page, a score of each page for each
// query from its attention over the means, and the selection of the pages with the largest scores.  The selected
// pages form a block table of their own, which chunk attention or a decode reads.  No reference counterpart.
//
//   mean[page] = (1 / 64) sum of the page's 64 rows, in bf16
//   score[t, p] = sum_h exp(s_hp) / sum_p' exp(s_hp'), s_hp = scale q[t, h] . mean[page p of t's sequence],
//     over the pages p that lie before the page of t itself
//   selected: the first `sink` pages, the newest `recent` (t's own page is the newest) and of those between the
//     ones with the largest scores, the lower page first among equals, NaN above everything.
#include <algorithm>

#include "dmla_host.h"
#include "dmla_q4.h"

namespace dmla {
namespace {

constexpr int kD = 576, kLat = 512, kPage = 64;

// ---- means ------------------------------------------------------------------------------------------
struct MeansArgs {
  const char* pool;
  const int32_t* block_table;
  const int32_t* seqlens;
  const int32_t* starts;   // nullable: 0
  bf16* means;
  int64_t kv_sp, kv_ss, bt_sb, m_sp;   // kv strides in bytes
  int B, num_pages, max_pages;
};

// A page per workgroup at a time: thread (g, c) adds rows 8 g .. 8 g + 7 of the 8 columns of piece c, the eight
// groups meet in LDS, in order.
// Bound: HBM, the pages' rows; a decode step has at most one new full page per sequence and is a launch.
constexpr int kMeanGroups = 8, kMeanThreads = kMeanGroups * (kD / 8);   // 576, nine waves
template <bool kQ4>
__global__ void __launch_bounds__(kMeanThreads) page_means_kernel(MeansArgs a) {
  __shared__ __attribute__((aligned(16))) float part[kMeanGroups][kD];
  const int g = threadIdx.x / (kD / 8), c = threadIdx.x % (kD / 8);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int64_t len = min((int64_t)a.seqlens[b], (int64_t)a.max_pages * kPage);
    const int first = a.starts != nullptr ? max(a.starts[b], 0) / kPage : 0;
    for (int64_t p = first + blockIdx.y; p < len / kPage; p += gridDim.y) {
      const int page = a.block_table[b * a.bt_sb + p];
      if (page < 0 || page >= a.num_pages) continue;   // (uniform)
      float x[8] = {};
#pragma unroll
      for (int r = 0; r < kPage / kMeanGroups; ++r) {
        const char* row = a.pool + page * a.kv_sp + (g * (kPage / kMeanGroups) + r) * a.kv_ss;
        bf16x8 v;
        if constexpr (!kQ4) v = *reinterpret_cast<const bf16x8*>(row + 16 * c);
        else if (c >= kLat / 8) v = *reinterpret_cast<const bf16x8*>(row + kQ4RopeOff + 16 * (c - kLat / 8));
        else v = q4_octet(*reinterpret_cast<const unsigned*>(row + 4 * c), q4_scale((uint8_t)row[kQ4ScaleOff + c / 4]));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += (float)v[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) part[g][8 * c + i] = x[i];
      __syncthreads();
      if (g == 0) {
        bf16x8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float s = x[i];
#pragma unroll
          for (int o = 1; o < kMeanGroups; ++o) s += part[o][8 * c + i];
          v[i] = (bf16)(s * (1.0f / kPage));
        }
        *reinterpret_cast<bf16x8*>(a.means + page * a.m_sp + 8 * c) = v;
      }
      __syncthreads();
    }
  }
}

// ---- the queries of a call ----------------------------------------------------------------------------
// Packed: sequence b has the queries cu[b] .. cu[b + 1] - 1, the newest of its tokens; cu = NULL: one query each.
struct Queries {
  const int32_t* cu;
  const int32_t* seqlens;
  int B, T, max_pages;
};

// Sequence of query t (>= B: none), by a wave.
__device__ __forceinline__ int sequence_of(const Queries& q, int t) {
  if (q.cu == nullptr) return t;
  const int lane = lane_id();
  int n = 0;
  for (int i0 = 0; i0 < q.B; i0 += 64) n += __popcll(__ballot(i0 + lane < q.B && q.cu[i0 + lane + 1] <= t));
  return n;
}
// Tokens that query t of sequence b sees (itself the last), 0 where it belongs to none.
__device__ __forceinline__ int visible(const Queries& q, int b, int t) {
  if (b >= q.B) return 0;
  const int64_t len = min((int64_t)max(q.seqlens[b], 0), (int64_t)q.max_pages * kPage);
  if (q.cu == nullptr) return (int)len;
  const int lo = q.cu[b], hi = min(q.cu[b + 1], q.T);
  if (t < lo || t >= hi) return 0;
  return (int)max((int64_t)0, len - (hi - 1 - t));
}

// ---- scores -------------------------------------------------------------------------------------------
struct ScoreArgs {
  const bf16* q;
  const bf16* means;
  const int32_t* block_table;
  Queries qs;
  float* scores;
  float2* stats;   // [chunks, T, H]: max (log2 units) and sum
  int64_t q_st, q_sh, m_sp, bt_sb, s_st;
  int H, num_pages;
  int blocks, passes;   // 16-row blocks of a query (at most kBlocks of a pass), passes over the heads
  int group;            // queries of a workgroup
  int chunk, chunks;    // pages of a workgroup, a multiple of 64
  float scale_log2;
};

constexpr int kBlocks = 8;                      // 16-row blocks in LDS: 128 rows (query, head), heads padded to 16
constexpr int kRowBytes = 2 * kD + 16;          // 16 rows at one place of a row lie in different banks
constexpr int kScoreThreads = 256, kScoreWaves = 4;
enum { kFused, kStats, kSum };

// kFused: one workgroup has all pages of its queries, their sums first and then the scores.  Else the pages are
// cut in chunks over workgroups, kStats leaves each chunk's maxima and sums and kSum reads all of them.
// A wave multiplies 16 pages (in registers) with the rows in LDS, 16x16x32 MFMAs; a lane then holds four heads of
// a page.  Scores of a page are summed in a fixed order, by one lane.
template <int kMode>
__global__ void __launch_bounds__(kScoreThreads) page_scores_kernel(ScoreArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_seq[kBlocks], s_pages[kBlocks];
  __shared__ float s_lse[16 * kBlocks];
  __shared__ float2 s_part[kScoreWaves][16 * kBlocks];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int t0 = blockIdx.x * a.group, nt = min(a.group, a.qs.T - t0);
  const int c0 = blockIdx.y * a.chunk, c1 = min(c0 + a.chunk, a.qs.max_pages);
  for (int i = wave; i < nt; i += kScoreWaves) {
    const int b = sequence_of(a.qs, t0 + i);
    const int n = visible(a.qs, b, t0 + i);
    if (lane == 0) {
      s_seq[i] = b;
      s_pages[i] = n > 0 ? (n - 1) / kPage : 0;   // pages before its own
    }
  }
  __syncthreads();
  const int nb = a.passes > 1 ? kBlocks : a.blocks * nt;   // blocks in use
  for (int pass = 0; pass < a.passes; ++pass) {
    const int head0 = pass * 16 * kBlocks;
    if (pass > 0) __syncthreads();   // the rows of the pass before are read
    for (int k = tid; k < nb * 16 * (kD / 8); k += kScoreThreads) {
      const int r = k / (kD / 8), c = k - r * (kD / 8);
      const int i = a.passes > 1 ? 0 : r / (16 * a.blocks);
      const int head = min(head0 + r - i * 16 * a.blocks, a.H - 1);
      *reinterpret_cast<bf16x8*>(smem + r * kRowBytes + 16 * c) =
          *reinterpret_cast<const bf16x8*>(a.q + (t0 + i) * a.q_st + head * a.q_sh + 8 * c);
    }
    if constexpr (kMode == kSum) {
      for (int r = tid; r < nb * 16; r += kScoreThreads) {
        const int i = a.passes > 1 ? 0 : r / (16 * a.blocks);
        const int head = min(head0 + r - i * 16 * a.blocks, a.H - 1);
        float m = kNegInf, l = 0.f;
        for (int c = 0; c < a.chunks; ++c) {
          const float2 s = a.stats[((int64_t)c * a.qs.T + t0 + i) * a.H + head];
          const float mm = fmaxf(m, s.x);
          if (mm != kNegInf) l = l * fast_exp2(m - mm) + s.y * fast_exp2(s.x - mm);
          else l += s.y;   // 0, or not a number
          m = mm;
        }
        s_lse[r] = m == kNegInf ? l : m + __log2f(l);
      }
    }
    __syncthreads();
    for (int i0 = 0; i0 < nt;) {   // the queries of one sequence at a time
      const int b = s_seq[i0];
      int i1 = i0 + 1, most = s_pages[i0];
      for (; i1 < nt && s_seq[i1] == b; ++i1) most = max(most, s_pages[i1]);
      // f(rb, page of this lane, scores of heads 16 (rb % blocks) + 4 g + 0 .. 3, their query): for every row block
      // of the sequence; -inf where there is nothing.
      auto tile = [&](int p0, auto f) {
        const int p = p0 + l16;
        const int page = p < min(most, c1) ? a.block_table[b * a.bt_sb + p] : -1;
        const bool there = page >= 0 && page < a.num_pages;
        const bf16* row = a.means + (there ? page : 0) * a.m_sp + 8 * g;
        bf16x8 k[kD / 32];
#pragma unroll
        for (int c = 0; c < kD / 32; ++c) k[c] = *reinterpret_cast<const bf16x8*>(row + 32 * c);
#pragma unroll
        for (int rb = 0; rb < kBlocks; ++rb) {
          const int i = a.passes > 1 ? 0 : rb / a.blocks;
          if (rb >= nb || i < i0 || i >= i1) continue;
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < kD / 32; ++c)
            x = mfma_bf16(*reinterpret_cast<const bf16x8*>(smem + (16 * rb + l16) * kRowBytes + 64 * c + 16 * g), k[c], x);
          const int head = head0 + 16 * (rb - i * a.blocks) + 4 * g;
          const bool seen = there && p < s_pages[i];
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = seen && head + e < a.H ? x[e] * a.scale_log2 : kNegInf;
          f(rb, p, x, i);
        }
      };
      if constexpr (kMode != kSum) {
        float m[kBlocks][4], l[kBlocks][4];
#pragma unroll
        for (int rb = 0; rb < kBlocks; ++rb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            m[rb][e] = kNegInf;
            l[rb][e] = 0.f;
          }
        auto merge = [](float& m0, float& l0, float m1, float l1) {
          const float mm = fmaxf(m0, m1);
          if (mm != kNegInf) l0 = l0 * fast_exp2(m0 - mm) + l1 * fast_exp2(m1 - mm);
          else l0 += l1;   // 0, or not a number
          m0 = mm;
        };
        for (int p0 = c0 + 16 * wave; p0 < min(most, c1); p0 += 16 * kScoreWaves)
          tile(p0, [&](auto rb, int, const f32x4& x, int) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool number = x[e] == x[e];
              merge(m[rb][e], l[rb][e], number ? x[e] : kNegInf, number ? (x[e] == kNegInf ? 0.f : 1.f) : x[e]);
            }
          });
#pragma unroll
        for (int rb = 0; rb < kBlocks; ++rb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) {
              const float m1 = __shfl_xor(m[rb][e], o, 64), l1 = __shfl_xor(l[rb][e], o, 64);
              merge(m[rb][e], l[rb][e], m1, l1);
            }
            if (l16 == 0) s_part[wave][16 * rb + 4 * g + e] = make_float2(m[rb][e], l[rb][e]);
          }
        __syncthreads();
        for (int r = tid; r < nb * 16; r += kScoreThreads) {
          const int i = a.passes > 1 ? 0 : r / (16 * a.blocks);
          if (i < i0 || i >= i1) continue;
          float mm = kNegInf, ll = 0.f;
#pragma unroll
          for (int w = 0; w < kScoreWaves; ++w) merge(mm, ll, s_part[w][r].x, s_part[w][r].y);
          if constexpr (kMode == kStats) {
            const int head = head0 + r - i * 16 * a.blocks;
            if (head < a.H) a.stats[((int64_t)blockIdx.y * a.qs.T + t0 + i) * a.H + head] = make_float2(mm, ll);
          } else {
            s_lse[r] = mm == kNegInf ? ll : mm + __log2f(ll);
          }
        }
        __syncthreads();
      }
      if constexpr (kMode != kStats) {
        for (int p0 = c0 + 16 * wave; p0 < c1; p0 += 16 * kScoreWaves) {
          auto put = [&](int i, int p, float v) {
            if (g != 0 || p >= c1) return;
            float* to = a.scores + (t0 + i) * a.s_st + p;
            *to = pass > 0 ? *to + v : v;
          };
          if (p0 >= most) {
            for (int i = i0; i < i1; ++i) put(i, p0 + l16, 0.f);
            continue;
          }
          float sum = 0.f;
          tile(p0, [&](auto rb, int p, const f32x4& x, int i) {
            float v = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (x[e] != kNegInf) v += fast_exp2(x[e] - s_lse[16 * rb + 4 * g + e]);   // (not a number stays)
            sum += group_sum(v);
            if (a.passes > 1 ? rb == kBlocks - 1 : (rb + 1) % a.blocks == 0) {
              put(i, p, sum);
              sum = 0.f;
            }
          });
        }
      }
      i0 = i1;
    }
  }
}

// ---- selection ----------------------------------------------------------------------------------------
struct SelectArgs {
  const float* scores;
  const int32_t* block_table;
  Queries qs;
  int32_t* sel_table;
  int32_t* sel_lens;
  int32_t* sel_index;
  int64_t s_st, bt_sb, st_st, si_st;
  int k, recent, sink;
};

// A score as an integer of the same order, above 0: -0 like 0, NaN above everything.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned u = __float_as_uint(x == 0.f ? 0.f : x);
  return x != x ? 0xffffffffu : u >> 31 ? ~u : u | 0x80000000u;
}

// A query per wave: its candidates' scores in registers (kN of a lane; kN = 0: read again for every bit), the
// smallest selected one found bit by bit with counts over the wave, then the selected pages in order by ballots.
constexpr int kSelectWaves = 4;
template <int kN>
__global__ void __launch_bounds__(64 * kSelectWaves) page_select_kernel(SelectArgs a) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * kSelectWaves + uniform(threadIdx.x >> 6);
  if (t >= a.qs.T) return;
  const int b = uniform(sequence_of(a.qs, t));
  const int seen = uniform(visible(a.qs, b, t));
  const int n = (seen + kPage - 1) / kPage;
  const int c0 = min(a.sink, n), c1 = max(c0, n - a.recent);   // candidates
  const bool all = n <= a.k;
  int left = a.k - a.sink - a.recent;                          // of them to select
  const float* row = a.scores + t * a.s_st;
  unsigned key[kN > 0 ? kN : 1];
  auto load = [&](int i) {
    const int p = 64 * i + lane;
    return p >= c0 && p < c1 ? ordered(row[p]) : 0u;
  };
  const int steps = (n + 63) / 64;
  if constexpr (kN > 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) key[i] = all ? 0u : load(i);
  }
  auto count = [&](auto test) {   // over the candidates
    int c = 0;
    if constexpr (kN > 0) {
#pragma unroll
      for (int i = 0; i < kN; ++i) c += __popcll(__ballot(test(key[i])));
    } else {
      for (int i = 0; i < steps; ++i) c += __popcll(__ballot(test(load(i))));
    }
    return c;
  };
  unsigned least = 0xffffffffu;   // of the selected
  int ties = 0;                   // of those equal to it
  if (!all && left > 0) {
    unsigned v = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const unsigned w = v | 1u << bit;
      if (count([&](unsigned x) { return x >= w; }) >= left) v = w;
    }
    least = v;
    ties = left - count([&](unsigned x) { return x > v; });
  }
  int at = 0;
  int32_t* table = a.sel_table + t * a.st_st;
  int32_t* index = a.sel_index + t * a.si_st;
  auto place = [&](int i, unsigned x) {
    const int p = 64 * i + lane;
    const uint64_t below = (1ull << lane) - 1;
    bool take = p < n;
    if (!all) {
      const bool candidate = p >= c0 && p < c1;
      const bool tie = candidate && left > 0 && x == least;
      const uint64_t tied = __ballot(tie);
      take = take && (!candidate || (left > 0 && (x > least || (tie && __popcll(tied & below) < ties))));
      ties -= min(ties, (int)__popcll(tied));
    }
    const uint64_t taken = __ballot(take);
    if (take) {
      const int to = at + __popcll(taken & below);
      index[to] = p;
      table[to] = a.block_table[b * a.bt_sb + p];
    }
    at += __popcll(taken);
  };
  if constexpr (kN > 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (64 * i < n) place(i, key[i]);
  } else {
    for (int i = 0; i < steps; ++i) place(i, all ? 0u : load(i));
  }
  for (int i = at + lane; i < a.k; i += 64) {
    index[i] = -1;
    table[i] = -1;
  }
  if (lane == 0) a.sel_lens[t] = seen - (n - at) * kPage;   // the last page is selected always, the others are full
}

int queries_validate(const char* what, const int32_t* cu, const int32_t* cache_seqlens, int64_t B, int64_t T,
                     int64_t max_pages, int64_t bt_sb) {
  if (B < 0 || T < 0 || max_pages < 0) return fail(DMLA_ERR_INVALID_ARG, "%s: negative size", what);
  if (cu == nullptr && B != T) return fail(DMLA_ERR_INVALID_ARG, "%s: without cu_seqlens_q there is one query per sequence", what);
  if (bt_sb < max_pages) return fail(DMLA_ERR_INVALID_ARG, "%s: block_table row stride < max_pages_per_seq", what);
  if (B > ((int64_t)1 << 24) || T > ((int64_t)1 << 30) || max_pages > ((int64_t)1 << 24))
    return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  if (T > 0 && B > 0 && cache_seqlens == nullptr) return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  return DMLA_OK;
}

// How the scores' work is cut (the workspace's size follows from it).
struct ScoreShape {
  int blocks, passes, group, chunk, chunks;
  int64_t groups;
};
ScoreShape score_shape(int64_t T, int64_t H, int64_t max_pages, bool packed) {
  ScoreShape s;
  const int64_t blocks = (H + 15) / 16;
  s.passes = (int)((blocks + kBlocks - 1) / kBlocks);
  s.blocks = (int)std::min<int64_t>(blocks, kBlocks);
  s.group = packed && s.passes == 1 ? kBlocks / s.blocks : 1;
  s.groups = (T + s.group - 1) / s.group;
  const int64_t most = std::max<int64_t>(1, (max_pages + 63) / 64);
  const int64_t want = std::max<int64_t>(1, 2 * device_cu_count() / std::max<int64_t>(1, s.groups));
  const int64_t each = (most + std::min(most, want) - 1) / std::min(most, want);
  s.chunk = (int)(64 * each);
  s.chunks = (int)((most + each - 1) / each);
  return s;
}

}  // namespace
}  // namespace dmla

using namespace dmla;

extern "C" int dmla_page_means(const void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                               const int32_t* starts, void* means, int64_t B, int64_t num_pages,
                               int64_t max_pages_per_seq, int64_t kv_sp, int64_t kv_ss, int64_t bt_sb, int64_t m_sp, int q4,
                               dmla_stream_t stream) {
  clear_error();
  const char* what = "dmla_page_means";
  if (B < 0 || num_pages < 0 || max_pages_per_seq < 0) return fail(DMLA_ERR_INVALID_ARG, "%s: negative size", what);
  // (Of an empty call any address does: empty tensors have none.)
  if (B > 0 && max_pages_per_seq > 0 && (!block_table || !cache_seqlens || (num_pages > 0 && (!kv_pool || !means))))
    return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  if (!aligned16(kv_pool) || !aligned16(means))
    return fail(DMLA_ERR_INVALID_ARG, "%s: kv_pool and means must be 16-byte aligned", what);
  const int64_t row = q4 ? kQ4RowBytes : 2 * kD;
  if (kv_ss % 16 != 0 || kv_sp % 16 != 0 || kv_ss < row || (q4 && kv_ss != row) || kv_sp < kPage * kv_ss)
    return fail(DMLA_ERR_INVALID_ARG, "%s: kv_pool strides must be multiples of 16 bytes and cover a row / page", what);
  if (!mult8(m_sp) || m_sp < kD) return fail(DMLA_ERR_INVALID_ARG, "%s: means' stride must be a multiple of 8 and cover a row", what);
  if (bt_sb < max_pages_per_seq) return fail(DMLA_ERR_INVALID_ARG, "%s: block_table row stride < max_pages_per_seq", what);
  if (B > ((int64_t)1 << 24) || num_pages > 0x7fffffff || max_pages_per_seq > ((int64_t)1 << 24))
    return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  if (B == 0 || max_pages_per_seq == 0 || num_pages == 0) return DMLA_OK;
  MeansArgs a = {};
  a.pool = static_cast<const char*>(kv_pool);
  a.block_table = block_table;
  a.seqlens = cache_seqlens;
  a.starts = starts;
  a.means = static_cast<bf16*>(means);
  a.kv_sp = kv_sp; a.kv_ss = kv_ss; a.bt_sb = bt_sb; a.m_sp = m_sp;
  a.B = (int)B; a.num_pages = (int)num_pages; a.max_pages = (int)max_pages_per_seq;
  const int64_t wgs = 8 * device_cu_count();
  const int64_t x = std::min(B, wgs), y = std::min<int64_t>(std::max<int64_t>(1, wgs / x), max_pages_per_seq);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)x, (unsigned)y), dim3(kMeanThreads), 0, (hipStream_t)stream, a);
  };
  if (q4) launch(page_means_kernel<true>);
  else launch(page_means_kernel<false>);
  return check_launch(what);
}

extern "C" int64_t dmla_page_scores_workspace_bytes(int64_t T, int64_t H, int64_t max_pages_per_seq, int packed) {
  if (T <= 0 || H <= 0 || max_pages_per_seq <= 0 || T > ((int64_t)1 << 30) || H > ((int64_t)1 << 16) ||
      max_pages_per_seq > ((int64_t)1 << 24))
    return 0;
  const ScoreShape s = score_shape(T, H, max_pages_per_seq, packed != 0);
  return s.chunks > 1 ? s.chunks * T * H * (int64_t)sizeof(float2) : 0;
}

extern "C" int dmla_page_scores(const void* q, const void* means, const int32_t* block_table, const int32_t* cache_seqlens,
                                const int32_t* cu_seqlens_q, float* scores, int64_t T, int64_t B, int64_t H, int64_t d_qk,
                                int64_t num_pages, int64_t max_pages_per_seq, int64_t q_st, int64_t q_sh, int64_t m_sp,
                                int64_t bt_sb, int64_t s_st, float softmax_scale, void* workspace, int64_t workspace_bytes,
                                dmla_stream_t stream) {
  clear_error();
  const char* what = "dmla_page_scores";
  const int rc = queries_validate(what, cu_seqlens_q, cache_seqlens, B, T, max_pages_per_seq, bt_sb);
  if (rc != DMLA_OK) return rc;
  if (H < 0 || num_pages < 0) return fail(DMLA_ERR_INVALID_ARG, "%s: negative size", what);
  if (d_qk != kD) return fail(DMLA_ERR_UNSUPPORTED, "%s: only d_qk=576 is compiled (got %lld)", what, (long long)d_qk);
  if (!(softmax_scale > 0.f) || !__builtin_isfinite(softmax_scale))
    return fail(DMLA_ERR_INVALID_ARG, "%s: softmax_scale must be finite and > 0", what);
  if (!aligned16(q) || !aligned16(means)) return fail(DMLA_ERR_INVALID_ARG, "%s: q and means must be 16-byte aligned", what);
  if (!mult8(q_st) || !mult8(q_sh) || !mult8(m_sp) || m_sp < kD)
    return fail(DMLA_ERR_INVALID_ARG, "%s: strides must be multiples of 8 elements and cover a row", what);
  if (s_st < max_pages_per_seq) return fail(DMLA_ERR_INVALID_ARG, "%s: scores' row stride < max_pages_per_seq", what);
  if (H > ((int64_t)1 << 16) || num_pages > 0x7fffffff) return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  if (T == 0 || max_pages_per_seq == 0) return DMLA_OK;
  if (!scores || (H > 0 && !q) || (B > 0 && !block_table) || (num_pages > 0 && !means))
    return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  if (H == 0 || num_pages == 0) return fail(DMLA_ERR_INVALID_ARG, "%s: no heads or no pages", what);
  const ScoreShape s = score_shape(T, H, max_pages_per_seq, cu_seqlens_q != nullptr);
  if (s.groups > 0x7fffffff || s.chunks > 65535) return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  const int64_t need = s.chunks > 1 ? s.chunks * T * H * (int64_t)sizeof(float2) : 0;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(DMLA_ERR_WORKSPACE, "%s: workspace of %lld bytes needed (got %lld)", what, (long long)need,
                (long long)workspace_bytes);
  if (need > 0 && !aligned16(workspace)) return fail(DMLA_ERR_INVALID_ARG, "%s: workspace must be 16-byte aligned", what);
  ScoreArgs a = {};
  a.q = static_cast<const bf16*>(q);
  a.means = static_cast<const bf16*>(means);
  a.block_table = block_table;
  a.qs = Queries{cu_seqlens_q, cache_seqlens, (int)B, (int)T, (int)max_pages_per_seq};
  a.scores = scores;
  a.stats = static_cast<float2*>(workspace);
  a.q_st = q_st; a.q_sh = q_sh; a.m_sp = m_sp; a.bt_sb = bt_sb; a.s_st = s_st;
  a.H = (int)H; a.num_pages = (int)num_pages;
  a.blocks = s.blocks; a.passes = s.passes; a.group = s.group; a.chunk = s.chunk; a.chunks = s.chunks;
  a.scale_log2 = softmax_scale * kLog2e;
  const dim3 grid((unsigned)s.groups, (unsigned)s.chunks);
  const size_t lds = (size_t)16 * (s.passes > 1 ? kBlocks : s.blocks * s.group) * kRowBytes;
  auto launch = [&](auto kernel) -> int {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return fail(DMLA_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    hipLaunchKernelGGL(kernel, grid, dim3(kScoreThreads), lds, (hipStream_t)stream, a);
    return check_launch(what);
  };
  if (s.chunks == 1) return launch(page_scores_kernel<kFused>);
  const int first = launch(page_scores_kernel<kStats>);
  return first != DMLA_OK ? first : launch(page_scores_kernel<kSum>);
}

extern "C" int dmla_page_select(const float* scores, const int32_t* block_table, const int32_t* cache_seqlens,
                                const int32_t* cu_seqlens_q, int32_t* sel_table, int32_t* sel_lens, int32_t* sel_index,
                                int64_t T, int64_t B, int64_t max_pages_per_seq, int64_t s_st, int64_t bt_sb, int64_t st_st,
                                int64_t si_st, int64_t top_pages, int64_t recent, int64_t sink, dmla_stream_t stream) {
  clear_error();
  const char* what = "dmla_page_select";
  const int rc = queries_validate(what, cu_seqlens_q, cache_seqlens, B, T, max_pages_per_seq, bt_sb);
  if (rc != DMLA_OK) return rc;
  if (recent < 1 || sink < 0 || top_pages < recent + sink)
    return fail(DMLA_ERR_INVALID_ARG, "%s: recent must be at least 1, sink at least 0, and top_pages cover both", what);
  if (top_pages > ((int64_t)1 << 24)) return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  if (s_st < max_pages_per_seq) return fail(DMLA_ERR_INVALID_ARG, "%s: scores' row stride < max_pages_per_seq", what);
  if (st_st < top_pages || si_st < top_pages)
    return fail(DMLA_ERR_INVALID_ARG, "%s: sel_table and sel_index rows must hold top_pages entries", what);
  if (T == 0) return DMLA_OK;
  if (!sel_table || !sel_lens || !sel_index || (max_pages_per_seq > 0 && (!scores || (B > 0 && !block_table))))
    return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  SelectArgs a = {};
  a.scores = scores;
  a.block_table = block_table;
  a.qs = Queries{cu_seqlens_q, cache_seqlens, (int)B, (int)T, (int)max_pages_per_seq};
  a.sel_table = sel_table;
  a.sel_lens = sel_lens;
  a.sel_index = sel_index;
  a.s_st = s_st; a.bt_sb = bt_sb; a.st_st = st_st; a.si_st = si_st;
  a.k = (int)top_pages; a.recent = (int)recent; a.sink = (int)sink;
  const dim3 grid((unsigned)((T + kSelectWaves - 1) / kSelectWaves));
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kSelectWaves), 0, (hipStream_t)stream, a);
  };
  if (max_pages_per_seq <= 64 * 2) launch(page_select_kernel<2>);
  else if (max_pages_per_seq <= 64 * 8) launch(page_select_kernel<8>);
  else if (max_pages_per_seq <= 64 * 32) launch(page_select_kernel<32>);
  else launch(page_select_kernel<0>);
  return check_launch(what);
}
