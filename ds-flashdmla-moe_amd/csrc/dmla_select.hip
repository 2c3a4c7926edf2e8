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
#include "dmla_pipe.h"
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

// A page per workgroup at a time: thread (g, c) adds the rows of group g in piece c, the groups meet in LDS, in order.
// Pieces are 16 bytes of a row: of bf16 rows 8 columns, of 4-bit rows 32 columns (16 of those, and eight of the rope's).
// Bound: of bf16 rows HBM (64 sequences of 500 pages 461 us, 5.1 TB/s), of 4-bit rows conversions and additions (271 us, 3.0
// TB/s; a word of codes and a byte of scale a load took 684); a decode step has at most one new full page per sequence
// and is a launch.
template <bool kQ4>
struct MeanShape {
  static constexpr int kPieces = kQ4 ? kLat / 32 + (kD - kLat) / 8 : kD / 8;
  static constexpr int kGroups = kQ4 ? 16 : 8, kThreads = kGroups * kPieces, kRows = kPage / kGroups;   // 384 or 576 threads
};
template <bool kQ4>
__global__ void __launch_bounds__(MeanShape<kQ4>::kThreads) page_means_kernel(MeansArgs a) {
  using Shape = MeanShape<kQ4>;
  __shared__ __attribute__((aligned(16))) float part[Shape::kGroups][kD];
  const int g = threadIdx.x / Shape::kPieces, c = threadIdx.x % Shape::kPieces;
  const bool codes = kQ4 && c < kLat / 32;
  const int offset = !kQ4 || codes ? 16 * c : kQ4RopeOff + 16 * (c - kLat / 32);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int64_t len = min((int64_t)a.seqlens[b], (int64_t)a.max_pages * kPage);
    const int first = a.starts != nullptr ? max(a.starts[b], 0) / kPage : 0;
    for (int64_t p = first + blockIdx.y; p < len / kPage; p += gridDim.y) {
      const int page = a.block_table[b * a.bt_sb + p];
      if (page < 0 || page >= a.num_pages) continue;   // (uniform)
      u32x4 v[Shape::kRows];
      int scale[Shape::kRows] = {};
#pragma unroll
      for (int r = 0; r < Shape::kRows; ++r) {
        const char* row = a.pool + page * a.kv_sp + (g * Shape::kRows + r) * a.kv_ss;
        v[r] = *reinterpret_cast<const u32x4*>(row + offset);
        if (codes) scale[r] = (uint8_t)row[kQ4ScaleOff + c];
      }
      if (codes) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          float x[8] = {};
#pragma unroll
          for (int r = 0; r < Shape::kRows; ++r) {
            const bf16x8 o = q4_octet(v[r][w], q4_scale(scale[r]));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] += (float)o[i];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) part[g][32 * c + 8 * w + i] = x[i];
        }
      } else {
        float x[8] = {};
#pragma unroll
        for (int r = 0; r < Shape::kRows; ++r) {
          const bf16x8 o = __builtin_bit_cast(bf16x8, v[r]);
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] += (float)o[i];
        }
        const int column = kQ4 ? kLat + 8 * (c - kLat / 32) : 8 * c;
#pragma unroll
        for (int i = 0; i < 8; ++i) part[g][column + i] = x[i];
      }
      __syncthreads();
      if (threadIdx.x < kD / 4) {
        f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int o = 0; o < Shape::kGroups; ++o) sum += *reinterpret_cast<const f32x4*>(&part[o][4 * threadIdx.x]);
        bf16x4 m;
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = (bf16)(sum[i] * (1.0f / kPage));
        *reinterpret_cast<bf16x4*>(a.means + page * a.m_sp + 4 * threadIdx.x) = m;
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
  float* kept;     // [T, H, kept_sp]: the products q . mean, where they are kept
  int64_t q_st, q_sh, m_sp, bt_sb, s_st, kept_sp;
  int H, num_pages;
  int blocks, passes;   // 16-row blocks of a query (at most kBlocks of a pass), passes over the heads
  int group;            // queries of a workgroup
  int chunk, chunks;    // pages of a workgroup, a multiple of kTile
  float scale_log2;
};

constexpr int kScoreThreads = 256, kScoreWaves = 4;
constexpr int kBlocks = 8;                                // 16-row blocks of a workgroup, heads padded to 16: two a wave
constexpr int kTile = 32;                                 // pages of a tile
constexpr int kSteps = kD / 16, kLatSteps = kLat / 16;    // MFMAs of a tile
constexpr int kMeanRow = 2 * kLat, kTileBytes = kTile * kMeanRow, kRopeBytes = kTile * 2 * (kD - kLat), kRing = 4;
constexpr int kCopies = 9;                                // of a wave and tile
constexpr int kIdTiles = 64;                              // tiles whose table entries are in LDS
constexpr int kQueryBytes = 32 * 2 * kD;                  // of a wave, in the tiles' memory
static_assert(kScoreWaves * kQueryBytes == kRing * (kTileBytes + kRopeBytes), "the queries fill it");
enum { kFused, kStats, kKeep, kSum };

// 16-byte unit u of row r of a tile lies at u ^ mean_swz(r): 16 rows' units at one place of a row lie in different banks.
__device__ __forceinline__ int mean_swz(int r) { return r & 15; }

// A head's largest score (0: none) and the inverse of its sum, over all chunks of the pages; of heads that are not there
// such that every weight is 0.  (Apart: their product's logarithm would lose the digits of a large maximum.)
__device__ __forceinline__ void head_sums(const ScoreArgs& a, int t, int head, float& top, float& inverse) {
  float m = kNegInf, l = 0.f;
  constexpr int kLoads = 4;   // in flight (one: 100000 tokens x 128 heads 28 us, four 21, sixteen 24)
  for (int c0 = 0; c0 < a.chunks; c0 += kLoads) {
    float2 s[kLoads];
#pragma unroll
    for (int c = 0; c < kLoads; ++c) s[c] = a.stats[((int64_t)min(c0 + c, a.chunks - 1) * a.qs.T + t) * a.H + min(head, a.H - 1)];
#pragma unroll
    for (int c = 0; c < kLoads; ++c) {
      if (c0 + c >= a.chunks) break;
      const float mm = fmaxf(m, s[c].x);
      l = mm == kNegInf ? l + s[c].y : l * fast_exp2(m - mm) + s[c].y * fast_exp2(s[c].x - mm);   // (0 or not a number)
      m = mm;
    }
  }
  top = head >= a.H ? __builtin_inff() : m == kNegInf ? 0.f : m;
  inverse = head >= a.H || l == 0.f ? 0.f : 1.f / l;
}

// kFused: one workgroup has all pages of its queries, their sums first and then the scores.  Else the pages are cut in
// chunks over workgroups: kStats leaves each chunk's maxima and sums and kSum reads all of them, with the products once
// more; kKeep leaves the products too, for page_sums_kernel.
//
// A wave holds 32 rows (query, head) in registers, as chunk attention does, and tiles of 32 mean rows come through LDS,
// three tiles ahead.  For the sums over pages the means are the MFMA's rows, so a lane has 16 pages of one head; for
// the sums over heads they are its columns, so a lane has 16 heads of one page.  Both sums are then in-lane, in a
// fixed order.
// Bound: a few tiles a workgroup by latency (a launch, 147 KB of queries 3 us, the first tile 2); a tile takes 1.2 us, the
// LDS reads of four waves that each need all of it; long tables by HBM (64 queries x 128 heads x 2000 pages, 280 MB with the
// products: 58 us).
template <int kMode>
__global__ void __launch_bounds__(kScoreThreads, 1) page_scores_kernel(ScoreArgs a) {
  __shared__ __attribute__((aligned(1024))) char mem[kRing * (kTileBytes + kRopeBytes)];
  __shared__ int s_seq[kBlocks], s_pages[kBlocks];
  __shared__ __attribute__((aligned(16))) float s_max[16 * kBlocks], s_inv[16 * kBlocks];
  __shared__ float s_part[2][kBlocks][kTile];
  __shared__ int s_ids[kIdTiles * kTile];
  const unsigned tiles = lds_addr((DMLA_LDS char*)mem), ropes = tiles + kRing * kTileBytes;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int t0 = blockIdx.x * a.group, nt = min(a.group, a.qs.T - t0);
  const int c0 = blockIdx.y * a.chunk, c1 = min(c0 + a.chunk, a.qs.max_pages);
  const bool multi = a.passes > 1;   // the heads of one query take several passes
  // Row r of the workgroup: query i, head `head0` + offset.
  auto query_of = [&](int r) { return multi ? 0 : min((r >> 4) / a.blocks, nt - 1); };
  auto head_of = [&](int r) { return multi ? r : (((r >> 4) % a.blocks) << 4) + (r & 15); };
  for (int pass = 0; pass < a.passes; ++pass) {
    const int head0 = pass * 16 * kBlocks;
    if (pass > 0) __syncthreads();
    // ---- queries: operand c holds dims 16 c + 8 hl .. of row 32 wave + l32; eight rows x 128 bytes a copy ----
    const unsigned mine = tiles + wave * kQueryBytes;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = 32 * wave + 8 * g + (lane >> 3);
      const int head = min(head0 + head_of(r), a.H - 1);
      const bf16* src = a.q + (t0 + query_of(r)) * a.q_st + head * a.q_sh + 8 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
      for (int i = 0; i < 9; ++i) dma16_addr(src + 64 * i, mine + (9 * g + i) * 1024);
    }
    if (pass == 0) {
      for (int i = wave; i < nt; i += kScoreWaves) {
        const int b = sequence_of(a.qs, t0 + i);
        const int n = visible(a.qs, b, t0 + i);
        if (lane == 0) {
          s_seq[i] = b;
          s_pages[i] = n > 0 ? (n - 1) / kPage : 0;   // pages before its own
        }
      }
    }
    if constexpr (kMode == kSum) {
      for (int r = tid; r < 16 * kBlocks; r += kScoreThreads) {
        const int head = head0 + head_of(r), i = query_of(r);
        head_sums(a, t0 + i, head, s_max[r], s_inv[r]);
      }
    }
    wait_vm<0>();
    bf16x8 q[kSteps];
    {
      const unsigned at = lds_sum(9 * 1024 * (l32 >> 3) + 128 * (l32 & 7) + 16 * (hl ^ (l32 & 7)), mine);
#pragma unroll
      for (int c = 0; c < kSteps; ++c) q[c] = *lds_ptr<const bf16x8>((at ^ (32 * (c & 3))) + 1024 * (c >> 2));
    }
    wait_lds();
    __syncthreads();   // the tiles' memory is free; the queries' pages are known

    for (int i0 = 0; i0 < nt;) {   // the queries of one sequence at a time
      const int b = uniform(s_seq[i0]);
      int i1 = i0 + 1, most = s_pages[i0];
      for (; i1 < nt && s_seq[i1] == b; ++i1) most = max(most, s_pages[i1]);
      i1 = uniform(i1);
      most = uniform(most);
      const int n_tiles = max(0, (min(most, c1) - c0 + kTile - 1) / kTile);
      auto rows_pages = [&](int r) {   // pages of row r's query, 0 where it is of another sequence
        const int i = query_of(r);
        return i >= i0 && i < i1 ? s_pages[i] : 0;
      };
      // Tiles in order, each through each(s, k, there, beside): operand reader, a bit per page in the pool, what runs after product c.
      auto stream = [&](auto each) {
        if (n_tiles == 0) return;
        // Table entries of tiles [s, s + kIdTiles / 2), -1 where there is no page of the pool.
        auto load_ids = [&](int s) {
          for (int k = tid; k < kIdTiles / 2 * kTile; k += kScoreThreads) {
            const int p = c0 + kTile * s + k;
            const int id = p < min(most, c1) ? a.block_table[b * a.bt_sb + p] : -1;
            s_ids[(kTile * s + k) % (kTile * kIdTiles)] = id < a.num_pages ? id : -1;
          }
        };
        // Tile s's pages of this wave (past the end: the last tile once more, so that the copies count the same), and copy i
        // of kCopies.
        auto pages_of = [&](int s) {
          return max(s_ids[(kTile * min(s, n_tiles - 1)) % (kTile * kIdTiles) + 8 * wave + (lane >> 3)], 0);   // not there: page 0, masked
        };
        auto copy = [&](int s, int id, int i) {
          const unsigned slot = (unsigned)(s % kRing);
          const int r = 8 * wave + i;
          if (i < 8) dma16(a.means + __builtin_amdgcn_readlane(id, 8 * i) * a.m_sp, 16 * (lane ^ mean_swz(r)), tiles + slot * kTileBytes + r * kMeanRow);
          else dma16_addr(a.means + id * a.m_sp + kLat + 8 * ((lane & 7) ^ (lane >> 3)), ropes + slot * kRopeBytes + wave * 1024);
        };
        load_ids(0);
        if (n_tiles > kIdTiles / 2) load_ids(kIdTiles / 2);
        __syncthreads();
        for (int s = 0; s < 3; ++s) {
          const int id = pages_of(s);
#pragma unroll
          for (int i = 0; i < kCopies; ++i) copy(s, id, i);
        }
        for (int s = 0; s < n_tiles; ++s) {
          // Half the entries ahead of their use, into the half that every wave is past.
          if (s > 1 && s % (kIdTiles / 2) == 1 && s - 1 + kIdTiles / 2 < n_tiles) load_ids(s - 1 + kIdTiles / 2);
          wait_vm<2 * kCopies>();   // tile s; those of two tiles more may be on their way (or stores of an earlier one)
          __syncthreads();          // tile s landed, tile s - 1 is read
          const int id = pages_of(s + 3);
          const unsigned key = lds_sum(kMeanRow * l32 + 16 * (hl ^ mean_swz(l32)), tiles + (unsigned)(s % kRing) * kTileBytes);
          const unsigned rope = lds_sum(128 * l32 + 16 * (hl ^ (l32 & 7)), ropes + (unsigned)(s % kRing) * kRopeBytes);
          each(s, [&](int c) {
            return *lds_ptr<const bf16x8>(c < kLatSteps ? (key ^ (32 * (c & 7))) + 256 * (c >> 3) : rope ^ (32 * (c - kLatSteps)));
          }, (unsigned)__ballot(s_ids[(kTile * s) % (kTile * kIdTiles) + l32] >= 0), [&](int c) {   // between its products
            if (c % 4 == 1) copy(s + 3, id, c / 4);
          });
        }
        wait_vm<0>();
        __syncthreads();   // the last tile is read, no copy is on its way
      };
      // A tile's products; operands are read kDepth MFMAs ahead (left to the compiler, each waits for its own: 3800
      // cycles a tile instead of 2800).
      auto product = [&](auto k, auto beside, auto multiply) {
        constexpr int kDepth = 8;
        bf16x8 mean[kDepth];
#pragma unroll
        for (int c = 0; c < kDepth; ++c) mean[c] = k(c);
        f32x16 x = {};
        static_for<kSteps>([&](auto c_tag) {
          constexpr int c = decltype(c_tag)::value;
          x = multiply(mean[c % kDepth], q[c], x);
          if constexpr (c + kDepth < kSteps) mean[c % kDepth] = k(c + kDepth);
          beside(c);
          in_order();
        });
        return x;
      };
      // Bit k: page k of tile s is one of the first n of the sequence.
      auto first_pages = [&](int s, int n) {
        const int k = n - c0 - kTile * s;
        return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1;
      };
      if constexpr (kMode != kSum) {
        float m = kNegInf, l = 0.f;   // of row 32 wave + l32
        const int limit = rows_pages(32 * wave + l32);
        const int r = 32 * wave + l32, i = query_of(r), head = head0 + head_of(r);
        // (Rows behind the last query are its rows again.)
        const bool own = i >= i0 && i < i1 && (multi || (r >> 4) / a.blocks < nt);
        float* keep = nullptr;
        if constexpr (kMode == kKeep)
          if (own && head < a.H) keep = a.kept + ((int64_t)(t0 + i) * a.H + head) * a.kept_sp + c0 + 4 * hl;
        stream([&](int s, auto k, unsigned there, auto beside) {
          f32x16 x = product(k, beside, [](const bf16x8& mean, const bf16x8& row, const f32x16& x) { return mfma32_bf16(mean, row, x); });
          if constexpr (kMode == kKeep) {
            if (keep != nullptr) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4*>(keep + kTile * s + 8 * j) = f32x4{x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
            }
          }
          const unsigned seen = (there & first_pages(s, limit)) >> (4 * hl);
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = seen >> (8 * (i >> 2) + (i & 3)) & 1 ? x[i] * a.scale_log2 : kNegInf;
          float top = x[0];
#pragma unroll
          for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
          const float mm = fmaxf(m, half_max(top));
          const float ms = mm == kNegInf ? 0.f : mm;
          l = m == mm ? l : l * fast_exp2(m - mm);
          m = mm;
#pragma unroll
          for (int i = 0; i < 16; ++i) l += fast_exp2(x[i] - ms);   // (not a number stays)
        });
        l = half_sum(l);
        if (hl == 0 && own) {
          if constexpr (kMode == kStats || kMode == kKeep) {
            if (head < a.H) a.stats[((int64_t)blockIdx.y * a.qs.T + t0 + i) * a.H + head] = make_float2(m, l);
          } else {
            s_max[r] = head >= a.H ? __builtin_inff() : m == kNegInf ? 0.f : m;
            s_inv[r] = head >= a.H || l == 0.f ? 0.f : 1.f / l;
          }
        }
        __syncthreads();
      }
      if constexpr (kMode == kFused || kMode == kSum) {
        // Scores of tile s: the sums of each query's blocks, posted by the waves.
        auto put = [&](int s) {
          const int i = tid >> 5, p = c0 + kTile * s + (tid & 31);
          if (i < i0 || i >= i1 || p >= c1) return;
          float v = 0.f;
          const int first = multi ? 0 : i * a.blocks, n = multi ? kBlocks : a.blocks;
          for (int j = 0; j < n; ++j) v += s_part[s & 1][first + j][tid & 31];
          float* to = a.scores + (t0 + i) * a.s_st + p;
          *to = pass > 0 ? *to + v : v;
        };
        float mx[16], inv[16];   // of rows 8 (i / 4) + 4 hl + i % 4 of the wave
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f32x4 u = *reinterpret_cast<const DMLA_LDS f32x4*>((const DMLA_LDS float*)s_max + 32 * wave + 8 * j + 4 * hl);
          const f32x4 v = *reinterpret_cast<const DMLA_LDS f32x4*>((const DMLA_LDS float*)s_inv + 32 * wave + 8 * j + 4 * hl);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mx[4 * j + i] = u[i];
            inv[4 * j + i] = v[i];
          }
        }
        const int limit0 = rows_pages(32 * wave), limit1 = rows_pages(32 * wave + 16);
        stream([&](int s, auto k, unsigned there, auto beside) {
          if (s > 0) put(s - 1);
          const f32x16 x = product(k, beside, [](const bf16x8& mean, const bf16x8& row, const f32x16& x) { return mfma32_bf16(row, mean, x); });
          float v0 = 0.f, v1 = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v0 += fast_exp2(__builtin_fmaf(x[i], a.scale_log2, -mx[i])) * inv[i];
            v1 += fast_exp2(__builtin_fmaf(x[8 + i], a.scale_log2, -mx[8 + i])) * inv[8 + i];
          }
          v0 = half_sum(v0);
          v1 = half_sum(v1);
          if (hl == 0) {
            s_part[s & 1][2 * wave][l32] = (there & first_pages(s, limit0)) >> l32 & 1 ? v0 : 0.f;
            s_part[s & 1][2 * wave + 1][l32] = (there & first_pages(s, limit1)) >> l32 & 1 ? v1 : 0.f;
          }
        });
        if (n_tiles > 0) put(n_tiles - 1);
        // Behind the last page that any of them sees: zeros.
        if (pass == 0)
          for (int s = n_tiles; c0 + kTile * s < c1; ++s) {
            const int i = tid >> 5, p = c0 + kTile * s + (tid & 31);
            if (i >= i0 && i < i1 && p < c1) a.scores[(t0 + i) * a.s_st + p] = 0.f;
          }
        __syncthreads();   // the last tile's sums are read
      }
      i0 = i1;
    }
  }
}

// The scores of a query's pages from what was kept of each head, 64 pages a wave (a lane has a page); with a.split > 1
// that many waves share the heads of a page, their sums in a fixed order.
// Bound: latency (what the first kernel kept is in the last-level cache).
constexpr int kSumHeads = 128, kSumLoads = 16;
__global__ void __launch_bounds__(kScoreThreads) page_sums_kernel(ScoreArgs a, int split) {
  __shared__ float s_max[kSumHeads], s_inv[kSumHeads], s_part[kScoreWaves][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int t = blockIdx.y, p = 64 * ((int)blockIdx.x * (kScoreWaves / split) + wave / split) + lane;
  const int b = sequence_of(a.qs, t), n = visible(a.qs, b, t);
  const int pages = uniform(n > 0 ? (n - 1) / kPage : 0);
  const bool any = 64 * (int)blockIdx.x * (kScoreWaves / split) < pages;   // of this workgroup's
  bool there = false;
  float v = 0.f;
  if (any) {
    if (p < pages) {
      const int id = a.block_table[b * a.bt_sb + p];
      there = id >= 0 && id < a.num_pages;
    }
    const float* x = a.kept + (int64_t)t * a.H * a.kept_sp + min(p, pages - 1);
    for (int h0 = 0; h0 < a.H; h0 += kSumHeads) {
      const int heads = min(kSumHeads, a.H - h0), each = (heads + split - 1) / split;
      const int first = (wave % split) * each, last = min(first + each, heads);
      __syncthreads();   // those before are read
      for (int h = tid; h < heads; h += kScoreThreads) head_sums(a, t, h0 + h, s_max[h], s_inv[h]);
      __syncthreads();
      for (int h = first; h < last; h += kSumLoads) {
        float k[kSumLoads];
#pragma unroll
        for (int i = 0; i < kSumLoads; ++i) k[i] = x[(int64_t)(h0 + min(h + i, last - 1)) * a.kept_sp];
#pragma unroll
        for (int i = 0; i < kSumLoads; ++i)
          if (h + i < last) v += fast_exp2(__builtin_fmaf(k[i], a.scale_log2, -s_max[h + i])) * s_inv[h + i];
      }
    }
  }
  if (split > 1) {
    s_part[wave][lane] = v;
    __syncthreads();
    if (wave % split != 0) return;
    for (int w = 1; w < split; ++w) v += s_part[wave + w][lane];
  }
  if (p < a.qs.max_pages) a.scores[t * a.s_st + p] = there ? v : 0.f;
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

// A query per wave: its candidates' scores and table entries in registers (kN of a lane; kN = 0: read again for every bit).
// The smallest selected score is found bit by bit, from the highest bit in which candidates differ, with counts over
// the wave, until the candidates at or above are as many as asked for; then the selected pages go out in order, their
// places from ballots.
// Bound: latency; a query of 512 pages takes 5 dependent loads and some 15 counts.
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
  const int left = a.k - a.sink - a.recent;                    // of them to select
  const float* row = a.scores + t * a.s_st;
  const int32_t* entries = a.block_table + b * a.bt_sb;
  unsigned key[kN > 0 ? kN : 1];
  int entry[kN > 0 ? kN : 1];
  auto load = [&](int i) {   // 0: no candidate
    const int p = 64 * i + lane;
    return p >= c0 && p < c1 ? ordered(row[p]) : 0u;
  };
  const int steps = (n + 63) / 64;
  if constexpr (kN > 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int p = 64 * i + lane;
      entry[i] = p < n ? entries[p] : 0;
      key[i] = all ? 0u : load(i);
    }
  }
  auto over = [&](auto f) {   // the candidates' keys of this lane
    if constexpr (kN > 0) {
#pragma unroll
      for (int i = 0; i < kN; ++i) f(key[i]);
    } else {
      for (int i = 0; i < steps; ++i) f(load(i));
    }
  };
  auto wave_sum = [&](int c) { return __builtin_amdgcn_readlane(lane_scan(c), 63); };
  auto at_least = [&](unsigned w) {
    int c = 0;
    over([&](unsigned x) { c += x >= w ? 1 : 0; });
    return wave_sum(c);
  };
  unsigned least = 0xffffffffu;   // selected: the keys above it, and the first `ties` of those equal to it
  int ties = 0;
  if (!all && left > 0) {
    unsigned ones = 0, zeros = 0;   // bits set, and not set, in some candidate
    over([&](unsigned x) {
      ones |= x;
      zeros |= x != 0 ? ~x : 0u;
    });
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      ones |= __shfl_xor(ones, o, 64);
      zeros |= __shfl_xor(zeros, o, 64);
    }
    const unsigned differ = ones & zeros;
    const int top = differ != 0 ? 31 - __builtin_clz(differ) : -1;
    unsigned v = top < 31 ? ones >> (top + 1) << (top + 1) : 0u;   // what they have in common
    if (top < 0) v = ones;
    int above = -1;   // candidates >= v, where counted
    for (int bit = top; bit >= 0 && above != left; --bit) {
      const unsigned w = v | 1u << bit;
      const int c = at_least(w);
      if (c >= left) {
        v = w;
        above = c;
      }
    }
    least = v;
    int c = 0;
    over([&](unsigned x) { c += x > v ? 1 : 0; });
    // (v need not be a candidate's key where exactly as many as asked for are at or above it)
    ties = left - wave_sum(c);
  }
  int at = 0;
  int32_t* table = a.sel_table + t * a.st_st;
  int32_t* index = a.sel_index + t * a.si_st;
  auto place = [&](int i, unsigned x, int e) {
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
      table[to] = e;
    }
    at += __popcll(taken);
  };
  if constexpr (kN > 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (64 * i < n) place(i, key[i], entry[i]);
  } else {
    for (int i = 0; i < steps; ++i) {
      const int p = 64 * i + lane;
      place(i, all ? 0u : load(i), p < n ? entries[p] : 0);
    }
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
  int64_t kept_sp;   // 0: the products are not kept

  int64_t stats_bytes(int64_t T, int64_t H) const { return (chunks > 1 ? chunks * T * H * (int64_t)sizeof(float2) : 0) + 15 & ~(int64_t)15; }
  int64_t bytes(int64_t T, int64_t H) const { return stats_bytes(T, H) + T * H * kept_sp * (int64_t)sizeof(float); }
};
// Up to here the products are kept (64 queries x 128 heads x 500 / 8000 pages: 26 / 234 us, computed again 31 / 247).
constexpr int64_t kKeepBytes = (int64_t)512 << 20;
ScoreShape score_shape(int64_t T, int64_t H, int64_t max_pages, bool packed) {
  ScoreShape s;
  const int64_t blocks = (H + 15) / 16;
  s.passes = (int)((blocks + kBlocks - 1) / kBlocks);
  s.blocks = (int)std::min<int64_t>(blocks, kBlocks);
  s.group = packed && s.passes == 1 ? kBlocks / s.blocks : 1;
  s.groups = (T + s.group - 1) / s.group;
  // As many chunks of the pages as fill the CUs once.
  const int64_t most = std::max<int64_t>(1, (max_pages + kTile - 1) / kTile);
  const int64_t want = std::min(most, std::max<int64_t>(1, device_cu_count() / std::max<int64_t>(1, s.groups)));
  const int64_t each = (most + want - 1) / want;
  s.chunk = (int)(kTile * each);
  s.chunks = (int)((most + each - 1) / each);
  s.kept_sp = s.chunks > 1 && T * H * most * kTile <= kKeepBytes / (int64_t)sizeof(float) ? most * kTile : 0;
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
  const dim3 grid((unsigned)x, (unsigned)y);
  if (q4) hipLaunchKernelGGL(page_means_kernel<true>, grid, dim3(MeanShape<true>::kThreads), 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL(page_means_kernel<false>, grid, dim3(MeanShape<false>::kThreads), 0, (hipStream_t)stream, a);
  return check_launch(what);
}

extern "C" int64_t dmla_page_scores_workspace_bytes(int64_t T, int64_t H, int64_t max_pages_per_seq, int packed) {
  if (T <= 0 || H <= 0 || max_pages_per_seq <= 0 || T > ((int64_t)1 << 30) || H > ((int64_t)1 << 16) ||
      max_pages_per_seq > ((int64_t)1 << 24))
    return 0;
  const ScoreShape s = score_shape(T, H, max_pages_per_seq, packed != 0);
  return s.bytes(T, H);
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
  const int64_t need = s.bytes(T, H);
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
  a.kept = reinterpret_cast<float*>(static_cast<char*>(workspace) + s.stats_bytes(T, H));
  a.kept_sp = s.kept_sp;
  a.q_st = q_st; a.q_sh = q_sh; a.m_sp = m_sp; a.bt_sb = bt_sb; a.s_st = s_st;
  a.H = (int)H; a.num_pages = (int)num_pages;
  a.blocks = s.blocks; a.passes = s.passes; a.group = s.group; a.chunk = s.chunk; a.chunks = s.chunks;
  a.scale_log2 = softmax_scale * kLog2e;
  const dim3 grid((unsigned)s.groups, (unsigned)s.chunks);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kScoreThreads), 0, (hipStream_t)stream, a);
    return check_launch(what);
  };
  if (s.chunks == 1) return launch(page_scores_kernel<kFused>);
  if (s.kept_sp > 0) {
    const int kept = launch(page_scores_kernel<kKeep>);
    if (kept != DMLA_OK) return kept;
    const int split = H > kSumHeads / kScoreWaves ? kScoreWaves : 1;
    const int64_t wide = 64 * (kScoreWaves / split);
    hipLaunchKernelGGL(page_sums_kernel, dim3((unsigned)((max_pages_per_seq + wide - 1) / wide), (unsigned)T), dim3(kScoreThreads), 0,
                       (hipStream_t)stream, a, split);   // (several chunks: no more than 1024 queries)
    return check_launch(what);
  }
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
