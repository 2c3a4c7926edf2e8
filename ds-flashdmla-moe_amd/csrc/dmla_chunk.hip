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
//  * The softmax reference of a row is its largest score in the first tile; P may grow to 2^32 past it.
#include <algorithm>

#include "dmla_host.h"
#include "dmla_pipe.h"

namespace dmla {
namespace {

constexpr int kDqk = 576, kDv = 512, kPage = 64;
constexpr int kTile = 32;                                  // keys of a tile
constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 128, kRowBlocks = kRows / 32;        // of a workgroup
constexpr int kColBlocks = 4;                              // 32 columns each, of a wave
constexpr int kSteps = kDqk / 16, kLatSteps = kDv / 16;    // MFMAs of a tile's scores
constexpr int kKeyRow = 1024, kKeyBytes = kTile * kKeyRow, kSlots = 4;
constexpr int kRopeBytes = kTile * 128;
constexpr int kProbBytes = kWaves * 2048;
constexpr int kQueryBytes = 32 * 2 * kDqk;                 // of a wave, in the keys' and the ropes' memory
static_assert(kWaves * kQueryBytes == kSlots * (kKeyBytes + kRopeBytes), "the queries fill it");
constexpr float kHeadroom = 32.0f;                         // log2 headroom of P over a row's reference

__device__ __forceinline__ int key_swz(int r) { return (r & 3) << 2 | (r >> 2 & 3); }

struct ChunkParams {
  const bf16* q;
  const char* kv;
  const int32_t* block_table;
  const int32_t* seqlens;
  const int32_t* cu;     // nullable: one query per sequence
  bf16* o;
  float* lse;            // nullable
  int64_t q_st, q_sh, kv_sp, kv_ss, bt_sb, o_st, o_sh;   // kv strides in bytes
  int T, B, H, num_pages, max_pages, causal;
  FastDiv hdiv;          // division by H
  float scale_log2;
};

// A sequence's queries: q0 .. q0 + n - 1, the first of them at token `base` of its len tokens.
struct Sequence {
  int q0, n, len;
};
__device__ __forceinline__ Sequence sequence(const ChunkParams& p, int b) {
  Sequence s;
  s.len = (int)min((int64_t)max(p.seqlens[b], 0), (int64_t)p.max_pages * kPage);
  if (p.cu == nullptr) {
    s.q0 = b;
    s.n = 1;
  } else {
    s.q0 = min(max(p.cu[b], 0), p.T);
    s.n = min(max(p.cu[b + 1], s.q0), p.T) - s.q0;
  }
  return s;
}

// 128 rows of a sequence from row0 on, and the key tiles [t0, t1) of them.
struct Piece {
  int b, q0, n, len, row0, t0, t1;
};

struct Lds {
  unsigned keys, rope, prob;   // addresses
  DMLA_LDS float* stat;        // [kRows]: sums
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
  // Address of a key tile; tiles come in ascending order.  A bad page reads page 0 instead.
  __device__ __forceinline__ const char* tile(const ChunkParams& p, const Piece& pc, int t) {
    if (t / 2 - first >= 64) fetch(p, pc, first + 64);
    int page = __builtin_amdgcn_readlane(pages, uniform((t / 2 - first) & 63));
    if (page < 0 || page >= p.num_pages) {
      bad = min(bad, t / 2);
      page = 0;
    }
    return p.kv + page * p.kv_sp + (t & 1) * kTile * p.kv_ss;
  }
};

__device__ __forceinline__ void run_piece(const ChunkParams& p, const Piece& pc, const Lds& lds) {
  const int lane = fresh_lane_id();
  const int l32 = lane & 31, hl = lane >> 5;
  const int wave = uniform(threadIdx.x >> 6);
  const int rows = min(pc.n * p.H - pc.row0, kRows);
  // Rows past the last one are the last one again, and not written.
  auto token_of = [&](int r) { return fast_div(pc.row0 + min(r, rows - 1), p.hdiv); };
  auto limit_of = [&](int r) { return p.causal ? pc.len - pc.n + token_of(r) : pc.len - 1; };   // last key
  const int lim = limit_of(32 * wave + l32);
  const int lim0 = uniform(limit_of(32 * wave));   // the wave's smallest

  // ---- copies: lane l copies 16 bytes into place l of each kilobyte ----
  Pages pages;
  auto copy_tile = [&](int s) {
    const int t = pc.t0 + s;
    const char* src = pages.tile(p, pc, t);
    // Rows past the sequence's end are its last row again.
    const int last = uniform(min(pc.len - t * kTile, kTile) - 1);
    const unsigned dst = lds.keys + (s % kSlots) * kKeyBytes + wave * 8 * kKeyRow;
    const int ln = fresh_lane_id();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      dma16(src + min(8 * wave + i, last) * p.kv_ss, 16 * (ln ^ key_swz(8 * wave + i)), dst + i * kKeyRow);
    const unsigned off = min(8 * wave + (ln >> 3), last) * (unsigned)p.kv_ss + 2 * kDv + 16 * ((ln & 7) ^ (ln >> 3));
    dma16(src, off, lds.rope + (s % kSlots) * kRopeBytes + wave * 1024);
  };

  // ---- queries: 36 operands of 16 dims; operand c holds dims 16 c + 8 hl .. of row l32 ----
  bf16x8 q[kSteps];
  {
    const unsigned mine = lds.keys + wave * kQueryBytes;   // the ropes' memory follows the keys'
    const int ln = fresh_lane_id();
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = pc.row0 + min(32 * wave + 8 * g + (ln >> 3), rows - 1);
      const int token = fast_div(r, p.hdiv), head = r - token * p.H;
      const bf16* src = p.q + (pc.q0 + token) * p.q_st + head * p.q_sh + 8 * ((ln & 7) ^ (ln >> 3));
#pragma unroll
      for (int i = 0; i < 9; ++i) dma16_addr(src + 64 * i, mine + (9 * g + i) * 1024);
    }
    wait_vm<0>();
    const unsigned a = lds_sum(9 * 1024 * (l32 >> 3) + 128 * (l32 & 7) + 16 * (hl ^ (l32 & 7)), mine);
#pragma unroll
    for (int c = 0; c < kSteps; ++c) q[c] = *lds_ptr<const bf16x8>((a ^ (32 * (c & 3))) + 1024 * (c >> 2));
    wait_lds();
    __syncthreads();   // the keys' memory is free
  }

  f32x16 acc[kRowBlocks][kColBlocks];   // O^T: register i is column 128 wave + 32 j + 16 hl + i of row l32
  float mref = kNegInf, mtrue = kNegInf, lsum = 0.f;   // reference, largest score seen, sum

  for (bool again = false;; again = true) {
#pragma unroll
    for (int n = 0; n < kRowBlocks; ++n)
#pragma unroll
      for (int j = 0; j < kColBlocks; ++j) acc[n][j] = mfma32_bf16(bf16x8{}, bf16x8{}, f32x16{});
    lsum = 0.f;
    if (pc.t0 < pc.t1) pages.fetch(p, pc, pc.t0 / 2);
#pragma nounroll
    for (int s = 0; s < pc.t1 - pc.t0; ++s) {
      const int t = pc.t0 + s;
      copy_tile(s);
      wait_vm<0>();
      __syncthreads();
      // scores: S^T[key 8 (i / 4) + 4 hl + i % 4][row l32]
      f32x16 x;
      const unsigned rope = lds_sum(128 * l32 + 16 * (hl ^ (l32 & 7)), lds.rope + (s % kSlots) * kRopeBytes);
      const unsigned key = lds_sum(kKeyRow * l32 + 16 * (hl ^ key_swz(l32)), lds.keys + (s % kSlots) * kKeyBytes);
      static_for<kSteps>([&](auto m_tag) {
        constexpr int m = decltype(m_tag)::value, c = m - 4;
        const bf16x8 k = *lds_ptr<const bf16x8>(m < 4 ? rope ^ (32 * m) : (key ^ (32 * (c & 7))) + 256 * (c >> 3));
        score_step<m == 0>(x, k, q[m < 4 ? kLatSteps + m : c]);
      });
      score_done(x);
      if (t * kTile + kTile - 1 > lim0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = t * kTile + 8 * (i >> 2) + 4 * hl + (i & 3) <= lim ? x[i] : kNegInf;
      }
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
      mx = half_max(mx) * p.scale_log2;   // scale > 0
      if (s == 0) mref = again ? mtrue : mx;
      mtrue = fmaxf(mtrue, mx);
      const float ms = mref == kNegInf ? 0.f : mref;
      bf16x8 pv[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float v = fast_exp2(__builtin_fmaf(x[e], p.scale_log2, -ms));
        lsum += v;
        pv[e >> 3][e & 7] = (bf16)v;
      }
      const unsigned at = lds_sum(16 * lane, lds.prob + wave * 2048);
#pragma unroll
      for (int u = 0; u < 2; ++u) *lds_ptr<bf16x8>(at + 1024 * u) = pv[u];
      __syncthreads();
      // values: groups of 16 keys (u) and 32 columns (j).  Row m of the operand is column
      // 4 (m / 8) + 16 (m / 4 % 2) + m % 4 of the block: a lane then ends with 16 neighbouring columns.
      const int r = (lane & 15) >> 2, g = lane >> 4 & 1;
      const unsigned val = lds_sum(kKeyRow * (4 * hl + r) + 256 * wave + 16 * (4 * r | ((g + 2 * (lane & 1)) ^ hl)) + 8 * ((lane & 3) >> 1),
                                   lds.keys + (s % kSlots) * kKeyBytes);
      const unsigned prob = lds_sum(16 * lane, lds.prob);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        bf16x8 pr[kRowBlocks];
#pragma unroll
        for (int n = 0; n < kRowBlocks; ++n) pr[n] = *lds_ptr<const bf16x8>(prob + 2048 * n + 1024 * u);
#pragma unroll
        for (int j = 0; j < kColBlocks; ++j) {
          const unsigned a = (val ^ (64 * j)) ;
          const bf16x8 v = concat(lds_read_tr16(lds_ptr<const bf16x4>(a + 16 * kKeyRow * u)),
                                  lds_read_tr16(lds_ptr<const bf16x4>((a ^ 32) + 16 * kKeyRow * u + 8 * kKeyRow)));
#pragma unroll
          for (int n = 0; n < kRowBlocks; ++n) acc[n][j] = mfma32_bf16(v, pr[n], acc[n][j]);
        }
      }
      __syncthreads();   // keys and probabilities are read
    }
    const bool over = __any(mtrue > mref + kHeadroom);
    if (lane == 0) lds.flag[wave] = over ? 1 : 0;
    __syncthreads();
    const bool repeat = (lds.flag[0] | lds.flag[1] | lds.flag[2] | lds.flag[3]) != 0;
    __syncthreads();
    if (again || !repeat) break;
  }

  // ---- output ----
  lsum = half_sum(lsum);
  agpr_settle();
  if (hl == 0) lds.stat[wave * 32 + l32] = lim >= pages.bad * (int64_t)kPage ? __builtin_nanf("") : lsum;
  __syncthreads();
  if (hl == 0 && 32 * wave + l32 < rows && p.lse != nullptr) {
    const int r = pc.row0 + 32 * wave + l32;
    const int token = fast_div(r, p.hdiv), head = r - token * p.H;
    const float sum = lds.stat[32 * wave + l32];
    p.lse[(int64_t)(pc.q0 + token) * p.H + head] = sum == 0.f ? kNegInf : (mref + __log2f(sum)) * kLn2;
  }
  // Through LDS, 32 rows at a time, so that a store covers whole lines: 256 bytes of each of 4 rows.  16-byte unit u
  // of row r lies at u ^ r.
  const unsigned mine = lds.keys + wave * 16 * 1024;
  const int g = lane >> 4, c = lane & 15;
  const unsigned put = lds_sum(512 * l32 + 16 * ((4 * hl) ^ l32), mine);
  const unsigned get = lds_sum(512 * g + 16 * ((2 * c) ^ g), mine);   // 8 columns of row g: this unit and the one beside it
#pragma unroll
  for (int n = 0; n < kRowBlocks; ++n) {
    const float sum = lds.stat[32 * n + l32];
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
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const int row = 32 * n + 4 * r + g;
      const f32x4 a = *lds_ptr<const f32x4>((get ^ (64 * r)) + 2048 * r), b = *lds_ptr<const f32x4>((get ^ (64 * r) ^ 16) + 2048 * r);
      if (row < rows) {
        const int token = fast_div(pc.row0 + row, p.hdiv), head = pc.row0 + row - token * p.H;
        bf16x8 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = (bf16)a[i];
          v[4 + i] = (bf16)b[i];
        }
        *reinterpret_cast<bf16x8*>(p.o + (pc.q0 + token) * p.o_st + head * p.o_sh + 128 * wave + 8 * c) = v;
      }
    }
  }
}

// One workgroup per 128 rows; those past the last clear the queries that no sequence has.
__global__ __launch_bounds__(kThreads, 1) void chunk_kernel(ChunkParams p) {
  __shared__ __attribute__((aligned(1024))) char mem[kSlots * (kKeyBytes + kRopeBytes) + kProbBytes];
  __shared__ __attribute__((aligned(16))) float stat[kRows];
  __shared__ __attribute__((aligned(16))) int flag[kWaves];
  __shared__ int found[4];
  const unsigned base = lds_addr((DMLA_LDS char*)mem);
  const Lds lds = {base, base + kSlots * kKeyBytes, base + kSlots * (kKeyBytes + kRopeBytes), (DMLA_LDS float*)stat,
                   (DMLA_LDS int*)flag};
  // The piece's sequence, by one wave.
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int64_t before = 0;
    int b = -1, row0 = 0;
    for (int b0 = 0; b0 < p.B && b < 0; b0 += 64) {
      const int64_t mine = b0 + lane < p.B ? ((int64_t)sequence(p, b0 + lane).n * p.H + kRows - 1) / kRows : 0;
      int64_t x = mine;
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
      }
      const unsigned long long past = __ballot(before + x > (int64_t)blockIdx.x);
      if (past != 0) {
        const int i = __builtin_ctzll(past);
        b = b0 + i;
        row0 = (int)((int64_t)blockIdx.x - before - __shfl(x - mine, i, 64)) * kRows;
      }
      before += __shfl(x, 63, 64);
    }
    if (lane == 0) {
      found[0] = b;
      found[1] = row0;
    }
  }
  __syncthreads();
  Piece pc;
  pc.b = uniform(found[0]);
  if (pc.b < 0) return;
  const Sequence s = sequence(p, pc.b);
  pc.q0 = uniform(s.q0);
  pc.n = uniform(s.n);
  pc.len = uniform(s.len);
  pc.row0 = uniform(found[1]);
  const int last = fast_div(min(pc.row0 + kRows, pc.n * p.H) - 1, p.hdiv);
  const int end = p.causal ? pc.len - pc.n + last + 1 : pc.len;   // keys of the last row
  pc.t0 = 0;
  pc.t1 = uniform((max(end, 0) + kTile - 1) / kTile);
  run_piece(p, pc, lds);
}

// Queries behind the last sequence: zeros, and -inf.
__global__ __launch_bounds__(256) void chunk_tail_kernel(ChunkParams p) {
  const int first = p.cu == nullptr ? p.B : min(max(p.cu[p.B], 0), p.T);
  const int64_t total = (int64_t)(p.T - first) * p.H * (kDv / 8);
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
    const int64_t row = u / (kDv / 8);
    const int c = (int)(u % (kDv / 8)), token = first + (int)(row / p.H), head = (int)(row % p.H);
    *reinterpret_cast<bf16x8*>(p.o + token * p.o_st + head * p.o_sh + 8 * c) = bf16x8{};
    if (c == 0 && p.lse != nullptr) p.lse[(int64_t)token * p.H + head] = kNegInf;
  }
}

}  // namespace
}  // namespace dmla

using namespace dmla;

extern "C" int64_t dmla_chunk_paged_workspace_bytes(int64_t T, int64_t B, int64_t H, int64_t max_pages_per_seq) {
  (void)T; (void)B; (void)H; (void)max_pages_per_seq;
  return 0;
}

extern "C" int dmla_chunk_paged(const void* q, const void* kv_pool, const int32_t* block_table, const int32_t* cache_seqlens,
                                const int32_t* cu_seqlens_q, void* o, float* lse, int64_t T, int64_t B, int64_t H,
                                int64_t d_qk, int64_t d_v, int64_t num_pages, int64_t max_pages_per_seq, int64_t q_st,
                                int64_t q_sh, int64_t kv_sp, int64_t kv_ss, int64_t bt_sb, int64_t o_st, int64_t o_sh,
                                float softmax_scale, int causal, void* workspace, int64_t workspace_bytes,
                                dmla_stream_t stream) {
  clear_error();
  const char* what = "dmla_chunk_paged";
  (void)workspace; (void)workspace_bytes;
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
      max_pages_per_seq > ((int64_t)1 << 24) || num_pages > 0x7fffffff)
    return fail(DMLA_ERR_UNSUPPORTED, "%s: size too large", what);
  if (T == 0 || H == 0) return DMLA_OK;
  if (!q || !o || (B > 0 && !cache_seqlens) || (B > 0 && max_pages_per_seq > 0 && !block_table) || (num_pages > 0 && !kv_pool))
    return fail(DMLA_ERR_INVALID_ARG, "%s: null pointer argument", what);
  if (B > 0 && (num_pages == 0 || max_pages_per_seq == 0))
    return fail(DMLA_ERR_INVALID_ARG, "%s: empty page pool or block table", what);
  ChunkParams p = {};
  p.q = static_cast<const bf16*>(q);
  p.kv = static_cast<const char*>(kv_pool);
  p.block_table = block_table;
  p.seqlens = cache_seqlens;
  p.cu = cu_seqlens_q;
  p.o = static_cast<bf16*>(o);
  p.lse = lse;
  p.q_st = q_st; p.q_sh = q_sh; p.kv_sp = 2 * kv_sp; p.kv_ss = 2 * kv_ss; p.bt_sb = bt_sb; p.o_st = o_st; p.o_sh = o_sh;
  p.T = (int)T; p.B = (int)B; p.H = (int)H; p.num_pages = (int)num_pages; p.max_pages = (int)max_pages_per_seq;
  p.causal = causal ? 1 : 0;
  p.hdiv = make_fastdiv((unsigned)H);
  p.scale_log2 = softmax_scale * kLog2e;
  const int64_t tiles = cu_seqlens_q == nullptr ? T * ((H + kRows - 1) / kRows) : T * H / kRows + std::min(B, T);
  if (tiles > 0)
    hipLaunchKernelGGL(chunk_kernel, dim3((unsigned)tiles), dim3(kThreads), 0, (hipStream_t)stream, p);
  if (cu_seqlens_q != nullptr)
    hipLaunchKernelGGL(chunk_tail_kernel, dim3(256), dim3(256), 0, (hipStream_t)stream, p);
  return check_launch(what);
}
