// csrc/dmla_chunk_cut.h on the CPU, a thread for each lane of a workgroup (see test_chunk_cut.py): barriers are barriers
// of all threads, ballots and scans those of a wave's 64.
#include <pthread.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
#define DMLA_LDS
#define DMLA_GLOBAL

typedef int i32x4 __attribute__((vector_size(16)));
typedef unsigned u32x4 __attribute__((vector_size(16)));
typedef uint16_t bf16;
using std::max;
using std::min;

namespace {

thread_local struct {
  int x;
} threadIdx;
pthread_barrier_t all_threads, wave_lanes[4];
int word[256];   // what the lanes of a wave show each other

void __syncthreads() { pthread_barrier_wait(&all_threads); }
// This wave's words, one of each lane, as f sees them.
template <typename F>
auto with_wave(int mine, F f) {
  const int wave = threadIdx.x / 64;
  word[threadIdx.x] = mine;
  pthread_barrier_wait(&wave_lanes[wave]);
  const auto r = f(word + 64 * wave);
  pthread_barrier_wait(&wave_lanes[wave]);
  return r;
}
int fresh_lane_id() { return threadIdx.x & 63; }
int uniform(int v) { return v; }
int lane_scan(int v) {
  return with_wave(v, [](const int* w) {
    unsigned s = 0;   // (as a GPU adds: past 32 bits it wraps)
    for (int i = 0; i <= (threadIdx.x & 63); ++i) s += (unsigned)w[i];
    return (int)s;
  });
}
unsigned long long __ballot(bool v) {
  return with_wave(v, [](const int* w) {
    unsigned long long m = 0;
    for (int i = 0; i < 64; ++i) m |= (unsigned long long)(w[i] != 0) << i;
    return m;
  });
}
bool __any(bool v) { return __ballot(v) != 0; }
struct FastDiv {
  int d;
};
int fast_div(int n, FastDiv d) { return n / d.d; }

}  // namespace

#include "dmla_chunk_cut.h"

using namespace dmla;

namespace {

// f on 256 threads that live as long as the process.
std::function<void()> job;
void on_a_workgroup(std::function<void()> f) {
  static std::vector<std::thread> threads;
  static pthread_barrier_t start, end;
  if (threads.empty()) {
    pthread_barrier_init(&all_threads, nullptr, kThreads);
    for (auto& w : wave_lanes) pthread_barrier_init(&w, nullptr, 64);
    pthread_barrier_init(&start, nullptr, kThreads + 1);
    pthread_barrier_init(&end, nullptr, kThreads + 1);
    for (int i = 0; i < kThreads; ++i) {
      threads.emplace_back([i] {
        threadIdx.x = i;
        for (;;) {
          pthread_barrier_wait(&start);
          job();
          pthread_barrier_wait(&end);
        }
      });
      threads.back().detach();
    }
  }
  job = f;
  pthread_barrier_wait(&start);
  pthread_barrier_wait(&end);
}

std::vector<int> numbers(int n) {
  std::vector<int> v(n);
  for (int& x : v)
    if (std::scanf("%d", &x) != 1) std::exit(1);
  return v;
}

}  // namespace

int main() {
  char what[16];
  while (std::scanf("%15s", what) == 1) {
    ChunkParams p = {};
    if (!std::strcmp(what, "cut")) {   // T B H max_pages causal n_ranges packed, the ranges wanted, lengths, starts
      const std::vector<int> a = numbers(8);
      const std::vector<int> ranges = numbers(a[7]), lens = numbers(a[1]), cu = numbers(a[6] ? a[1] + 1 : 0);
      p.T = a[0]; p.B = a[1]; p.H = a[2]; p.max_pages = a[3]; p.causal = a[4]; p.n_ranges = a[5];
      p.seqlens = lens.data();
      p.cu = a[6] ? cu.data() : nullptr;
      p.hdiv = FastDiv{p.H};
      p.two_by_h = 2.0f / (float)p.H;
      p.weight_shift = chunk_weight_shift(p.T, p.B, p.H, p.max_pages);
      p.weight_scale = std::ldexp(1.0f, -p.weight_shift);
      std::vector<i32x4> links(p.n_ranges);
      p.links = links.data();
      for (int range : ranges) {
        static Window window;
        on_a_workgroup([&] {   // what chunk_kernel does around its pieces
          if (!cut(p, &window, range)) return;
          i32x4* pieces = &window.piece[0][0];
          next_piece(p, &window, pieces, range);
          for (int turn = 0;; turn ^= 1) {
            i32x4* now = pieces + 3 * turn;
            i32x4* other = pieces + 3 * (turn ^ 1);
            __syncthreads();
            const i32x4 q = now[0], k = now[1];
            if (q[2] == 0) break;
            next_piece(p, &window, other, range);
            if (threadIdx.x == 0)   // range, sequence, first row, rows, tokens, key tiles, slot
              std::printf("%d %d %d %d %d %d %d %d ", range, k[1], q[1], q[2], k[0], k[2], k[3], now[2][0]);
            __syncthreads();
          }
        });
      }
      std::printf("\n");
    } else if (!std::strcmp(what, "weight")) {   // T B H max_pages causal, lengths, starts
      const std::vector<int> a = numbers(5);
      const std::vector<int> lens = numbers(a[1]), cu = numbers(a[1] + 1);
      p.T = a[0]; p.B = a[1]; p.H = a[2]; p.max_pages = a[3]; p.causal = a[4];
      p.seqlens = lens.data();
      p.cu = cu.data();
      p.two_by_h = 2.0f / (float)p.H;
      p.weight_shift = chunk_weight_shift(p.T, p.B, p.H, p.max_pages);
      p.weight_scale = std::ldexp(1.0f, -p.weight_shift);
      int64_t sum = 0;
      bool ascending = true;
      for (int b = 0; b < p.B; ++b) {
        const Sequence s = sequence(p, b);
        const Weights w = weights(p, s, kRowsLog2);
        const int n = row_tiles(p, s, kRowsLog2);
        sum += weight(p, w, n);
        for (int i = 0, before = 0; i < 64; ++i) {
          const int v = weight(p, w, (int)((int64_t)n * (i + 1) / 64));
          ascending = ascending && v >= before;
          before = v;
        }
      }
      std::printf("%lld %d %d\n", (long long)sum, p.weight_shift, ascending ? 1 : 0);
    } else if (!std::strcmp(what, "careful")) {   // pages of the pool, causal tokens: from, last limit, end tile; odd tokens; table
      const std::vector<int> a = numbers(6);
      const std::vector<int> odd = numbers(a[4]), table = numbers(a[5]);
      p.num_pages = a[0];
      p.kv_ss = 1152;
      p.kv_sp = 64 * p.kv_ss;
      std::vector<char> pool(p.num_pages * p.kv_sp + 16);
      char* base = pool.data() + (-reinterpret_cast<uintptr_t>(pool.data()) & 15);
      for (int at : odd) {   // page * 64 + row; an infinity in one of its latents
        const uint16_t inf = 0x7f80;
        std::memcpy(base + at / 64 * p.kv_sp + at % 64 * p.kv_ss + 2 * (at % 512), &inf, 2);
      }
      p.kv = base;
      p.block_table = table.data();
      Piece pc = {};
      pc.t1 = a[3];
      static int flag[kWaves];
      Pass pass = {};
      on_a_workgroup([&] {
        // As a pass ends: each wave posts a word, all read the four.
        if (fresh_lane_id() == 0) flag[threadIdx.x / 64] = threadIdx.x < 64;
        __syncthreads();
        const bool again = (flag[0] | flag[1] | flag[2] | flag[3]) != 0;
        Pass r = {};
        if (again) r = careful_pass(p, pc, flag, a[1], a[2]);
        if (threadIdx.x == 0) pass = r;
      });
      std::printf("%d %d %d\n", pass.careful ? 1 : 0, pass.from, pass.to);
    } else {
      return 1;
    }
  }
  std::fflush(stdout);
  _Exit(0);
}
