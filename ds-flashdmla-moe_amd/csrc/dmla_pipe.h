// Pieces of tile loops whose order is written by hand, and of kernels whose accumulators fill the AGPR file.
#pragma once
#include <type_traits>

#include "dmla_common.h"

namespace dmla {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// f(0), f(1), .., f(kN - 1) with compile-time arguments.
template <int kN, typename F, int kI = 0>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (kI < kN) {
    f(std::integral_constant<int, kI>{});
    static_for<kN, F, kI + 1>(f);
  }
}

// Nothing moves across: the order of a pipelined loop body is the source's.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

// Address lane_off + add as one register that the compiler does not see into: it would keep an address per
// read up to date in a loop otherwise.
__device__ __forceinline__ unsigned lds_sum(int lane_off, unsigned add) {
  unsigned a;
  asm("v_add_u32 %0, %1, %2" : "=v"(a) : "v"(lane_off), "s"(add));
  return a;
}
template <typename T>
__device__ __forceinline__ DMLA_LDS T* lds_ptr(unsigned addr) {
  return reinterpret_cast<DMLA_LDS T*>(static_cast<uintptr_t>(addr));
}

// Wait until at most N vector-memory (LDS) operations of this wave are outstanding; they end in order, and no
// memory access moves across.
template <int N>
__device__ __forceinline__ void wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
  asm volatile("" ::: "memory");
}
template <int N = 0>
__device__ __forceinline__ void wait_lds() {
  static_assert(N >= 0 && N < 16, "lgkmcnt field");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f | (N << 8));
  asm volatile("" ::: "memory");
}

// The output accumulators fill the AGPR file.  Where ordinary code touches them, the compiler gives them a
// home among the VGPRs as well and spills the queries; these accesses leave them where they are.  The
// compiler does not see into the assembly, so agpr_settle() keeps them clear of MFMAs on the same register.
__device__ __forceinline__ float agpr_read(float x) {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(x));
  return v;
}
// Longer than any MFMA takes to write its result, or a write to reach one.
__device__ __forceinline__ void agpr_settle() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }

// One step of the score product, x += k q (x = k q for the first of a tile).  In assembly because the
// AGPRs have no room for x beside the accumulators and the compiler gives every MFMA of a kernel the same
// register file.  It does not see the waits that such an operand needs.  An operand written by the vector ALU
// has to be two instructions old.  (An s_nop in every step would cost half an MFMA: 24.0 against 18.4 ns for
// an MFMA with four conversions beside it, 15.4 alone.)  Steps on the same x follow each other without a
// wait.  score_done() stands between the last and the first read.
template <bool kFirst>
__device__ __forceinline__ void score_step(f32x16& x, const bf16x8& k, const bf16x8& q) {
  if constexpr (kFirst) asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(x) : "v"(k), "v"(q));
  else asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(x) : "v"(k), "v"(q));
}
__device__ __forceinline__ void score_done(f32x16& x) { asm("s_nop 15\n\ts_nop 7" : "+v"(x)); }

}  // namespace dmla
