// The 4-bit latent cache row, shared by the kernels that write and read it.
//
// A row holds the 576 values of one token in 400 bytes (25 pieces of 16 bytes):
//   bytes 0..255    e2m1 codes of the 512 latent values, value 2i in the low half of byte i
//   bytes 256..271  one scale byte per block of 32 values: 2^(byte - 127); 255 means not a number
//   bytes 272..399  the 64 rope values in bf16, as they came
// A code is sign (bit 3) and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A block's scale is the least power of
// two with which none of its values exceeds 6, between 2^-125 and 2^125 (values past 6 x 2^125 are
// held as that), so code x scale is exact in bf16 and reading a row back rounds nothing.  The rope
// values carry the position and stay in bf16.  A block that holds an infinity or a NaN is all NaN.
#pragma once
#include <type_traits>

#include "dmla_common.h"

namespace dmla {

constexpr int kQ4RowBytes = 400;
constexpr int kQ4ScaleOff = 256;
constexpr int kQ4RopeOff = 272;
constexpr int kQ4Chunks = kQ4RowBytes / 16;   // 16-byte pieces of a row
constexpr int kQ4MinExp = -125, kQ4MaxExp = 125;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// The scale byte of a block whose largest |value| has the fp32 bits `top` (a bf16 value).  With
// top = m 2^k, 1 <= m < 2: top <= 6 2^e = 1.5 2^(e + 2) needs e = k - 2 for m <= 1.5, else k - 1.
__device__ __forceinline__ int q4_scale_byte(unsigned top) {
  const int k = (int)(top >> 23) - 127;   // zero and subnormals: below the least scale
  const int e = k - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
  return top >= 0x7f800000u ? 255 : min(max(e, kQ4MinExp), kQ4MaxExp) + 127;
}

// The float whose value a scale byte stands for.  Of byte 255 it is an infinity, which the code
// conversions below turn into NaN for every code.
__device__ __forceinline__ float q4_scale(int byte) { return __uint_as_float((unsigned)byte << 23); }

// The same scale from byte kByte of a word of four: the conversions below take the exponent and ignore the
// sign and mantissa bits of their scale, so one shift does (byte 3 to bits 23..30, the others below it).
template <int kByte>
__device__ __forceinline__ float q4_scale_of(unsigned word) {
  return __uint_as_float(kByte == 3 ? word >> 1 : word << (23 - 8 * kByte));
}

// Values 2i and 2i + 1 of the four code bytes in w, i = kByte.
template <int kByte>
__device__ __forceinline__ bf16x2 q4_pair(unsigned w, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte);
}

// The eight values of the four code bytes in w.
__device__ __forceinline__ bf16x8 q4_octet(unsigned w, float scale) {
  const bf16x2 a = q4_pair<0>(w, scale), b = q4_pair<1>(w, scale), c = q4_pair<2>(w, scale), d = q4_pair<3>(w, scale);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// ---- key rows as an MFMA operand ----------------------------------------------------------------
// Score product of 32 keys with 32 queries: 32 bf16 MFMAs (32x32x16) of the latent dims and 4 of the rope
// dims, lane l holding key l % 32.  Which dims the two lane halves hold is free as long as the queries
// agree: in MFMA 4 a + j half h takes the dims 64 a + 32 h + 8 j + x, so a lane reads 16 bytes of codes, a
// scale block, for four MFMAs.  Rows of 400 bytes put 16 consecutive rows of such a read into 16 different
// 16-byte columns of the LDS banks.
constexpr int kQ4Steps = 36;        // MFMAs of a 32-key tile
constexpr int kQ4LatentSteps = 32;

// First dim of half h in MFMA c, in units of 8 dims.
__host__ __device__ constexpr int q4_operand_unit(int h, int c) {
  return c < kQ4LatentSteps ? 8 * (c / 4) + 4 * h + c % 4 : 2 * c + h;
}
// Codes of MFMAs 4 a .. 4 a + 3, all scales of the half (byte 2 (a % 2) of word a / 2), and rope operand c of
// this lane's row.
__device__ __forceinline__ u32x4 q4_key_codes(const DMLA_LDS char* row, int h, int a) {
  return *reinterpret_cast<const DMLA_LDS u32x4*>(row + 32 * a + 16 * h);
}
__device__ __forceinline__ u32x4 q4_key_scales(const DMLA_LDS char* row, int h) {
  return *reinterpret_cast<const DMLA_LDS u32x4*>(row + kQ4ScaleOff) >> (unsigned)(8 * h);
}
__device__ __forceinline__ bf16x8 q4_key_rope(const DMLA_LDS char* row, int h, int c) {
  return lds_read_b128(reinterpret_cast<const DMLA_LDS bf16x8*>(row + kQ4RopeOff + 32 * c + 16 * h));
}
template <int kA>
__device__ __forceinline__ float q4_key_scale(const u32x4& scales) {
  return q4_scale_of<2 * (kA % 2)>(scales[kA / 2]);
}

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

}  // namespace dmla
