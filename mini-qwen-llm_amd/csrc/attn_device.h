// Device-side pieces that the attention kernels share: element types with their 32 x 32
// MFMAs, the order of a staged tile's 16-byte chunks, and direct loads from a uniform base.
#pragma once

#include "mqk_device.h"

namespace mqk {
namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// 16 bytes of zeros: what the columns past a head size that is no whole tile are read from.
__device__ const u32x4_t g_zero16 = {0, 0, 0, 0};

struct AttnBf16 : Bf16 {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kExp = 0x7F80u;
  static constexpr float kLift = 0.f;  // (powers of 2 that a weight is rounded above its value)
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) { return mfma_32x32x16(a, b, c); }
};
struct AttnFp16 : Fp16 {
  static constexpr int kBytes = 2;
  static constexpr uint32_t kExp = 0x7C00u;
  static constexpr float kLift = 7.f;  // (normal numbers end at 2^-14; the largest is just below 2^16)
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
    typedef _Float16 f16x8_v __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_v, a), __builtin_bit_cast(f16x8_v, b), c, 0,
                                                  0, 0);
  }
};
struct AttnF32 {
  static constexpr int kBytes = 4;
  static constexpr uint32_t kExp = 0x7F800000u;
  // four k-steps of 2: slot h of step e is element e of half h's four
  static __device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b, f32x16_t c) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
    return c;
  }
};

// Where chunk c (16 bytes) of row r lies in a staged row of C chunks.  K rows are read a
// chunk column at a time (32 rows, one chunk): 16 neighbouring rows take 16 different bank
// groups.  V rows are read 4 at a time, 4 neighbouring chunks each (16-bit types), or one
// row by each half of the wave, 4 rows apart (fp32).
template <int C>
__device__ __forceinline__ int k_slot(int r, int c) {
  return C >= 16 ? (c ^ (r & 15)) : (c ^ ((r >> 1) & 7));
}
template <int C, int BYTES>
__device__ __forceinline__ int v_slot(int r, int c) {
  if (BYTES == 4) return c ^ (((r >> 2) & 1) << 3);
  return C >= 16 ? (c ^ ((r & 3) << 2)) : (c ^ (((r >> 1) & 1) << 2));
}

__device__ __forceinline__ float max_halves(float x) {  // over lanes l and l + 32, to both
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// First token and length of sequence s: offsets in device memory, clamped into the tensor,
// or equal lengths.
__device__ __forceinline__ int64_t seq_at(const int32_t* cu, int64_t each, int64_t total, int s) {
  const int64_t at = cu ? int64_t(cu[s]) : each * s;
  return at < 0 ? 0 : at > total ? total : at;
}

// L2 -> LDS as dma16, from a wave-uniform base plus a 32-bit offset of the lane.  The load may
// read M0 one wait state after it is written, and its base five after a vector instruction
// wrote that (v_readlane, where the compiler keeps the base in a vector register), of which
// the compiler sees to none inside the asm.
__device__ __forceinline__ void dma16_from(const unsigned char* base, uint32_t off, uint32_t lds_base) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 2\n\t"
      "global_load_lds_dwordx4 %2, %3\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(off), "s"(base)
      : "memory");
}

// Four of them, STEP bytes of LDS apart: M0 is saved once, and has its wait state before each.
template <int STEP>
__device__ __forceinline__ void dma16x4_from(const unsigned char* b0, const unsigned char* b1, const unsigned char* b2,
                                             const unsigned char* b3, uint32_t o0, uint32_t o1, uint32_t o2, uint32_t o3,
                                             uint32_t lds_base) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 2\n\t"
      "global_load_lds_dwordx4 %2, %6\n\t"
      "s_add_u32 m0, m0, %10\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %3, %7\n\t"
      "s_add_u32 m0, m0, %10\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %4, %8\n\t"
      "s_add_u32 m0, m0, %10\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %5, %9\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(__builtin_amdgcn_readfirstlane(lds_base)), "v"(o0), "v"(o1), "v"(o2), "v"(o3), "s"(b0), "s"(b1), "s"(b2),
        "s"(b3), "n"(STEP)
      : "memory", "scc");
}

}  // namespace
}  // namespace mqk
