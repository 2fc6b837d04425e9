// The 16-bit matrix instruction of the attention and adapter kernels, and what its operands and results are made of:
// v_mfma_f32_16x16x32 with bf16 or fp16 operands and fp32 sums. Lane l gives row (column) l & 15 and the 8 terms from 8 (l / 16) of
// its operand, and holds rows 4 (l / 16) + v, v = 0 .. 3, of column l & 15 of the result.
#pragma once
#include "gpic_device.h"

namespace gpic {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8v __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));

constexpr float kInf = __builtin_huge_valf();

template <bool F16>
__device__ __forceinline__ f32x4_t mfma16(s16x8 a, s16x8 b, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8v, a), __builtin_bit_cast(f16x8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (F16) return __builtin_bit_cast(uint32_t, f16x2v{(_Float16)lo, (_Float16)hi});
  else return pack_bf16(lo, hi);
}
template <bool F16>
__device__ __forceinline__ void floats8(s16x8 x, float (&f)[8]) {
  if constexpr (F16) {
    const f16x8v h = __builtin_bit_cast(f16x8v, x);
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = (float)h[e];
  } else {
    const u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int e = 0; e < 8; e++) f[e] = e & 1 ? bf16_hi(w[e >> 1]) : bf16_lo(w[e >> 1]);
  }
}
// The two values of a word.
template <bool F16>
__device__ __forceinline__ float low16(uint32_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(f16x2v, w)[0];
  else return bf16_lo(w);
}
template <bool F16>
__device__ __forceinline__ float high16(uint32_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(f16x2v, w)[1];
  else return bf16_hi(w);
}
// Rounded to the type and back.
template <bool F16>
__device__ __forceinline__ float round16(float f) {
  if constexpr (F16) return (float)(_Float16)f;
  else return bf16_round(f);
}

__device__ __forceinline__ uint32_t lds_at(const void *p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p;
}
// Sixteen bytes a lane from its own address to LDS [lds, lds + 1 KiB) in lane order, past the registers. The loads are counted in
// vmcnt but not by the compiler, so staged() comes before the reads of what they bring, or the barrier that hands it on.
__device__ __forceinline__ void to_lds(const void *src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(lds) : "memory", "m0");
}
// (with loads of later tiles behind them that may stay in flight)
template <int kInFlight>
__device__ __forceinline__ void staged_but() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kInFlight) : "memory");
}
__device__ __forceinline__ void staged() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Rows of a staged tile: 16-byte chunk c of row r lies in place c ^ swz(r).
// A read by rows takes 16 lanes at a time, those of one group with rows 0-3 and 12-15 and those of the next with rows 4-11: the
// values for the former are pairs (x, x ^ 1), so that the latter's, one chunk on, are the other pairs. A read by columns takes 8
// rows: the values of each half are of different pairs.
template <int DP>
__device__ __forceinline__ int swz(int r) {
  const int u = DP == 64 ? r >> 1 & 7 : r & 15, half = DP == 64 ? 4 : 8, high = u / half;
  return ((u + high * half / 2) & (half - 1)) << 1 | high;
}

// Sixteen zero bytes, for the lanes of a staged tile that have none of their own.
__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

}  // namespace gpic
