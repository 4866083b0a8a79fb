// A cache in 8 bits: e4m3 values (four significant bits, up to 448, steps of 2^-9 below 2^-6; no infinity) and, for each
// block of 16 tokens and head, a power of two as its biased exponent (2^(byte - 127)).
//
// A power of two costs an e4m3 value no precision, and a value times its scale is a bfloat16 number: bytes 10 to
// 246, scales of 2^-117 to 2^119, keep it between bfloat16's ends (2^-126 and 448 * 2^119). So what the cache stands
// for is read as bfloat16 exactly, and a block whose scale grows is brought to the new one by a shift of exponents
// (only what falls below 2^-6 of the new scale is rounded again). A block with a scale beyond
// those ends, of a cache that was quantised elsewhere, is read as bfloat16 rounds it, and an append that goes on with it brings
// its older tokens to a scale within them.
#pragma once
#include "pp_common.h"

#define FP8_BLOCK 16  // tokens of a block
#define FP8_LOW 10    // least and largest byte of a scale that an append writes
#define FP8_HIGH 246
#define FP8_TOP 0x7f600000u  // bits of 448 * 2^119

typedef __bf16 fp8_bf16x2 __attribute__((ext_vector_type(2)));
typedef float fp8_f32x2 __attribute__((ext_vector_type(2)));

// Least scale whose 448-fold holds a magnitude (its bits), as a byte.
__device__ __forceinline__ int fp8_scale(uint32_t top) { return min(max((int)((top + 0x1fffffu) >> 23) - 8, FP8_LOW), FP8_HIGH); }
// 2^(127 - byte): what values are multiplied by (byte within its range)
__device__ __forceinline__ float fp8_inverse(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float fp8_factor(uint32_t byte) { return __uint_as_float(byte << 23); }
// Bits 7, 15, 23 and 31 of a word: whether its values are NaN.
__device__ __forceinline__ uint32_t fp8_bad(uint32_t word) { return (word & 0x7f7f7f7fu) + 0x01010101u; }
// Four values, at most 448 or NaN, as a word.
__device__ __forceinline__ uint32_t fp8_pack(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// Two values of a word times a scale, as a pair of bfloat16.
template <bool HIGH>
__device__ __forceinline__ uint32_t fp8_bf16(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, HIGH));
}
// What brings values of the scale `held`, any byte, to that of `byte`, one of an append's: 255 is no number.
__device__ __forceinline__ float fp8_step(int held, int byte) {
  return __uint_as_float(held == 255 ? 0x7fc00000u : held - byte < -126 ? 0u : (uint32_t)(127 + held - byte) << 23);
}
// A word's values times f, rounded again. Where f is above 1 (a block whose scale was beyond FP8_HIGH) what bfloat16 still has room
// for is at most 448, the rest NaN.
__device__ __forceinline__ float fp8_held(float x) { return fabsf(x) < 512.0f ? fminf(fmaxf(x, -448.0f), 448.0f) : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ uint32_t fp8_rescale(uint32_t word, float f) {
  const fp8_f32x2 x = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, false), y = __builtin_amdgcn_cvt_pk_f32_fp8((int)word, true);
  return fp8_pack(fp8_held(x[0] * f), fp8_held(x[1] * f), fp8_held(y[0] * f), fp8_held(y[1] * f));
}
// x * inv as the cache takes it: beyond 448 (only where the scale is the largest) 448, NaN for what is not finite.
__device__ __forceinline__ float fp8_odd(float x, float inv) {
  if (!(fabsf(x) < __builtin_inff())) return __uint_as_float(0x7fc00000u);
  return fminf(fmaxf(x * inv, -448.0f), 448.0f);
}
