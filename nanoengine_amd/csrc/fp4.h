// The 4-bit block format of the DSA caches, for gfx950.
//
// A block is 32 consecutive elements: 16 bytes of e2m1 codes (element 2i in the
// low nibble of byte i; codes 0..7 are 0, .5, 1, 1.5, 2, 3, 4, 6, bit 3 the sign)
// and one UE8M0 scale byte. value = code * 2^(byte - 127); byte 255 makes the
// whole block NaN. Up to byte 252, the largest that the writers store, every value is a
// bf16 value (two significant bits times a power of two, subnormal ones
// included); at bytes 253 and 254 the codes from 4 and from 2 on are 2^128 and
// more, which bf16 holds as infinities.
//   MLA row (400 B)     : [256 B codes of 512 dims][16 scale bytes][64 bf16 rope]
//   indexer page (4352 B): [64 keys x 64 B codes of 128 dims][64 x 4 scale bytes]
// Rounding: the scale is the smallest 2^k with amax <= 6 * 2^k, so that no finite
// element is cut off at the largest code (k is kept in [-40, 125]: below, blocks
// that no attention could tell from zero; above, 6 * 2^k would not be finite). An
// element is off by at most 2^k, half the step between the largest codes' 4 and
// 6, ties going to the even code; an infinity becomes the largest code.
#pragma once

#include "dsa_common.h"

namespace dsa {

constexpr int kFp4MinExp = -40, kFp4MaxExp = 125;
constexpr int kFp4NaN = 255;
constexpr int kMla4RowBytes = 400;
constexpr int kMla4ScaleOff = 256;
constexpr int kMla4RopeOff = 272;
constexpr int kIdx4KeyBytes = 64;
constexpr int kIdx4KeyScales = 4;

// Scale byte of a block from its largest magnitude: amax = 1.m * 2^(e-127) is at
// most 6 * 2^k = 1.5 * 2^(k+2) where k = e - 129, plus 1 when 1.m > 1.5.
__device__ __forceinline__ int fp4_scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int k = (int)(u >> 23) - 129 + ((u & 0x7fffffu) > 0x400000u ? 1 : 0);
  return min(max(k, kFp4MinExp), kFp4MaxExp) + 127;
}

// The scale as the float operand of the conversion instructions, which use its
// exponent field only (0 stands for 2^-127, 255 gives NaN).
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight floats -> eight codes, element i in nibble i (round to nearest even, saturating).
__device__ __forceinline__ uint32_t f32x8_to_fp4(const float (&x)[8], float scale) {
  uint32_t w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
}

// Eight codes -> eight bf16 (exact).
__device__ __forceinline__ v4i fp4x8_to_bf16(uint32_t codes, float scale) {
  v4i r;
  r[0] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  r[1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  r[2] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  r[3] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return r;
}

// Eight bf16 -> floats.
__device__ __forceinline__ void bf16x8_to_f32(v4i raw, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (uint32_t)raw[i];
    x[2 * i] = bf16_to_f32((uint16_t)w);
    x[2 * i + 1] = bf16_to_f32((uint16_t)(w >> 16));
  }
}

// A block held by four neighbouring lanes, eight elements each: its scale byte
// (in all four) and this lane's eight codes.
__device__ __forceinline__ uint32_t fp4_quantise_block(const float (&x)[8], int* byte) {
  float amax = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax = fmaxf(amax, fabsf(x[i]));
    nan |= x[i] != x[i];
  }
  // a NaN counts as above every magnitude while the lanes agree on the largest
  uint32_t key = nan ? 0xffffffffu : __float_as_uint(amax);
  key = max(key, (uint32_t)__shfl_xor((int)key, 1, 64));
  key = max(key, (uint32_t)__shfl_xor((int)key, 2, 64));
  if (key == 0xffffffffu) {
    *byte = kFp4NaN;
    return 0u;
  }
  *byte = fp4_scale_byte(__uint_as_float(key));
  return f32x8_to_fp4(x, fp4_scale((uint32_t)*byte));
}

}  // namespace dsa
