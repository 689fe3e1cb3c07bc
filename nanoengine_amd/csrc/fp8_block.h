// Activations in fp8 with one scale per 128 elements of a row, shared by the writers
// (norm_quant.hip) and the product that reads them (fp8_gemm.hip).
//
//   code = e4m3fn(x / s), s the block's scale, in one of two forms:
//     kScaleF32   s = max(amax, 2^-40) / 448 as float32
//     kScaleE8M0  the smallest power of two 2^(byte - 127) that is not below that, as its byte
// The floor keeps blocks of zeros (and of nothing but values below 2^-40) at a scale whose
// inverse is a normal number. Nothing finite saturates. A NaN gets the NaN code and leaves
// the other elements of its block as they are; an infinity gets the NaN code, with the scale
// infinite (f32) or the largest that is not (e8m0): products with such a row are NaN either way.
#pragma once

#include "dsa_common.h"

namespace dsa {

constexpr int kBlock = 128;
enum ScaleKind : int { kScaleF32 = 0, kScaleE8M0 = 1 };
constexpr float kAmaxFloor = 0x1p-40f;
constexpr float kFp8Max = 448.f;

// Exponent byte of the smallest power of two >= s: s positive and normal, or infinite.
__device__ __forceinline__ uint32_t e8m0_ceil(float s) {
  const uint32_t u = __float_as_uint(s);
  const uint32_t byte = (u >> 23) + ((u & 0x7fffffu) ? 1u : 0u);
  return byte < 254u ? byte : 254u;
}

// A block's scale from its largest magnitude; *inv is what its elements are multiplied by
// (for f32 scales the rounded inverse: off by half a step of 2^-24, before a rounding of 2^-4).
template <int KIND>
__device__ __forceinline__ uint32_t block_scale(float amax, float* inv) {
  const float s = fmaxf(amax, kAmaxFloor) / kFp8Max;
  if (KIND == kScaleF32) {
    *inv = 1.f / s;
    return __float_as_uint(s);
  }
  const uint32_t byte = e8m0_ceil(s);
  // 2^(127 - byte), exact: byte 254 gives a subnormal that the products keep
  *inv = __uint_as_float(byte < 254u ? (254u - byte) << 23 : 0x400000u);
  return byte;
}

}  // namespace dsa
