// Activations in fp8 with one scale per 128 elements of a row, shared by the writers
// (norm_quant.hip) and the product that reads them (fp8_gemm.hip).
//
//   code = e4m3fn(x / s), s the block's scale, in one of two forms:
//     kScaleF32   s = max(amax, 2^-40) / 448 as float32
//     kScaleE8M0  the smallest power of two 2^(byte - 127) that is not below that, as its byte
// The floor keeps blocks of zeros (and of nothing but values below 2^-40) at a scale that is
// a normal number, as its inverse is. Nothing finite saturates. A NaN gets the NaN code and leaves
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

// A block's scale from its largest magnitude, as it is stored.
template <int KIND>
__device__ __forceinline__ uint32_t block_scale(float amax) {
  const float s = fmaxf(amax, kAmaxFloor) / kFp8Max;
  return KIND == kScaleF32 ? __float_as_uint(s) : e8m0_ceil(s);
}

// Eight elements of a block over its scale, in two words of four codes. For a power of two that is a product with its exact
// inverse (byte 254 has a subnormal one, which the products keep). For a float32 scale q = y (1 / s) is off by a step or so,
// which gives codes next to a tie their neighbours' value (1 of 2000 in rows of bf16); the remainder q s - y is exact in
// one fused operation, and q - remainder (1 / s) is y / s rounded once (Markstein, 1990: IBM J. Res. Dev. 34). Eight
// divisions instead took 8192 x 8192 from 38 to 47 us. (Remainders lose bits where |q| is far below the smallest code's
// half, 2^-10. An infinite scale counts as 0 in them: what is finite over it is 0.)
template <int KIND>
__device__ __forceinline__ uint2 block_codes(const float* y, uint32_t scale) {
  float q[8];
  if (KIND == kScaleF32) {
    const float s = __uint_as_float(scale), inv = 1.f / s, by = inv == 0.f ? 0.f : s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float first = y[j] * inv;
      q[j] = fmaf(-fmaf(first, by, -y[j]), inv, first);  // (so written, a zero keeps its sign)
    }
  } else {
    const float inv = __uint_as_float(scale < 254u ? (254u - scale) << 23 : 0x400000u);
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = y[j] * inv;
  }
  return make_uint2(f32x4_to_fp8(q[0], q[1], q[2], q[3]), f32x4_to_fp8(q[4], q[5], q[6], q[7]));
}

}  // namespace dsa
