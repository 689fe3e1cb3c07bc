// Root-mean-square norm with the residual's addition and an fp8 output, and the fp8
// rounding alone, for gfx950.
//
//   h = bf16(x + residual)                (or x; kept as the new residual stream)
//   y = h * (mean(h^2) + eps)^-1/2 * w    in f32 from the h that is kept
//   out = bf16(y); codes, scales = fp8 of y by blocks of 128 (fp8_block.h)
//
// One pass: a row stays in registers between its sum of squares and its outputs. Lanes
// take eight consecutive elements (16 bytes), so a block of 128 is 16 neighbouring lanes
// and its largest magnitude four shuffles. Codes and the bf16 output are each rounded
// once, from the same f32 y. The sum of squares is f32 in a fixed order: a row's results do
// not depend on the rows beside it.
//
// Memory bounds the norm of many rows: 8192 x 8192 with residual, its sum, fp8 and bf16 out, 604 MB, in
// 102 us (5.9 TB/s; a plain copy reaches 5.1). Few rows are one pass of latencies: 4 x 8192 in 3.8 us,
// of which an empty launch is more than half. A wave a row up to 512 elements (1000 x 512 in 2.9 us),
// then as many waves as give a lane one load up to 8192 (with half as many waves 4 x 8192 takes 4.2 and
// 8192 x 8192 105). Reading the weights before the sum made nothing faster. The rounding alone: 5001 x
// 1600, 24 MB, in 5.9 us.
#include "dsa_common.h"
#include "fp8_block.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

constexpr int kLane = 8;               // elements a lane takes at a time
constexpr int kMaxNormDim = 32768;     // 1024 threads, four times eight elements each
constexpr int kQuantThreads = 256;

struct NormParams {
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* residual;  // may be null
  int64_t residual_stride;
  uint16_t* sum;             // may be null; may be x or residual
  int64_t sum_stride;
  const void* weight;        // bf16 or f32
  float eps;
  int64_t rows;
  int dim;
  uint16_t* out;             // may be null
  int64_t out_stride;
  uint8_t* codes;            // may be null
  int64_t code_stride;
  void* scales;
  int64_t scale_stride;
};

// Elements i .. i + 7 of a row of n as bf16 pairs; zeros past its end. VEC: n a multiple of
// eight, 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ v4i load8(const uint16_t* row, int i, int n) {
  v4i r = {0, 0, 0, 0};
  if (VEC) {
    if (i < n) r = *reinterpret_cast<const v4i*>(row + i);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = i + 2 * j < n ? row[i + 2 * j] : 0u, hi = i + 2 * j + 1 < n ? row[i + 2 * j + 1] : 0u;
      r[j] = (int)(lo | (hi << 16));
    }
  }
  return r;
}

// Outputs are streamed past the L2, which has nothing more to do with them (8192 x 8192 110 -> 105 us, 5001 x
// 1600 6.5 -> 5.9; inputs read so cost more, 118 and 7.0).
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* row, int i, int n, v4i v) {
  if (VEC) {
    if (i < n) __builtin_nontemporal_store(v, reinterpret_cast<v4i*>(row + i));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) row[i + j] = (uint16_t)((uint32_t)v[j >> 1] >> (16 * (j & 1)));
  }
}

__device__ __forceinline__ void unpack8(v4i v, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float((uint32_t)v[j] << 16);
    x[2 * j + 1] = __uint_as_float((uint32_t)v[j] & 0xffff0000u);
  }
}

__device__ __forceinline__ v4i pack8(const float* x) {
  v4i v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = pack2(x[2 * j], x[2 * j + 1]);
  return v;
}

template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* row, int i, int n, uint2 c) {
  if (VEC) {
    if (i < n) __builtin_nontemporal_store((uint64_t)c.y << 32 | c.x, reinterpret_cast<uint64_t*>(row + i));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j < n) row[i + j] = (uint8_t)((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
  }
}

// The block of 16 neighbouring lanes' eight elements each, at elements i .. of a row of n.
template <int KIND, bool VEC>
__device__ __forceinline__ void quantise(const float* y, int i, int n, uint8_t* codes, void* scales) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(y[j]));
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) amax = fmaxf(amax, shfl_xor(amax, off));
  const uint32_t s = block_scale<KIND>(amax);
  store_codes<VEC>(codes, i, n, block_codes<KIND>(y, s));
  if (i % kBlock == 0 && i < n) {
    if (KIND == kScaleF32) static_cast<uint32_t*>(scales)[i / kBlock] = s;
    else static_cast<uint8_t*>(scales)[i / kBlock] = (uint8_t)s;
  }
}

// THREADS lanes a row, CHUNKS times eight elements each. Workgroups of 256 threads hold
// four rows of one wave each; wider ones a row.
template <int THREADS, int CHUNKS, int KIND, bool VEC, bool WF32>
__global__ void __launch_bounds__(THREADS < 256 ? 256 : THREADS) rms_norm_kernel(const NormParams P) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  constexpr int kWaves = THREADS / 64;
  __shared__ float part[kWaves];
  const int t = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / THREADS;
  if (row >= P.rows) return;  // whole waves, and no barrier among several rows
  const int n = P.dim;
  const uint16_t* x = P.x + row * P.x_stride;
  const uint16_t* res = P.residual ? P.residual + row * P.residual_stride : nullptr;

  float h[CHUNKS][8];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) unpack8(load8<VEC>(x, kLane * (c * THREADS + t), n), h[c]);
  if (res) {
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float r[8];
      unpack8(load8<VEC>(res, kLane * (c * THREADS + t), n), r);
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] += h[c][j];
      const v4i s = pack8(r);
      unpack8(s, h[c]);
      if (P.sum) store8<VEC>(P.sum + row * P.sum_stride, kLane * (c * THREADS + t), n, s);
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += h[c][j] * h[c][j];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) ss += shfl_xor(ss, off);
  if (kWaves > 1) {
    if ((t & 63) == 0) part[t >> 6] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) ss += part[w];
  }
  const float rstd = 1.f / sqrtf(ss / (float)n + P.eps);

  uint8_t* codes = P.codes ? P.codes + row * P.code_stride : nullptr;
  void* scales = KIND == kScaleF32 ? (void*)(static_cast<uint32_t*>(P.scales) + row * P.scale_stride)
                                   : (void*)(static_cast<uint8_t*>(P.scales) + row * P.scale_stride);
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int i = kLane * (c * THREADS + t);
    float w[8], y[8];
    if (WF32) {
      const float* wf = static_cast<const float*>(P.weight);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = i + j < n ? wf[i + j] : 0.f;
    } else {
      unpack8(load8<VEC>(static_cast<const uint16_t*>(P.weight), i, n), w);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = h[c][j] * rstd * w[j];
    if (P.out) store8<VEC>(P.out + row * P.out_stride, i, n, pack8(y));
    if (codes) quantise<KIND, VEC>(y, i, n, codes, scales);
  }
}

// The rounding alone: 16 lanes a block, blocks of a row beside each other.
template <int KIND, bool VEC>
__global__ void __launch_bounds__(kQuantThreads)
act_quant_kernel(const uint16_t* __restrict__ x, int64_t x_stride, int64_t blocks, int per_row, int dim,
                 uint8_t* __restrict__ codes, int64_t code_stride, void* __restrict__ scales, int64_t scale_stride) {
  const int64_t b = ((int64_t)blockIdx.x * kQuantThreads + threadIdx.x) >> 4;
  if (b >= blocks) return;  // 16 lanes together
  const int64_t row = b / per_row;
  const int i = (int)(b - row * per_row) * kBlock + kLane * (threadIdx.x & 15);
  float y[8];
  unpack8(load8<VEC>(x + row * x_stride, i, dim), y);
  void* s = KIND == kScaleF32 ? (void*)(static_cast<uint32_t*>(scales) + row * scale_stride)
                              : (void*)(static_cast<uint8_t*>(scales) + row * scale_stride);
  quantise<KIND, VEC>(y, i, dim, codes + row * code_stride, s);
}

template <int THREADS, int CHUNKS, int KIND>
int launch_norm(const NormParams& P, bool vec, bool wf32, hipStream_t st) {
  constexpr int kRows = THREADS < 256 ? 256 / THREADS : 1;
  const int64_t groups = (P.rows + kRows - 1) / kRows;
  if (!launch_holds(groups, kRows * THREADS))
    return set_error(kUnsupported, "dsa_rms_norm: %lld rows of %d take 2^32 threads or more", (long long)P.rows, P.dim);
  const dim3 grid((unsigned)groups), block(kRows * THREADS);
  if (vec && wf32) hipLaunchKernelGGL((rms_norm_kernel<THREADS, CHUNKS, KIND, true, true>), grid, block, 0, st, P);
  else if (vec) hipLaunchKernelGGL((rms_norm_kernel<THREADS, CHUNKS, KIND, true, false>), grid, block, 0, st, P);
  else if (wf32) hipLaunchKernelGGL((rms_norm_kernel<THREADS, CHUNKS, KIND, false, true>), grid, block, 0, st, P);
  else hipLaunchKernelGGL((rms_norm_kernel<THREADS, CHUNKS, KIND, false, false>), grid, block, 0, st, P);
  return check_launch("dsa_rms_norm");
}

template <int KIND>
int norm_by_dim(const NormParams& P, bool vec, bool wf32, hipStream_t st) {
  const int lanes = (P.dim + kLane - 1) / kLane;
  if (lanes <= 64) return launch_norm<64, 1, KIND>(P, vec, wf32, st);
  if (lanes <= 256) return launch_norm<256, 1, KIND>(P, vec, wf32, st);
  if (lanes <= 512) return launch_norm<512, 1, KIND>(P, vec, wf32, st);
  if (lanes <= 1024) return launch_norm<1024, 1, KIND>(P, vec, wf32, st);
  if (lanes <= 2048) return launch_norm<1024, 2, KIND>(P, vec, wf32, st);
  return launch_norm<1024, 4, KIND>(P, vec, wf32, st);
}

bool aligned(const void* p, int64_t stride, int elements) {  // 2-byte or 1-byte elements, `elements` to a load
  return !p || (!(reinterpret_cast<uintptr_t>(p) & (elements == 8 ? 15 : 7)) && !(stride & 7));
}

}  // namespace
}  // namespace dsa

extern "C" {

int dsa_rms_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride, void* residual_out,
                 int64_t residual_out_stride, const void* weight, int weight_is_f32, float eps, int64_t rows, int dim,
                 void* out, int64_t out_stride, uint8_t* codes, int64_t code_stride, void* scales,
                 int64_t scale_stride, int scale_kind, void* stream) {
  using namespace dsa;
  if (rows < 0 || rows > INT32_MAX || dim < 1) return set_error(kInvalidArgument, "dsa_rms_norm: bad sizes");
  if (dim > kMaxNormDim) return set_error(kUnsupported, "dsa_rms_norm: dim %d (at most %d)", dim, kMaxNormDim);
  if (!(eps >= 0.f) || eps > 3e38f) return set_error(kInvalidArgument, "dsa_rms_norm: eps must be finite and not negative");
  if (scale_kind != kScaleF32 && scale_kind != kScaleE8M0)
    return set_error(kInvalidArgument, "dsa_rms_norm: unknown scale kind %d", scale_kind);
  if (rows == 0) return kOk;
  if (!x || !weight || (!out && !codes)) return set_error(kInvalidArgument, "dsa_rms_norm: null pointer");
  if (!codes != !scales) return set_error(kInvalidArgument, "dsa_rms_norm: codes and scales go together");
  if (residual_out && !residual) return set_error(kInvalidArgument, "dsa_rms_norm: residual_out without residual");
  const int64_t blocks = (dim + kBlock - 1) / kBlock;
  if (rows > 1 && (x_stride < dim || (residual && residual_stride < dim) || (residual_out && residual_out_stride < dim) ||
                   (out && out_stride < dim) || (codes && (code_stride < dim || scale_stride < blocks))))
    return set_error(kInvalidArgument, "dsa_rms_norm: rows overlap");
  if (out && out == residual_out)
    return set_error(kInvalidArgument, "dsa_rms_norm: out and residual_out are the same memory");
  if (rows > 1 && ((out && out == x && out_stride != x_stride) ||
                   (residual_out && ((residual_out == x && residual_out_stride != x_stride) ||
                                     (residual_out == residual && residual_out_stride != residual_stride)))))
    return set_error(kInvalidArgument, "dsa_rms_norm: in place, rows need the same stride");
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) |
        reinterpret_cast<uintptr_t>(residual_out) | reinterpret_cast<uintptr_t>(out)) & 1) ||
      (reinterpret_cast<uintptr_t>(weight) & (weight_is_f32 ? 3 : 1)) ||
      (scale_kind == kScaleF32 && (reinterpret_cast<uintptr_t>(scales) & 3)))
    return set_error(kInvalidArgument, "dsa_rms_norm: pointers must be aligned to their elements");
  const NormParams P = {static_cast<const uint16_t*>(x), x_stride, static_cast<const uint16_t*>(residual),
                        residual_stride, static_cast<uint16_t*>(residual_out), residual_out_stride, weight, eps, rows,
                        dim, static_cast<uint16_t*>(out), out_stride, codes, code_stride, scales, scale_stride};
  const bool vec = dim % kLane == 0 && aligned(x, x_stride, 8) && aligned(residual, residual_stride, 8) &&
                   aligned(residual_out, residual_out_stride, 8) && aligned(out, out_stride, 8) &&
                   aligned(weight, 0, 8) && aligned(codes, code_stride, 4);
  return scale_kind == kScaleF32 ? norm_by_dim<kScaleF32>(P, vec, weight_is_f32, (hipStream_t)stream)
                                 : norm_by_dim<kScaleE8M0>(P, vec, weight_is_f32, (hipStream_t)stream);
}

int dsa_act_quant(const void* x, int64_t x_stride, int64_t rows, int dim, uint8_t* codes, int64_t code_stride,
                  void* scales, int64_t scale_stride, int scale_kind, void* stream) {
  using namespace dsa;
  if (rows < 0 || rows > INT32_MAX || dim < 1) return set_error(kInvalidArgument, "dsa_act_quant: bad sizes");
  if (scale_kind != kScaleF32 && scale_kind != kScaleE8M0)
    return set_error(kInvalidArgument, "dsa_act_quant: unknown scale kind %d", scale_kind);
  if (rows == 0) return kOk;
  if (!x || !codes || !scales) return set_error(kInvalidArgument, "dsa_act_quant: null pointer");
  const int per_row = (int)(((int64_t)dim + kBlock - 1) / kBlock);
  if (rows > 1 && (x_stride < dim || code_stride < dim || scale_stride < per_row))
    return set_error(kInvalidArgument, "dsa_act_quant: rows overlap");
  if ((reinterpret_cast<uintptr_t>(x) & 1) || (scale_kind == kScaleF32 && (reinterpret_cast<uintptr_t>(scales) & 3)))
    return set_error(kInvalidArgument, "dsa_act_quant: pointers must be aligned to their elements");
  const int64_t blocks = rows * per_row;
  const int64_t groups = (blocks + kQuantThreads / 16 - 1) / (kQuantThreads / 16);
  if (!launch_holds(groups, kQuantThreads))
    return set_error(kUnsupported, "dsa_act_quant: %lld blocks of 128 take 2^32 threads or more", (long long)blocks);
  const bool vec = dim % kLane == 0 && aligned(x, x_stride, 8) && aligned(codes, code_stride, 4);
  const dim3 grid((unsigned)groups), block(kQuantThreads);
  const hipStream_t st = (hipStream_t)stream;
  const uint16_t* xb = static_cast<const uint16_t*>(x);
#define DSA_QUANT(KIND, VEC)                                                                                        \
  hipLaunchKernelGGL((act_quant_kernel<KIND, VEC>), grid, block, 0, st, xb, x_stride, blocks, per_row, dim, codes, \
                     code_stride, scales, scale_stride)
  if (scale_kind == kScaleF32) {
    if (vec) DSA_QUANT(kScaleF32, true); else DSA_QUANT(kScaleF32, false);
  } else {
    if (vec) DSA_QUANT(kScaleE8M0, true); else DSA_QUANT(kScaleE8M0, false);
  }
#undef DSA_QUANT
  return check_launch("dsa_act_quant");
}

}  // extern "C"
