// Products of fp8 matrices with a scale for each block of 128, for gfx950.
//
//   out[m, n] = sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k]
//
// a: activations [M, K], b: weights [N, K], both e4m3fn with K contiguous; scales float32,
// or powers of two as e8m0 bytes, which the matrix instruction applies itself.
//
// The products run on v_mfma_scale_f32_32x32x64_f8f6f4 with the weights as its rows, so that
// a lane ends up with one activation row's results for four neighbouring columns at a time.
// A workgroup's tiles of a and b go straight from HBM into LDS, a block of 128 deep, two
// buffers deep: while one is multiplied the next is on its way. A row's eight 16-byte pieces
// are stored in the order piece ^ (row & 7): eight rows' reads of one piece fall on
// different banks.
#include <algorithm>

#include "dsa_common.h"
#include "fp8_block.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

struct GemmParams {
  const uint8_t *a, *b;
  int64_t a_stride, b_stride;
  const void *sa, *sb;
  int64_t sa_stride, sb_stride;
  int m, n, k;
  int kblocks;
  int mtiles, ntiles, splits;
  void* out;          // bf16 or f32; partial sums of split s at s * m * n
  int64_t out_stride;
};

// What rows' pieces past the end of K are read from.
__device__ __align__(16) const uint8_t g_gemm_zero[16] = {};

__device__ __forceinline__ void dma16(const void* g, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)reinterpret_cast<uintptr_t>(p); }

enum OutKind : int { kOutBf16 = 0, kOutF32 = 1 };

template <int KIND>
__device__ __forceinline__ uint32_t load_scale(const void* s, int64_t i) {
  return KIND == kScaleF32 ? static_cast<const uint32_t*>(s)[i] : (uint32_t)static_cast<const uint8_t*>(s)[i];
}

__device__ __forceinline__ int pack2(float a, float b) { return __builtin_bit_cast(int, (v2bf){(__bf16)a, (__bf16)b}); }

template <int OUT>
__device__ __forceinline__ void store4(void* out, int64_t at, bool whole, int left, const float* v) {
  if (OUT == kOutBf16) {
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    const v2i p = {pack2(v[0], v[1]), pack2(v[2], v[3])};
    if (whole) *reinterpret_cast<v2i*>(o) = p;
    else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = (uint16_t)((uint32_t)p[j >> 1] >> (16 * (j & 1)));
  } else {
    float* o = static_cast<float*>(out) + at;
    if (whole) *reinterpret_cast<v4f*>(o) = (v4f){v[0], v[1], v[2], v[3]};
    else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = v[j];
  }
}

// A tile of BM activation rows and BN weight rows; a wave takes WM x WN of it.
template <int BM, int BN, int WM, int WN, int KIND, int OUT>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64) fp8_gemm_kernel(const GemmParams P) {
  constexpr int kWaves = (BM / WM) * (BN / WN);
  constexpr int kMt = WM / 32, kNt = WN / 32;
  constexpr int kStage = (BM + BN) * kBlock;
  constexpr int kLoads = (BM + BN) / 8;            // instructions of a stage: eight rows each
  constexpr int kPer = (kLoads + kWaves - 1) / kWaves;
  static_assert(kLoads % kWaves == 0 && BM % 8 == 0, "rows dealt out evenly");
  static_assert(kBlock % WN == 0, "one weight scale a wave");
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % (P.mtiles * P.ntiles), split = blockIdx.x / (P.mtiles * P.ntiles);
  const int m0 = (tile % P.mtiles) * BM, n0 = (tile / P.mtiles) * BN;
  const int kb0 = (int)((int64_t)P.kblocks * split / P.splits), kb1 = (int)((int64_t)P.kblocks * (split + 1) / P.splits);
  const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
  const int c32 = lane & 31, half = lane >> 5;

  // this lane's pieces of a stage; rows past the matrix repeat its last one
  const uint8_t* src[kPer];
  const int piece = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = 8 * (wave + i * kWaves) + (lane >> 3);
    src[i] = row < BM ? P.a + (int64_t)min(m0 + row, P.m - 1) * P.a_stride
                      : P.b + (int64_t)min(n0 + row - BM, P.n - 1) * P.b_stride;
    src[i] += 16 * piece;
  }
  auto issue = [&](int kb, int buf) {
    const uint32_t dst = lds_addr(smem) + buf * kStage + wave * 1024;
    const bool there = kb * kBlock + 16 * piece < P.k;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      dma16(there ? src[i] + (int64_t)kb * kBlock : g_gemm_zero, dst + i * kWaves * 1024);
  };

  int64_t sa_at[kMt];
#pragma unroll
  for (int i = 0; i < kMt; ++i) sa_at[i] = (int64_t)min(m0 + wm + 32 * i + c32, P.m - 1) * P.sa_stride;
  const int64_t sb_at = (int64_t)min((n0 + wn) / kBlock, (P.n - 1) / kBlock) * P.sb_stride;
  uint32_t sa[kMt], sb;
  auto load_scales = [&](int kb) {
#pragma unroll
    for (int i = 0; i < kMt; ++i) sa[i] = load_scale<KIND>(P.sa, sa_at[i] + kb);
    sb = load_scale<KIND>(P.sb, sb_at + kb);
  };

  v16f acc[kNt][kMt];
#pragma unroll
  for (int i = 0; i < kNt; ++i)
#pragma unroll
    for (int j = 0; j < kMt; ++j) acc[i][j] = (v16f){};

  // offsets of this lane's two 16-byte pieces of each 64-deep half of a row
  uint32_t off[2][2];
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
#pragma unroll
    for (int j = 0; j < 2; ++j) off[ks][j] = c32 * kBlock + 16 * ((4 * ks + 2 * half + j) ^ (lane & 7));

  if (kb0 < kb1) {
    load_scales(kb0);
    issue(kb0, 0);
  }
  for (int kb = kb0; kb < kb1; ++kb) {
    const int buf = (kb - kb0) & 1;
    // this wave's share of the block has landed and its reads of the other buffer are done; past
    // the barrier so are the others'
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    uint32_t ca[kMt], cb;  // this block's scales, read one block ahead
#pragma unroll
    for (int i = 0; i < kMt; ++i) {
      asm volatile("" : "+v"(sa[i]));
      ca[i] = sa[i];
    }
    asm volatile("" : "+v"(sb));
    cb = sb;
    if (kb + 1 < kb1) {
      load_scales(kb + 1);
      issue(kb + 1, buf ^ 1);
    }
    const uint8_t* at = smem + buf * kStage + wm * kBlock;
    const uint8_t* bt = smem + buf * kStage + (BM + wn) * kBlock;
    auto operand = [&](const uint8_t* base, int ks) {
      const v4i x = *reinterpret_cast<const v4i*>(base + off[ks][0]), y = *reinterpret_cast<const v4i*>(base + off[ks][1]);
      return (v8i){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    v8i fa[kMt][2], fb[kNt][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int i = 0; i < kNt; ++i) fb[i][ks] = operand(bt + i * 32 * kBlock, ks);
#pragma unroll
      for (int j = 0; j < kMt; ++j) fa[j][ks] = operand(at + j * 32 * kBlock, ks);
    }
    if (KIND == kScaleE8M0) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int j = 0; j < kMt; ++j)
#pragma unroll
          for (int i = 0; i < kNt; ++i)
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[i][ks], fa[j][ks], acc[i][j], 0, 0, 0, cb, 0,
                                                                        ca[j]);
    } else {
#pragma unroll
      for (int j = 0; j < kMt; ++j) {
        const float s = __uint_as_float(ca[j]) * __uint_as_float(cb);
#pragma unroll
        for (int i = 0; i < kNt; ++i) {
          v16f part = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[i][0], fa[j][0], (v16f){}, 0, 0, 0, 127, 0, 127);
          part = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[i][1], fa[j][1], part, 0, 0, 0, 127, 0, 127);
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][j][r] += part[r] * s;
        }
      }
    }
  }

  // lane (c32, half): row c32 of an activation tile, columns 8g + 4 half .. + 3 of a weight tile
  void* out = P.out;
  if (P.splits > 1) out = static_cast<float*>(P.out) + (int64_t)split * P.m * P.n;
  const bool aligned = !((reinterpret_cast<uintptr_t>(out) & (OUT == kOutBf16 ? 7 : 15)) | (P.out_stride & 3));
#pragma unroll
  for (int j = 0; j < kMt; ++j) {
    const int m = m0 + wm + 32 * j + c32;
    if (m >= P.m) continue;
#pragma unroll
    for (int i = 0; i < kNt; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int n = n0 + wn + 32 * i + 8 * g + 4 * half;
        const float v[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        if (n < P.n) store4<OUT>(out, (int64_t)m * P.out_stride + n, aligned && n + 4 <= P.n, P.n - n, v);
      }
  }
}

// out = the sum of the splits' partial sums, in order.
template <int OUT>
__global__ void __launch_bounds__(256)
fp8_gemm_sum_kernel(const float* __restrict__ part, int splits, int m, int n, void* __restrict__ out, int64_t out_stride) {
  const int per_row = (n + 3) / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / per_row;
  if (row >= m) return;
  const int c = (int)(i - row * per_row) * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const bool whole = n % 4 == 0;
  for (int s = 0; s < splits; ++s) {
    const float* p = part + ((int64_t)s * m + row) * n + c;
    if (whole) {
      const v4f x = *reinterpret_cast<const v4f*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += x[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j < n) v[j] += p[j];
    }
  }
  const bool aligned = !((reinterpret_cast<uintptr_t>(out) & (OUT == kOutBf16 ? 7 : 15)) | (out_stride & 3));
  store4<OUT>(out, row * out_stride + c, aligned && whole, n - c, v);
}

// Tile and split of a shape.
struct Plan {
  int bm, bn, splits;
};

Plan plan_of(int m, int n, int k, int cus) {
  const int kblocks = (k + kBlock - 1) / kBlock;
  Plan p = {32, 64, 1};
  auto tiles = [&](int bm, int bn) { return (int64_t)((m + bm - 1) / bm) * ((n + bn - 1) / bn); };
  if (tiles(256, 256) >= cus) p = {256, 256, 1};
  else if (m > 64) p = {128, 128, 1};
  else if (m > 32) p = {64, 128, 1};
  const int64_t t = tiles(p.bm, p.bn);
  // as many parts as fill the CUs twice, of at least four blocks each
  if (p.bm < 256) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({2 * cus / std::max<int64_t>(t, 1), kblocks / 4, 16}));
  return p;
}

int device_cus() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
    return 256;
  return n;
}

template <int BM, int BN, int WM, int WN, int KIND, int OUT>
int launch_tile(GemmParams P, hipStream_t st) {
  constexpr int kSmem = 2 * (BM + BN) * kBlock;
  auto kern = fp8_gemm_kernel<BM, BN, WM, WN, KIND, OUT>;
  if (kSmem > 64 * 1024) {
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != hipSuccess) return set_error(kLaunchFailed, "dsa_fp8_gemm: %s", hipGetErrorString(e));
  }
  P.mtiles = (P.m + BM - 1) / BM;
  P.ntiles = (P.n + BN - 1) / BN;
  const int64_t groups = (int64_t)P.mtiles * P.ntiles * P.splits;
  if (groups > INT32_MAX) return set_error(kUnsupported, "dsa_fp8_gemm: more than 2^31 tiles");
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3((BM / WM) * (BN / WN) * 64), kSmem, st, P);
  return check_launch("dsa_fp8_gemm");
}

template <int KIND, int OUT>
int launch_plan(const Plan& p, const GemmParams& P, hipStream_t st) {
  if (p.bm == 256) return launch_tile<256, 256, 128, 64, KIND, OUT>(P, st);
  if (p.bm == 128) return launch_tile<128, 128, 64, 64, KIND, OUT>(P, st);
  if (p.bm == 64) return launch_tile<64, 128, 64, 32, KIND, OUT>(P, st);
  return launch_tile<32, 64, 32, 32, KIND, OUT>(P, st);
}

}  // namespace
}  // namespace dsa

extern "C" {

size_t dsa_fp8_gemm_workspace_bytes(int m, int n, int k) {
  using namespace dsa;
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Plan p = plan_of(m, n, k, device_cus());
  return p.splits > 1 ? (size_t)p.splits * m * n * sizeof(float) : 0;
}

int dsa_fp8_gemm(const uint8_t* a, int64_t a_stride, const void* a_scale, int64_t a_scale_stride, const uint8_t* b,
                 int64_t b_stride, const void* b_scale, int64_t b_scale_stride, int scale_kind, int m, int n, int k,
                 void* out, int64_t out_stride, int out_is_f32, void* workspace, size_t workspace_bytes,
                 void* stream) {
  using namespace dsa;
  if (m < 0 || n < 0 || k < 1) return set_error(kInvalidArgument, "dsa_fp8_gemm: bad sizes");
  if (k & 15) return set_error(kUnsupported, "dsa_fp8_gemm: k %d is no multiple of 16", k);
  if (scale_kind != kScaleF32 && scale_kind != kScaleE8M0)
    return set_error(kInvalidArgument, "dsa_fp8_gemm: unknown scale kind %d", scale_kind);
  if (m == 0 || n == 0) return kOk;
  if (!a || !a_scale || !b || !b_scale || !out) return set_error(kInvalidArgument, "dsa_fp8_gemm: null pointer");
  const int kblocks = (k + kBlock - 1) / kBlock;
  if ((m > 1 && (a_stride < k || a_scale_stride < kblocks || out_stride < n)) || (n > 1 && b_stride < k) ||
      (n > kBlock && b_scale_stride < kblocks))
    return set_error(kInvalidArgument, "dsa_fp8_gemm: rows overlap");
  if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) || ((a_stride | b_stride) & 15))
    return set_error(kInvalidArgument, "dsa_fp8_gemm: rows of a and b must be 16-byte aligned");
  if ((scale_kind == kScaleF32 && ((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) & 3)) ||
      (reinterpret_cast<uintptr_t>(out) & (out_is_f32 ? 3 : 1)))
    return set_error(kInvalidArgument, "dsa_fp8_gemm: pointers must be aligned to their elements");
  const Plan p = plan_of(m, n, k, device_cus());
  const size_t need = p.splits > 1 ? (size_t)p.splits * m * n * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return set_error(kWorkspaceTooSmall, "dsa_fp8_gemm: workspace %zu bytes, %zu needed", workspace_bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(kInvalidArgument, "dsa_fp8_gemm: the workspace must be 16-byte aligned");
  GemmParams P = {a, b, a_stride, b_stride, a_scale, b_scale, a_scale_stride, b_scale_stride, m, n, k, kblocks,
                  0, 0, p.splits, out, out_stride};
  const hipStream_t st = (hipStream_t)stream;
  if (p.splits > 1) {
    P.out = workspace;
    P.out_stride = n;
    const int rc = scale_kind == kScaleF32 ? launch_plan<kScaleF32, kOutF32>(p, P, st) : launch_plan<kScaleE8M0, kOutF32>(p, P, st);
    if (rc != kOk) return rc;
    const int64_t threads = (int64_t)m * ((n + 3) / 4);
    const dim3 grid((unsigned)((threads + 255) / 256));
    if (out_is_f32)
      hipLaunchKernelGGL(fp8_gemm_sum_kernel<kOutF32>, grid, dim3(256), 0, st, static_cast<const float*>(workspace),
                         p.splits, m, n, out, out_stride);
    else
      hipLaunchKernelGGL(fp8_gemm_sum_kernel<kOutBf16>, grid, dim3(256), 0, st, static_cast<const float*>(workspace),
                         p.splits, m, n, out, out_stride);
    return check_launch("dsa_fp8_gemm");
  }
  if (out_is_f32)
    return scale_kind == kScaleF32 ? launch_plan<kScaleF32, kOutF32>(p, P, st) : launch_plan<kScaleE8M0, kOutF32>(p, P, st);
  return scale_kind == kScaleF32 ? launch_plan<kScaleF32, kOutBf16>(p, P, st) : launch_plan<kScaleE8M0, kOutBf16>(p, P, st);
}

}  // extern "C"
