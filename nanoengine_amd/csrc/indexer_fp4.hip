// Lightning-indexer logits over a 4-bit paged key cache (format: fp4.h), for gfx950.
//
//   logits[b*n+j, t] = sum_h w[b*n+j, h] * relu(q[b,j,h,:] . k[t,:])
//
// One wave per page of 64 keys: lane t holds key t in registers, the query's 64
// heads pass by in LDS.
#include "dsa_common.h"
#include "fp4.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

constexpr int kPage = 64, kDim = 128, kHeads = 64;
constexpr int kPageBytes4 = kPage * (kIdx4KeyBytes + kIdx4KeyScales);

__global__ void __launch_bounds__(64)
indexer_logits_fp4_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ kv, int64_t num_pages,
                          const float* __restrict__ weights, const int32_t* __restrict__ ctx,
                          const int32_t* __restrict__ bt, int64_t bt_stride, int next_n, int64_t max_ctx,
                          float* __restrict__ logits, int64_t stride, int clean) {
  __shared__ float qs[kDim];
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.y, p = blockIdx.x, t = p * kPage + lane;
  const int64_t L = min((int64_t)ctx[row], max_ctx);
  int64_t longest = 0;  // of the batch entry's rows
  for (int j = 0; j < next_n; ++j) longest = max(longest, min((int64_t)ctx[row / next_n * next_n + j], max_ctx));
  if (p * kPage >= longest) {
    if (clean && t < max_ctx) logits[row * stride + t] = -__builtin_inff();
    return;
  }
  const int64_t page = bt[row / next_n * bt_stride + p];
  if (page < 0 || page >= num_pages) {
    if (t < max_ctx) logits[row * stride + t] = -__builtin_inff();
    return;
  }
  const uint8_t* base = kv + page * kPageBytes4;
  float k[kDim];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const v4i codes = *reinterpret_cast<const v4i*>(base + lane * kIdx4KeyBytes + 16 * b);
    const float s = fp4_scale(base[kPage * kIdx4KeyBytes + lane * kIdx4KeyScales + b]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[8];
      bf16x8_to_f32(fp4x8_to_bf16((uint32_t)codes[i], s), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) k[32 * b + 8 * i + e] = x[e];
    }
  }
  float sum = 0.f;
  for (int h = 0; h < kHeads; ++h) {
    const uint32_t two = *reinterpret_cast<const uint16_t*>(q + (row * kHeads + h) * kDim + 2 * lane);
    __syncthreads();
    qs[2 * lane] = __builtin_amdgcn_cvt_f32_fp8((int)two, 0);
    qs[2 * lane + 1] = __builtin_amdgcn_cvt_f32_fp8((int)two, 1);
    __syncthreads();
    float dot = 0.f;
#pragma unroll
    for (int d = 0; d < kDim; ++d) dot = fmaf(qs[d], k[d], dot);
    sum = fmaf(weights[row * kHeads + h], dot > 0.f || dot != dot ? dot : 0.f, sum);
  }
  if (t < max_ctx) logits[row * stride + t] = t < L ? sum : -__builtin_inff();
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_indexer_logits_fp4(const uint8_t* q_fp8, const uint8_t* kv_cache, int64_t num_pages,
                                      const float* weights, const int32_t* context_lens, const int32_t* block_tables,
                                      int64_t block_table_stride, int batch, int next_n, int num_heads, int head_dim,
                                      int page_size, int64_t max_context_len, float* logits, int64_t logits_stride,
                                      int clean_logits, void* stream) {
  using namespace dsa;
  if (num_heads != kHeads || head_dim != kDim)
    return set_error(kUnsupported, "indexer_fp4: num_heads=%d head_dim=%d unsupported (need 64, 128)", num_heads,
                     head_dim);
  if (page_size != kPage) return set_error(kUnsupported, "indexer_fp4: page_size=%d unsupported (need 64)", page_size);
  if (next_n != 1 && next_n != 2)
    return set_error(kUnsupported, "indexer_fp4: next_n=%d unsupported (1 or 2)", next_n);
  if (batch < 0 || max_context_len < 0 || num_pages < 0 || logits_stride < max_context_len)
    return set_error(kInvalidArgument, "indexer_fp4: bad sizes");
  if (batch == 0 || max_context_len == 0) return kOk;
  if (!q_fp8 || !kv_cache || !weights || !context_lens || !block_tables || !logits)
    return set_error(kInvalidArgument, "indexer_fp4: null pointer");
  if ((reinterpret_cast<uintptr_t>(q_fp8) | reinterpret_cast<uintptr_t>(kv_cache)) & 15)
    return set_error(kInvalidArgument, "indexer_fp4: q and kv_cache must be 16-byte aligned");
  const int64_t pages = (max_context_len + kPage - 1) / kPage;
  if (pages > INT32_MAX || (int64_t)batch * next_n > 65535)
    return set_error(kUnsupported, "indexer_fp4: at most 65535 rows");
  hipLaunchKernelGGL(indexer_logits_fp4_kernel, dim3((unsigned)pages, (unsigned)(batch * next_n)), dim3(64), 0,
                     (hipStream_t)stream, q_fp8, kv_cache, num_pages, weights, context_lens, block_tables,
                     block_table_stride, next_n, max_context_len, logits, logits_stride, clean_logits);
  return check_launch("dsa_indexer_logits_fp4");
}
