// Sparse MLA decode over a 4-bit paged MLA cache (format: fp4.h), for gfx950.
//
// One wave per (token, head): lane l holds query dims 8l .. 8l+7 and rope dim l, the
// selected rows pass by one at a time with a running maximum and sum.
#include "dsa_common.h"
#include "fp4.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

__global__ void __launch_bounds__(64)
sparse_mla_fp4_kernel(const uint16_t* __restrict__ q, int64_t q_tok_stride, int64_t q_head_stride,
                      const uint8_t* __restrict__ kv, int64_t blk_stride, int block_size, int64_t num_blocks,
                      const int32_t* __restrict__ idx, int64_t idx_stride, int H, int topk, float scale,
                      uint16_t* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x;
  const int64_t th = blockIdx.x, t = th / H, h = th % H;
  const uint16_t* qr = q + t * q_tok_stride + h * q_head_stride;
  float qn[8];
  bf16x8_to_f32(*reinterpret_cast<const v4i*>(qr + 8 * lane), qn);
  const float qp = bf16_to_f32(qr[512 + lane]);
  float m = -__builtin_inff(), l = 0.f, o[8] = {};
  for (int i = 0; i < topk; ++i) {
    const int32_t slot = idx[t * idx_stride + i];
    if (slot < 0 || slot / block_size >= num_blocks) continue;
    const uint8_t* row = kv + (int64_t)(slot / block_size) * blk_stride + (int64_t)(slot % block_size) * kMla4RowBytes;
    float v[8];
    bf16x8_to_f32(fp4x8_to_bf16(*reinterpret_cast<const uint32_t*>(row + 4 * lane),
                                fp4_scale(row[kMla4ScaleOff + (lane >> 2)])), v);
    float s = qp * bf16_to_f32(*reinterpret_cast<const uint16_t*>(row + kMla4RopeOff + 2 * lane));
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(qn[e], v[e], s);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += shfl_xor(s, off);
    s *= scale;
    const float mn = fmaxf(m, s), a = __expf(m - mn), p = __expf(s - mn);
    m = mn;
    l = fmaf(l, a, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = fmaf(o[e], a, p * v[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  v4i w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = (int)pack_bf16_rne(o[2 * e] * inv, o[2 * e + 1] * inv);
  *reinterpret_cast<v4i*>(out + th * 512 + 8 * lane) = w;
  if (lane == 0 && lse) lse[th] = l == 0.f ? -__builtin_inff() : m + logf(l);
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_sparse_mla_decode_fp4(const void* q, int64_t q_token_stride, int64_t q_head_stride,
                                         const uint8_t* kv_cache, int64_t kv_block_stride_bytes, int kv_block_size,
                                         int64_t kv_num_blocks, const int32_t* indices, int64_t idx_stride,
                                         int num_tokens, int num_heads, int topk, float sm_scale, void* out,
                                         float* lse, int num_splits, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  using namespace dsa;
  (void)num_splits; (void)workspace; (void)workspace_bytes;
  if (num_tokens < 0 || num_heads <= 0 || (num_heads % 16) != 0)
    return set_error(kUnsupported, "sparse_mla_fp4: num_heads=%d must be a positive multiple of 16", num_heads);
  if (topk <= 0 || topk % 64 != 0)
    return set_error(kUnsupported, "sparse_mla_fp4: topk=%d must be a positive multiple of 64", topk);
  if (kv_block_size <= 0 || kv_num_blocks < 0 || kv_block_stride_bytes < (int64_t)kv_block_size * kMla4RowBytes ||
      kv_block_stride_bytes % 16)
    return set_error(kInvalidArgument, "sparse_mla_fp4: bad cache geometry");
  if (num_tokens == 0) return kOk;
  if (!q || !kv_cache || !indices || !out) return set_error(kInvalidArgument, "sparse_mla_fp4: null pointer");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kv_cache) | reinterpret_cast<uintptr_t>(out)) & 15) ||
      (q_token_stride % 8) || (q_head_stride % 8))
    return set_error(kInvalidArgument, "sparse_mla_fp4: q, kv_cache and out must be 16-byte aligned");
  if ((int64_t)num_tokens * num_heads > INT32_MAX) return set_error(kInvalidArgument, "sparse_mla_fp4: grid too large");
  hipLaunchKernelGGL(sparse_mla_fp4_kernel, dim3((unsigned)(num_tokens * num_heads)), dim3(64), 0, (hipStream_t)stream,
                     static_cast<const uint16_t*>(q), q_token_stride, q_head_stride, kv_cache, kv_block_stride_bytes,
                     kv_block_size, kv_num_blocks, indices, idx_stride, num_heads, topk, sm_scale,
                     static_cast<uint16_t*>(out), lse);
  return check_launch("dsa_sparse_mla_decode_fp4");
}
