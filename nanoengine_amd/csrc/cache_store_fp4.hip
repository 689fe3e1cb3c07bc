// Writers and readers of the 4-bit DSA caches (format: fp4.h), for gfx950.
//
// A lane holds eight consecutive dims (one 16-byte load of bf16), so a block of 32
// is four neighbouring lanes and its largest magnitude two shuffles; a lane's eight
// codes are one 4-byte store. An MLA row is one wave (64 lanes x 8 dims), an indexer
// key 16 lanes, four keys to a wave. What bounds both directions is the launch for a
// decode batch and the bytes for a prefill chunk: 128 MLA rows stored in 2.9 us and read
// back in 2.7, 8192 in 5.2 and 4.9 (12.7 MB each way, 2.5 TB/s with the launch in it);
// 33 indexer keys 2.0 and 1.9 us, 8192 of them 2.9 and 2.9 (2.7 MB).
#include "dsa_common.h"
#include "fp4.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

constexpr int kStoreThreads = 256;

__device__ __forceinline__ int64_t slot_at(const void* slots, int slot_is_64, int64_t i) {
  return slot_is_64 ? static_cast<const int64_t*>(slots)[i] : (int64_t)static_cast<const int32_t*>(slots)[i];
}

__global__ void __launch_bounds__(kStoreThreads)
mla_kv_store_fp4_kernel(const uint16_t* __restrict__ kv, int64_t row_stride, const void* __restrict__ slots,
                        int slot_is_64, int n, uint8_t* __restrict__ cache, int64_t block_stride, int block_size,
                        int64_t num_blocks) {
  const int lane = threadIdx.x & 63;
  const int tok = blockIdx.x * (kStoreThreads / 64) + (threadIdx.x >> 6);
  if (tok >= n) return;
  const int64_t slot = slot_at(slots, slot_is_64, tok);
  if (slot < 0 || slot / block_size >= num_blocks) return;
  const uint16_t* src = kv + (int64_t)tok * row_stride;
  uint8_t* row = cache + (slot / block_size) * block_stride + (slot % block_size) * kMla4RowBytes;
  float x[8];
  bf16x8_to_f32(*reinterpret_cast<const v4i*>(src + 8 * lane), x);
  int byte;
  const uint32_t codes = fp4_quantise_block(x, &byte);
  *reinterpret_cast<uint32_t*>(row + 4 * lane) = codes;
  if ((lane & 3) == 0) row[kMla4ScaleOff + (lane >> 2)] = (uint8_t)byte;
  if (lane < 8)
    *reinterpret_cast<v4i*>(row + kMla4RopeOff + 16 * lane) = *reinterpret_cast<const v4i*>(src + 512 + 8 * lane);
}

__global__ void __launch_bounds__(kStoreThreads)
mla_kv_load_fp4_kernel(const uint8_t* __restrict__ cache, int64_t block_stride, int block_size, int64_t num_blocks,
                       const void* __restrict__ slots, int slot_is_64, int n, uint16_t* __restrict__ out,
                       int64_t out_stride) {
  const int lane = threadIdx.x & 63;
  const int tok = blockIdx.x * (kStoreThreads / 64) + (threadIdx.x >> 6);
  if (tok >= n) return;
  const int64_t slot = slot_at(slots, slot_is_64, tok);
  uint16_t* dst = out + (int64_t)tok * out_stride;
  v4i nope = {0, 0, 0, 0}, rope = {0, 0, 0, 0};
  if (slot >= 0 && slot / block_size < num_blocks) {
    const uint8_t* row = cache + (slot / block_size) * block_stride + (slot % block_size) * kMla4RowBytes;
    nope = fp4x8_to_bf16(*reinterpret_cast<const uint32_t*>(row + 4 * lane),
                         fp4_scale(row[kMla4ScaleOff + (lane >> 2)]));
    if (lane < 8) rope = *reinterpret_cast<const v4i*>(row + kMla4RopeOff + 16 * lane);
  }
  *reinterpret_cast<v4i*>(dst + 8 * lane) = nope;
  if (lane < 8) *reinterpret_cast<v4i*>(dst + 512 + 8 * lane) = rope;
}

__global__ void __launch_bounds__(kStoreThreads)
indexer_k_store_fp4_kernel(const uint16_t* __restrict__ k, int64_t row_stride, const void* __restrict__ slots,
                           int slot_is_64, int n, uint8_t* __restrict__ cache, int page_size, int64_t num_pages) {
  const int tok = blockIdx.x * (kStoreThreads / 16) + (threadIdx.x >> 4), sub = threadIdx.x & 15;
  // lanes past the last key repeat it and write nothing: a block's lanes stay together in the shuffles
  const int src_tok = min(tok, n - 1);
  const int64_t slot = slot_at(slots, slot_is_64, src_tok);
  float x[8];
  bf16x8_to_f32(*reinterpret_cast<const v4i*>(k + (int64_t)src_tok * row_stride + 8 * sub), x);
  int byte;
  const uint32_t codes = fp4_quantise_block(x, &byte);
  if (tok >= n || slot < 0 || slot / page_size >= num_pages) return;
  const int64_t off = slot % page_size;
  uint8_t* page = cache + slot / page_size * page_size * (kIdx4KeyBytes + kIdx4KeyScales);
  *reinterpret_cast<uint32_t*>(page + off * kIdx4KeyBytes + 4 * sub) = codes;
  if ((sub & 3) == 0) page[(int64_t)page_size * kIdx4KeyBytes + off * kIdx4KeyScales + (sub >> 2)] = (uint8_t)byte;
}

// fp8 keys with one f32 scale a key, the ragged prefill scorer's operand: the
// scale is 2^-6 of the key's largest block scale, so that the largest code becomes
// 6 * 2^6 of e4m3's 448. A block 2^14 or less below the largest keeps its codes
// exactly (0.5 * 2^(6-14) is 2^-9, e4m3's smallest step); further down they are
// rounded to that step, 2^-17 of the largest code. A NaN block becomes fp8 NaNs.
__global__ void __launch_bounds__(kStoreThreads)
indexer_k_load_fp4_kernel(const uint8_t* __restrict__ cache, int page_size, int64_t num_pages,
                          const void* __restrict__ slots, int slot_is_64, int n, uint8_t* __restrict__ key_out,
                          float* __restrict__ scale_out) {
  const int tok = blockIdx.x * (kStoreThreads / 16) + (threadIdx.x >> 4), sub = threadIdx.x & 15;
  if (tok >= n) return;
  const int64_t slot = slot_at(slots, slot_is_64, tok);
  uint32_t codes = 0u, bytes = 0u;
  if (slot >= 0 && slot / page_size < num_pages) {
    const int64_t off = slot % page_size;
    const uint8_t* page = cache + slot / page_size * page_size * (kIdx4KeyBytes + kIdx4KeyScales);
    codes = *reinterpret_cast<const uint32_t*>(page + off * kIdx4KeyBytes + 4 * sub);
    bytes = *reinterpret_cast<const uint32_t*>(page + (int64_t)page_size * kIdx4KeyBytes + off * kIdx4KeyScales);
  }
  int top = 7;  // a scale of 2^-126 at least
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = (int)((bytes >> (8 * i)) & 255u);
    if (b != kFp4NaN) top = max(top, b);
  }
  const int b = (int)((bytes >> (8 * (sub >> 2))) & 255u);
  // the block's scale over the key's: 2^(b - top + 6)
  const float rel = b == kFp4NaN ? fp4_scale(kFp4NaN) : fp4_scale((uint32_t)max(b - top + 6 + 127, 1));
  float x[8];
  bf16x8_to_f32(fp4x8_to_bf16(codes, rel), x);
  uint2 w;
  w.x = f32x4_to_fp8(x[0], x[1], x[2], x[3]);
  w.y = f32x4_to_fp8(x[4], x[5], x[6], x[7]);
  *reinterpret_cast<uint2*>(key_out + (int64_t)tok * 128 + 8 * sub) = w;
  if (sub == 0) scale_out[tok] = __uint_as_float((uint32_t)(top - 6) << 23);
}

dim3 store_grid(int num_tokens, int lanes_each) {
  return dim3((unsigned)((num_tokens - 1) / (kStoreThreads / lanes_each) + 1));
}

bool bad_mla_cache(int64_t stride, int block_size, int64_t num_blocks) {
  return block_size <= 0 || num_blocks < 0 || stride < (int64_t)block_size * kMla4RowBytes;
}

}  // namespace
}  // namespace dsa

extern "C" {

int dsa_mla_kv_store_fp4(const void* kv, int64_t kv_row_stride, const void* slots, int slot_is_64, int num_tokens,
                         uint8_t* kv_cache, int64_t kv_block_stride_bytes, int kv_block_size, int64_t kv_num_blocks,
                         void* stream) {
  using namespace dsa;
  if (num_tokens < 0 || bad_mla_cache(kv_block_stride_bytes, kv_block_size, kv_num_blocks))
    return set_error(kInvalidArgument, "dsa_mla_kv_store_fp4: bad sizes");
  if (num_tokens == 0) return kOk;
  if (!kv || !slots || !kv_cache) return set_error(kInvalidArgument, "dsa_mla_kv_store_fp4: null pointer");
  if (((reinterpret_cast<uintptr_t>(kv) | reinterpret_cast<uintptr_t>(kv_cache)) & 15) || (kv_row_stride & 7) ||
      (kv_block_stride_bytes & 15))
    return set_error(kInvalidArgument, "dsa_mla_kv_store_fp4: kv and cache rows must be 16-byte aligned");
  hipLaunchKernelGGL(mla_kv_store_fp4_kernel, store_grid(num_tokens, 64), dim3(kStoreThreads), 0, (hipStream_t)stream,
                     static_cast<const uint16_t*>(kv), kv_row_stride, slots, slot_is_64, num_tokens, kv_cache,
                     kv_block_stride_bytes, kv_block_size, kv_num_blocks);
  return check_launch("dsa_mla_kv_store_fp4");
}

int dsa_mla_kv_load_fp4(const uint8_t* kv_cache, int64_t kv_block_stride_bytes, int kv_block_size,
                        int64_t kv_num_blocks, const void* slots, int slot_is_64, int num_tokens, void* out,
                        int64_t out_row_stride, void* stream) {
  using namespace dsa;
  if (num_tokens < 0 || out_row_stride < 576 || bad_mla_cache(kv_block_stride_bytes, kv_block_size, kv_num_blocks))
    return set_error(kInvalidArgument, "dsa_mla_kv_load_fp4: bad sizes");
  if (num_tokens == 0) return kOk;
  if (!out || !slots || !kv_cache) return set_error(kInvalidArgument, "dsa_mla_kv_load_fp4: null pointer");
  if (((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(kv_cache)) & 15) || (out_row_stride & 7) ||
      (kv_block_stride_bytes & 15))
    return set_error(kInvalidArgument, "dsa_mla_kv_load_fp4: output and cache rows must be 16-byte aligned");
  hipLaunchKernelGGL(mla_kv_load_fp4_kernel, store_grid(num_tokens, 64), dim3(kStoreThreads), 0, (hipStream_t)stream, kv_cache,
                     kv_block_stride_bytes, kv_block_size, kv_num_blocks, slots, slot_is_64, num_tokens,
                     static_cast<uint16_t*>(out), out_row_stride);
  return check_launch("dsa_mla_kv_load_fp4");
}

int dsa_indexer_k_store_fp4(const void* k, int64_t k_row_stride, const void* slots, int slot_is_64, int num_tokens,
                            uint8_t* cache, int page_size, int64_t num_pages, void* stream) {
  using namespace dsa;
  if (num_tokens < 0 || page_size <= 0 || num_pages < 0)
    return set_error(kInvalidArgument, "dsa_indexer_k_store_fp4: bad sizes");
  if (num_tokens == 0) return kOk;
  if (!k || !slots || !cache) return set_error(kInvalidArgument, "dsa_indexer_k_store_fp4: null pointer");
  if ((reinterpret_cast<uintptr_t>(k) & 15) || (k_row_stride & 7) || (reinterpret_cast<uintptr_t>(cache) & 3))
    return set_error(kInvalidArgument, "dsa_indexer_k_store_fp4: keys must be 16-byte aligned, the cache 4-byte");
  hipLaunchKernelGGL(indexer_k_store_fp4_kernel, store_grid(num_tokens, 16), dim3(kStoreThreads), 0, (hipStream_t)stream,
                     static_cast<const uint16_t*>(k), k_row_stride, slots, slot_is_64, num_tokens, cache, page_size,
                     num_pages);
  return check_launch("dsa_indexer_k_store_fp4");
}

int dsa_indexer_k_load_fp4(const uint8_t* cache, int page_size, int64_t num_pages, const void* slots, int slot_is_64,
                           int num_tokens, uint8_t* key_out, float* scale_out, void* stream) {
  using namespace dsa;
  if (num_tokens < 0 || page_size <= 0 || num_pages < 0)
    return set_error(kInvalidArgument, "dsa_indexer_k_load_fp4: bad sizes");
  if (num_tokens == 0) return kOk;
  if (!key_out || !scale_out || !slots || !cache)
    return set_error(kInvalidArgument, "dsa_indexer_k_load_fp4: null pointer");
  if ((reinterpret_cast<uintptr_t>(cache) & 3) || (reinterpret_cast<uintptr_t>(key_out) & 7))
    return set_error(kInvalidArgument, "dsa_indexer_k_load_fp4: keys must be 8-byte aligned, the cache 4-byte");
  hipLaunchKernelGGL(indexer_k_load_fp4_kernel, store_grid(num_tokens, 16), dim3(kStoreThreads), 0, (hipStream_t)stream, cache,
                     page_size, num_pages, slots, slot_is_64, num_tokens, key_out, scale_out);
  return check_launch("dsa_indexer_k_load_fp4");
}

}  // extern "C"
