// Lightning-indexer logits over a 4-bit paged key cache (format: fp4.h), for gfx950.
//
//   logits[b*n+j, t] = sum_h w[b*n+j, h] * relu(q[b,j,h,:] . k[t,:])
//
// A page of 64 keys is 4352 bytes against the 8448 of fp8 pages, 240 flop to the
// byte. The products run on bf16 MFMAs, exact with f32 sums: the block-scaled MFMA
// would take the codes as they are, but keeps only ~13 bits below the largest of its
// products.
// What bounds it: 128 rows of 65536 positions take 140 to 148 us from a graph, by the
// card (570 MB read, 34 MB written: 4.2 TB/s; 0.95 PFLOP/s at 144). Where they took 140, the
// same loop without its products took 120 us, without the ReLU and weights 127, the
// page loads and score stores alone 113, the loads alone 87: the reads share HBM with
// the score stores, and the products run at the clock (1.8 GHz) that their power
// leaves. Two query tokens (64 rows of 30000: 63 us, 0.99 PFLOP/s) are bound by the
// products.
//
// Persistent kernel, one workgroup of 8 waves per CU; every wave owns one contiguous
// range of the flattened (batch entry, page) space and no barrier after the start.
//   pages : straight from HBM into the wave's two page buffers in LDS, one page
//           ahead, 1 KB of whole 64-byte keys to an instruction. Lane l's source
//           piece is swizzled so that 16 consecutive keys' reads of one block fall
//           on all banks. (Three and four buffers, three waves a SIMD, and pages dealt
//           out one by one to the waves of a workgroup all take the same time.)
//   keys  : the B operand of v_mfma_f32_32x32x16_bf16. Lane (c32, h) reads 16 bytes
//           of codes, one 32-dim block with one scale: dims 64c + 32h .. +31 of key c32 of
//           a 32-key tile, converted eight at a time into the operands of four k-steps.
//   query : the A operand, 64 heads in the same order of dims, resident in registers
//           with the head weights.
//   order : the sums of one eight-product unit stand between the products of the
//           next (150 -> 141 us).
//   sum   : a lane ends up with 32 of a key's 64 heads; the lane halves' sums of the
//           two key tiles change places in one swap, so that lane t holds key t.
#include <algorithm>

#include "dsa_common.h"
#include "fp4.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kPage = 64, kDim = 128, kHeads = 64;
constexpr int kCodeBytes = kPage * kIdx4KeyBytes;                        // 4096
constexpr int kPageBytes4 = kPage * (kIdx4KeyBytes + kIdx4KeyScales);    // 4352
constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kBufs = 2;            // page buffers a wave: one page in flight, one multiplied
constexpr int kPageLoads = 5;       // instructions of a page: 4 x 1 KB of codes, the scales
constexpr int kAdvance = 62;        // pages per refill of a wave's 64 block-table entries
constexpr int kMaxBatch = 4096;     // entries of a launch (their page prefix lies in LDS)
constexpr int kFillChunk = 1024;    // positions past a row's pages that a wave fills at a time
constexpr int kWeightBytes = 2 * kHeads * sizeof(float);  // a wave's head weights (two query tokens only)
constexpr size_t smem_bytes(int next_n, int batch) {
  return (size_t)kWaves * (kBufs * kPageBytes4 + (next_n == 2 ? kWeightBytes : 0)) +
         ((size_t)batch + 1 + kWaves) * sizeof(int32_t);
}
static_assert(smem_bytes(2, kMaxBatch) <= 160 * 1024, "LDS budget");
static_assert(kAdvance + kBufs - 1 < 64, "window refill geometry");

// Source of a page outside the cache (its scores are replaced by -inf).
__device__ __align__(16) uint8_t g_idx4_zero_page[kPageBytes4];

struct Idx4Params {
  const uint8_t *q, *kv;
  int64_t num_pages;
  const float* weights;
  const int32_t *ctx, *bt;
  int64_t bt_stride;
  int batch;
  int64_t max_ctx;
  float* logits;
  int64_t stride;
  int clean;
};

// A page into LDS at `lds` (wave-uniform). The immediate offset moves both addresses.
__device__ __forceinline__ void load_page4(const uint8_t* page, uint32_t lds, uint32_t lane_off, uint32_t lane4) {
  asm volatile("s_waitcnt lgkmcnt(0)\n\t"
               "global_load_lds_dwordx4 %0, %1 nt\n\tglobal_load_lds_dwordx4 %0, %1 offset:%3 nt\n\t"
               "global_load_lds_dwordx4 %0, %1 offset:%4 nt\n\tglobal_load_lds_dwordx4 %0, %1 offset:%5 nt"
               ::"v"(lane_off), "s"(page), "{m0}"(lds), "n"(1024), "n"(2 * 1024), "n"(3 * 1024) : "memory");
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, %1 nt"
               ::"v"(lane4), "s"(page + kCodeBytes), "{m0}"(lds + kCodeBytes) : "memory");
}

// max(x, 0), NaN for a NaN
__device__ __forceinline__ float relu_nan(float x) { return __builtin_elementwise_maximum(x, 0.f); }

template <int NQ>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2)))
indexer_logits_fp4_kernel(const Idx4Params P) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int h = lane >> 5, c32 = lane & 31;
  uint8_t* ring = smem + wave * kBufs * kPageBytes4;
  // two query tokens' operands leave no registers for their head weights
  constexpr bool kWLds = NQ == 2;
  float* wl = reinterpret_cast<float*>(smem + kWaves * kBufs * kPageBytes4 + wave * kWeightBytes);
  int32_t* prefix =
      reinterpret_cast<int32_t*>(smem + kWaves * (kBufs * kPageBytes4 + (kWLds ? kWeightBytes : 0)));  // [batch + 1]
  int32_t* wsum = prefix + P.batch + 1;                                                                // [kWaves]

  // pages of each batch entry (the longest of its query tokens) -> exclusive prefix
  int32_t carry = 0;
  for (int base = 0; base < P.batch; base += kThreads) {
    const int i = base + (int)threadIdx.x;
    int np = 0;
    if (i < P.batch) {
      int lm = 0;
#pragma unroll
      for (int j = 0; j < NQ; ++j) lm = max(lm, P.ctx[i * NQ + j]);
      np = (int)((min((int64_t)lm, P.max_ctx) + kPage - 1) / kPage);
    }
    int v = np;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(v, off, 64);
      if (lane >= off) v += x;
    }
    if (lane == 63) wsum[wave] = v;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w2 = 0; w2 < kWaves; ++w2) {
      if (w2 < wave) before += wsum[w2];
      carry += wsum[w2];
    }
    if (i < P.batch) prefix[i] = before + v - np;
    __syncthreads();
  }
  if (threadIdx.x == 0) prefix[P.batch] = carry;
  __syncthreads();

  const int64_t total = carry;
  const int64_t nwaves = (int64_t)gridDim.x * kWaves, gw = (int64_t)blockIdx.x * kWaves + wave;

  // this wave's range of the flattened pages
  const int64_t p0 = total * gw / nwaves, p1 = total * (gw + 1) / nwaves;
  const int n = (int)(p1 - p0);

  // block-table window: lane l holds page p0 + wb + l as (batch entry, cache page)
  int wb = 0, win_b = 0, win_page = -1;
  auto refill = [&](int from) {
    const int64_t p = p0 + from + lane;
    int bl = 0, page = -1;
    if (p < p1) {
      int lo = 0, hi = P.batch - 1;  // last batch entry with prefix <= p: the one whose pages hold p
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= p) lo = mid; else hi = mid - 1;
      }
      bl = lo;
      page = P.bt[(int64_t)bl * P.bt_stride + (p - prefix[bl])];
    }
    // the load's wait belongs here: left to the first use, it stands in the page loop and drains the
    // pages in flight at every turn
    asm volatile("" : "+v"(page));
    win_b = bl;
    win_page = page;
  };
  if (n > 0) refill(0);

  const uint32_t lane_off = 64u * (lane >> 2) + 16u * ((lane & 3) ^ (lane >> 4));
  auto issue = [&](int k) {
    const int page = __builtin_amdgcn_readlane(win_page, k - wb);
    const uint8_t* src = page >= 0 && page < P.num_pages ? P.kv + (int64_t)page * kPageBytes4 : g_idx4_zero_page;
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(ring + (k % kBufs) * kPageBytes4);
    load_page4(src, __builtin_amdgcn_readfirstlane(lds), lane_off, 4u * lane);
  };

  // the current batch entry: query operands (k-step 4c + j of head tile ht: dims 64c + 32h + 8j .. +7
  // of head 32ht + c32), head weights of the accumulator's rows, lengths
  v8bf qa[NQ][2][8];
  float w[2][16];  // NQ == 1
  int L[NQ];
  auto enter = [&](int b) {
    // (lane ids that the compiler cannot see through keep the address arithmetic here, not in registers
    // across the loop)
    int c32_o = c32, h_o = h;
    asm volatile("" : "+v"(c32_o), "+v"(h_o));
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int64_t row = (int64_t)b * NQ + j;
#pragma unroll
      for (int ht = 0; ht < 2; ++ht) {
        const uint8_t* qh = P.q + (row * kHeads + 32 * ht + c32_o) * kDim + 32 * h_o;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const v4i raw = *reinterpret_cast<const v4i*>(qh + 64 * c + 16 * u);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int lo = raw[2 * e], hi = raw[2 * e + 1];
              const v4i op = {__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
                              __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
                              __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
                              __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
              qa[j][ht][4 * c + 2 * u + e] = __builtin_bit_cast(v8bf, op);
            }
          }
#pragma unroll
        for (int r = 0; r < 16 && !kWLds; ++r)
          w[ht][r] = P.weights[row * kHeads + 32 * ht + 8 * (r >> 2) + 4 * h_o + (r & 3)];
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kWLds) wl[j * kHeads + lane] = P.weights[row * kHeads + lane];
      L[j] = (int)min((int64_t)P.ctx[row], P.max_ctx);
    }
  };

  auto compute = [&](int k, int b, int64_t first) {
    const int page = __builtin_amdgcn_readlane(win_page, k - wb);
    const uint8_t* buf = ring + (k % kBufs) * kPageBytes4;
    int c32_o = c32;
    asm volatile("" : "+v"(c32_o));
    // A unit is the eight products of one key tile, query token and head tile. Between its products stand
    // the sum of the unit before and the next tile's conversions: with products and vector work in turns, the
    // SIMD's two waves covered each other's only by chance.
    float part[NQ][2];
    v16f acc[2];
    auto read_key = [&](int tt, v4i (&raw)[2], uint32_t& sb) {
      const int key = 32 * tt + c32_o;
      sb = *reinterpret_cast<const uint32_t*>(buf + kCodeBytes + 4 * key) >> (8 * h);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        raw[c] = *reinterpret_cast<const v4i*>(buf + 64 * key + 16 * ((2 * c + h) ^ ((key >> 2) & 3)));
    };
    auto convert = [&](v8bf (&kb)[8], const v4i (&raw)[2], uint32_t sb, int c) {
      const float sc = fp4_scale((sb >> (16 * c)) & 255u);
#pragma unroll
      for (int i = 0; i < 4; ++i) kb[4 * c + i] = __builtin_bit_cast(v8bf, fp4x8_to_bf16((uint32_t)raw[c][i], sc));
    };
    auto products = [&](v16f& c, const v8bf (&q8)[8], const v8bf (&kb)[8]) {
#pragma unroll
      for (int r = 0; r < 16; ++r) c[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q8[ks], kb[ks], c, 0, 0, 0);
    };
    auto weigh = [&](const v16f& c, int j, int ht) {
      float a = 0.f, b2 = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        v4f wv;
        if constexpr (kWLds) wv = *reinterpret_cast<const v4f*>(wl + j * kHeads + 32 * ht + 8 * g + 4 * h);
        else wv = v4f{w[ht][4 * g], w[ht][4 * g + 1], w[ht][4 * g + 2], w[ht][4 * g + 3]};
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          a = fmaf(wv[r], relu_nan(c[4 * g + r]), a);
          b2 = fmaf(wv[r + 1], relu_nan(c[4 * g + r + 1]), b2);
        }
      }
      return a + b2;
    };
    auto spread = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // one MFMA
        __builtin_amdgcn_sched_group_barrier(0x2, 6, 0);  // up to six vector operations
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    if constexpr (NQ == 1) {
      v4i raw[2][2];
      uint32_t sb[2];
      read_key(0, raw[0], sb[0]);
      read_key(1, raw[1], sb[1]);
      v8bf kb[2][8];
      convert(kb[0], raw[0], sb[0], 0);
      convert(kb[0], raw[0], sb[0], 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // tile u / 2, head tile u % 2
        products(acc[u & 1], qa[0][u & 1], kb[u >> 1]);
        if (u < 2) convert(kb[1], raw[1], sb[1], u);
        if (u == 1) part[0][0] = weigh(acc[0], 0, 0);
        if (u == 2) part[0][0] += weigh(acc[1], 0, 1);
        if (u == 3) part[0][1] = weigh(acc[0], 0, 0);
        spread();
      }
      part[0][1] += weigh(acc[1], 0, 1);
    } else {
      // a loop over the tiles: unrolled, the second one's operands would take the registers of the first's
#pragma unroll 1
      for (int tt = 0; tt < 2; ++tt) {
        v4i raw[2];
        uint32_t sb;
        read_key(tt, raw, sb);
        v8bf kb[8];
        convert(kb, raw, sb, 0);
        convert(kb, raw, sb, 1);
        __builtin_amdgcn_sched_barrier(0);
        float sum[NQ];
#pragma unroll
        for (int u = 0; u < 2 * NQ; ++u) {  // query token u / 2, head tile u % 2
          products(acc[u & 1], qa[u >> 1][u & 1], kb);
          if (u > 0) {
            const float x = weigh(acc[(u - 1) & 1], (u - 1) >> 1, (u - 1) & 1);
            sum[(u - 1) >> 1] = (u - 1) & 1 ? sum[(u - 1) >> 1] + x : x;
          }
          spread();
        }
        sum[NQ - 1] += weigh(acc[1], NQ - 1, 1);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          if (tt == 0) part[j][0] = sum[j];
          else part[j][1] = sum[j];
        }
      }
    }
    const int64_t t = (p0 + k - first) * kPage + lane;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      // lane halves: {tile 0 of both, tile 1 of both}
      const auto sw =
          __builtin_amdgcn_permlane32_swap(__float_as_uint(part[j][0]), __float_as_uint(part[j][1]), false, false);
      const float v = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
      const bool ok = t < L[j] && page >= 0 && page < P.num_pages;
      // one store a page and query token, whatever the length: the waits below count it
      if (t < P.max_ctx) P.logits[((int64_t)b * NQ + j) * P.stride + t] = ok ? v : -__builtin_inff();
    }
  };

  if (n > 0) issue(0);
  // entry by entry, so that the query's registers are the inner loop's constants
  for (int k = 0; k < n;) {
    const int b = __builtin_amdgcn_readlane(win_b, k - wb);
    const int first = __builtin_amdgcn_readfirstlane(prefix[b]);
    const int k_end = (int)min((int64_t)n, __builtin_amdgcn_readfirstlane(prefix[b + 1]) - p0);
    enter(b);
    for (; k < k_end; ++k) {
      // Page k has landed when no more is outstanding than what was issued after it:
      // the loads of page k + 1 and, but for the first page, the stores of page k - 1
      // (all return in order; whatever else the compiler put between only waits longer).
      if (k + 1 < n) {
        issue(k + 1);
        if (k == 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPageLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPageLoads + NQ) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      }
      compute(k, b, first);
      if (k + 1 - wb == kAdvance) {
        // the pages loaded ahead came from this window's last lanes
        wb += kAdvance;
        refill(wb);
      }
    }
  }

  // positions past the rows' pages, after the pages: the waits above would wait for these stores too
  if (P.clean) {
    const int64_t chunks = (P.max_ctx + kFillChunk - 1) / kFillChunk, tasks = (int64_t)P.batch * chunks;
    for (int64_t i = gw; i < tasks; i += nwaves) {
      const int b = (int)(i / chunks);
      const int64_t at = (i - b * chunks) * kFillChunk;
      const int64_t begin = max(at, (int64_t)(prefix[b + 1] - prefix[b]) * kPage);
      const int64_t end = min(at + kFillChunk, P.max_ctx);
#pragma unroll
      for (int j = 0; j < NQ; ++j)
        for (int64_t t = begin + lane; t < end; t += 64)
          P.logits[((int64_t)b * NQ + j) * P.stride + t] = -__builtin_inff();
    }
  }
}

int grid_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) {
    (void)hipGetLastError();
    return 256;
  }
  return cus;
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
  if (batch < 0 || max_context_len < 0 || num_pages < 0 || logits_stride < max_context_len ||
      max_context_len > INT32_MAX)
    return set_error(kInvalidArgument, "indexer_fp4: bad sizes");
  if (batch == 0 || max_context_len == 0) return kOk;
  if (!q_fp8 || !kv_cache || !weights || !context_lens || !block_tables || !logits)
    return set_error(kInvalidArgument, "indexer_fp4: null pointer");
  if ((reinterpret_cast<uintptr_t>(q_fp8) | reinterpret_cast<uintptr_t>(kv_cache)) & 15)
    return set_error(kInvalidArgument, "indexer_fp4: q and kv_cache must be 16-byte aligned");
  const auto kernel = next_n == 1 ? indexer_logits_fp4_kernel<1> : indexer_logits_fp4_kernel<2>;
  if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                          (int)smem_bytes(next_n, kMaxBatch)) != hipSuccess)
    return set_error(kLaunchFailed, "indexer_fp4: cannot reserve %zu B of LDS", smem_bytes(next_n, kMaxBatch));
  const int cus = grid_cus();
  // entries of one launch: their page prefix fits LDS and 32 bits
  const int64_t max_pages = (max_context_len + kPage - 1) / kPage;
  const int most = (int)std::min<int64_t>(kMaxBatch, INT32_MAX / max_pages);
  for (int b0 = 0; b0 < batch; b0 += most) {
    const int nb = std::min(most, batch - b0);
    const int64_t rows = (int64_t)b0 * next_n;
    const Idx4Params P{q_fp8 + rows * kHeads * kDim, kv_cache, num_pages, weights + rows * kHeads, context_lens + rows,
                       block_tables + b0 * block_table_stride, block_table_stride, nb, max_context_len,
                       logits + rows * logits_stride, logits_stride, clean_logits};
    hipLaunchKernelGGL(kernel, dim3((unsigned)cus), dim3(kThreads), smem_bytes(next_n, nb), (hipStream_t)stream, P);
    if (int rc = check_launch("dsa_indexer_logits_fp4")) return rc;
  }
  return kOk;
}
