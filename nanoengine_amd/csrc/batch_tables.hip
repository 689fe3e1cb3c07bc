// Block tables and slot maps of a batch from its requests' lengths, for gfx950.
//
// Request b holds c_b cached tokens and adds n_b. With pages of P tokens it owns
// old_b = ceil(c_b / P) blocks and takes need_b = ceil((c_b + n_b) / P) - old_b more,
// from the free list in request order:
//   block_tables[b, old_b + i] = free[head + sum_{a<b} need_a + i]
// Its new token j is row r = sum_{a<b} n_a + j of the batch, at position c_b + j, in
//   slot = block_tables[b, pos / P] * P + pos % P.
// Every workgroup takes 256 rows, one a thread, and forms both prefix sums of the whole
// batch for itself in LDS (a batch is a few KB of lengths in L2), so that one launch
// does without any exchange between workgroups: a row of a fresh page takes its block
// from the free list, not from the table entry that another workgroup may be writing.
// A fresh page starts with its first new token, whose row writes the table entry.
// The call is bound by its launch and three dependent reads (lengths, free list or table,
// and the search for the row's request between them), not by its bytes: 4 requests
// 4.1 us from a graph, 64 of two tokens 4.5, 96 with 131072 new tokens 5.1 (33 keys
// stored and read back, two launches: 3.9).
#include "dsa_common.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

constexpr int kTabThreads = 256;
constexpr int kTabWaves = kTabThreads / 64;
constexpr int kTabMaxBatch = 8192;  // three arrays of 4 bytes a request in LDS

struct TabParams {
  const int32_t *cached, *added;
  int batch;
  int32_t* tables;
  int64_t bt_stride;
  int bt_width, page_size;
  int page_shift;              // log2(page_size), or -1
  const int32_t* free_blocks;  // null: the tables hold the new pages already
  int64_t num_free;
  const int32_t* free_head;    // null: 0
  void* slots;
  int slots_64;
  void* positions;  // may be null
  int pos_64;
  int32_t* seq_lens;  // may be null
  int64_t rows;
  void *cu_q, *cu_k;  // may be null
  int cu_64;
  int64_t* status;
};

enum Fault : int { kBadLength = 1, kTableNarrow = 2, kFreeShort = 4, kRowsShort = 8, kCuOverflow = 16 };

__device__ __forceinline__ void put(void* p, int is_64, int64_t i, int64_t v) {
  if (is_64) static_cast<int64_t*>(p)[i] = v;
  else static_cast<int32_t*>(p)[i] = (int32_t)v;
}

// (tokens and page size are below 2^31, so that 32 bits hold their sum)
__device__ __forceinline__ uint32_t page_at(const TabParams& P, uint32_t pos) {
  return P.page_shift >= 0 ? pos >> P.page_shift : pos / (uint32_t)P.page_size;
}
__device__ __forceinline__ uint32_t pages_of(const TabParams& P, int64_t tokens) {
  return page_at(P, (uint32_t)tokens + (uint32_t)P.page_size - 1u);
}

__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {  // inclusive
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t x = __shfl_up(v, off, 64);
    if (lane >= off) v += x;
  }
  return v;
}

// kPer: consecutive requests a thread sums by itself before the workgroup's scan.
template <int kPer>
__global__ void __launch_bounds__(kTabThreads) batch_tables_kernel(const TabParams P) {
  extern __shared__ __align__(16) uint32_t tab_smem[];
  __shared__ int64_t wsum[3][kTabWaves];
  __shared__ int s_fault[kTabWaves];
  __shared__ int64_t s_longest[kTabWaves];
  // per request: its first row and its first free-list entry, each at most 2^32 - 1, which is past every
  // row and free-list entry there is; its cached tokens
  uint32_t *row0 = tab_smem, *take0 = row0 + P.batch, *cached = take0 + P.batch;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool first_wg = blockIdx.x == 0;

  int64_t rows_before = 0, take_before = 0, keys_before = 0, longest = 0;
  int fault = 0;
  if (first_wg && threadIdx.x == 0) {
    if (P.cu_q) put(P.cu_q, P.cu_64, 0, 0);
    if (P.cu_k) put(P.cu_k, P.cu_64, 0, 0);
  }
  for (int base = 0; base < P.batch; base += kTabThreads * kPer) {
    const int b0 = base + (int)threadIdx.x * kPer;
    int64_t c[kPer], n[kPer];
    uint32_t need[kPer];
    int64_t sum[3] = {0, 0, 0};  // rows, blocks taken, keys
#pragma unroll
    for (int i = 0; i < kPer; ++i) {  // (without conditions: all loads go out at once)
      const int b = min(b0 + i, P.batch - 1);
      c[i] = P.cached[b];
      n[i] = P.added[b];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      need[i] = 0u;
      // a negative length, or a total past int32, makes the request empty
      const bool ok = c[i] >= 0 && n[i] >= 0 && c[i] + n[i] <= INT32_MAX;
      if (b0 + i < P.batch && !ok) fault |= kBadLength;
      if (b0 + i >= P.batch || !ok) c[i] = n[i] = 0;
      const uint32_t total = pages_of(P, c[i] + n[i]);
      if (P.free_blocks) need[i] = total - pages_of(P, c[i]);
      if (total > (uint32_t)P.bt_width && n[i] > 0) fault |= kTableNarrow;
      longest = max(longest, c[i] + n[i]);
      sum[0] += n[i];
      sum[1] += need[i];
      sum[2] += c[i] + n[i];
    }
    int64_t at[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int64_t incl = wave_scan(sum[k], lane);
      at[k] = incl - sum[k];
      if (lane == 63) wsum[k][wave] = incl;
    }
    __syncthreads();
    at[0] += rows_before;
    at[1] += take_before;
    at[2] += keys_before;
#pragma unroll
    for (int w = 0; w < kTabWaves; ++w) {
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (w < wave) at[k] += wsum[k][w];
      rows_before += wsum[0][w];
      take_before += wsum[1][w];
      keys_before += wsum[2][w];
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (b0 + i >= P.batch) break;
      row0[b0 + i] = (uint32_t)min(at[0], (int64_t)UINT32_MAX);
      take0[b0 + i] = (uint32_t)min(at[1], (int64_t)UINT32_MAX);
      cached[b0 + i] = (uint32_t)c[i];
      at[0] += n[i];
      at[1] += need[i];
      at[2] += c[i] + n[i];
      if (first_wg) {
        // an int32 total that does not fit is stored as the largest one, with its fault bit
        const int64_t most = P.cu_64 ? INT64_MAX : INT32_MAX;
        if (P.cu_q) put(P.cu_q, P.cu_64, b0 + i + 1, min(at[0], most));
        if (P.cu_k) put(P.cu_k, P.cu_64, b0 + i + 1, min(at[2], most));
      }
    }
    __syncthreads();
  }
  const int64_t head = P.free_head ? (int64_t)*P.free_head : 0;
  if (first_wg) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      fault |= __shfl_xor(fault, off, 64);
      longest = max(longest, (int64_t)__shfl_xor(longest, off, 64));
    }
    if (lane == 0) {
      s_fault[wave] = fault;
      s_longest[wave] = longest;
    }
  }
  __syncthreads();
  if (first_wg && threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kTabWaves; ++w) {
      fault |= s_fault[w];
      longest = max(longest, s_longest[w]);
    }
    if (take_before > 0 && (head < 0 || head + take_before > P.num_free)) fault |= kFreeShort;
    if (rows_before > P.rows) fault |= kRowsShort;
    if (!P.cu_64 && ((P.cu_q && rows_before > INT32_MAX) || (P.cu_k && keys_before > INT32_MAX))) fault |= kCuOverflow;
    P.status[0] = fault;
    P.status[1] = rows_before;
    P.status[2] = take_before;
    P.status[3] = longest;
  }

  const int64_t r = (int64_t)blockIdx.x * kTabThreads + threadIdx.x;
  if (r < P.rows) {
    int64_t slot = -1;
    uint32_t pos = 0, len = 0;
    if (r < rows_before) {
      int lo = 0, hi = P.batch - 1;  // last request whose first row is <= r: the one that has rows there
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (row0[mid] <= (uint32_t)r) lo = mid; else hi = mid - 1;
      }
      pos = cached[lo] + (uint32_t)r - row0[lo];
      len = pos + 1;
      const uint32_t page = page_at(P, pos), off = pos - page * (uint32_t)P.page_size;
      const uint32_t old = pages_of(P, cached[lo]);
      int64_t block = -1;
      if (page < (uint32_t)P.bt_width) {
        int32_t* entry = P.tables + lo * P.bt_stride + page;
        if (!P.free_blocks || page < old) {
          block = *entry;
        } else {
          const int64_t f = head + take0[lo] + (page - old);
          if (f >= 0 && f < P.num_free) {
            block = P.free_blocks[f];
            if (off == 0) *entry = (int32_t)block;
          }
        }
      }
      if (block >= 0) slot = block * P.page_size + off;
      if (!P.slots_64 && slot > INT32_MAX) slot = -1;
    }
    put(P.slots, P.slots_64, r, slot);
    if (P.positions) put(P.positions, P.pos_64, r, pos);
    if (P.seq_lens) P.seq_lens[r] = (int32_t)len;
  }
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_batch_tables(const int32_t* cached_lens, const int32_t* new_lens, int batch, int32_t* block_tables,
                                int64_t bt_stride, int bt_width, int page_size, const int32_t* free_blocks,
                                int64_t num_free, const int32_t* free_head, void* slots, int slots_are_64,
                                void* positions, int positions_are_64, int32_t* seq_lens, int64_t num_rows,
                                void* cu_seqlens_q, void* cu_seqlens_k, int cu_is_64, int64_t* status, void* stream) {
  using namespace dsa;
  if (batch < 0 || page_size <= 0 || bt_width < 0 || bt_stride < bt_width || num_free < 0 || num_rows < 0)
    return set_error(kInvalidArgument, "dsa_batch_tables: bad sizes");
  if (batch > kTabMaxBatch)
    return set_error(kUnsupported, "dsa_batch_tables: batch=%d (at most %d requests)", batch, kTabMaxBatch);
  if (num_free > INT32_MAX || num_rows > INT32_MAX)
    return set_error(kUnsupported, "dsa_batch_tables: more than 2^31 - 1 rows or free blocks");
  if (!status || (batch > 0 && (!cached_lens || !new_lens || !block_tables)) || (num_rows > 0 && !slots))
    return set_error(kInvalidArgument, "dsa_batch_tables: null pointer");
  // One row a thread: a row's reads depend on each other, and four rows in turn took
  // four times their latency (131072 rows of 96 requests: 9.3 us, now 5.2), although
  // every workgroup forms the prefix sums (128 requests 4.7 us, 1000 6.6, 4000 15.3).
  const int64_t nwg = num_rows > 0 ? (num_rows - 1) / kTabThreads + 1 : 1;
  const int shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
  const TabParams P{cached_lens, new_lens, batch, block_tables, bt_stride, bt_width, page_size, shift, free_blocks,
                    num_free, free_head, slots, slots_are_64, positions, positions_are_64, seq_lens, num_rows,
                    cu_seqlens_q, cu_seqlens_k, cu_is_64, status};
  const size_t smem = 3 * (size_t)batch * sizeof(uint32_t);
  // 4000 requests of two tokens: 27.7 us with one request a thread, 15.3 with four or eight; 300: 6.3 and 7.9
  const auto kernel = batch <= kTabThreads ? batch_tables_kernel<1> : batch_tables_kernel<4>;
  if (smem > 32 * 1024 && hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                              (int)smem) != hipSuccess)
    return set_error(kLaunchFailed, "dsa_batch_tables: cannot reserve %zu B of LDS", smem);
  hipLaunchKernelGGL(kernel, dim3((unsigned)nwg), dim3(kTabThreads), smem, (hipStream_t)stream, P);
  return check_launch("dsa_batch_tables");
}
