// Block tables and slot maps of a batch from its requests' lengths, for gfx950.
//
// Request b holds c_b cached tokens and adds n_b. With pages of P tokens it owns
// old_b = ceil(c_b / P) blocks and takes need_b = ceil((c_b + n_b) / P) - old_b more,
// from the free list in request order:
//   block_tables[b, old_b + i] = free[head + sum_{a<b} need_a + i]
// Its new token j is row r = sum_{a<b} n_a + j of the batch, at position c_b + j, in
//   slot = block_tables[b, pos / P] * P + pos % P.
// Every workgroup takes kRowsPerWG rows and forms both prefix sums of the whole
// batch for itself in LDS (a batch is a few KB of lengths in L2), so that one launch
// does without any exchange between workgroups: a row of a fresh page takes its block
// from the free list, not from the table entry that another workgroup may be writing.
// A fresh page starts with its first new token, whose row writes the table entry.
// The call is bound by its launch and two dependent reads, not by its bytes.
#include "dsa_common.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

constexpr int kTabThreads = 256;
constexpr int kTabWaves = kTabThreads / 64;
constexpr int kRowsPerWG = 1024;
constexpr int kTabMaxBatch = 8192;  // two prefix arrays of 8 bytes a request within 160 KB of LDS

struct TabParams {
  const int32_t *cached, *added;
  int batch;
  int32_t* tables;
  int64_t bt_stride;
  int bt_width, page_size;
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

// Lengths of request b; a negative one, or a total past int32, makes it empty.
__device__ __forceinline__ bool request(const TabParams& P, int b, int64_t* c, int64_t* n) {
  *c = P.cached[b];
  *n = P.added[b];
  const bool ok = *c >= 0 && *n >= 0 && *c + *n <= INT32_MAX;
  if (!ok) *c = *n = 0;
  return ok;
}

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int page_size) {
  return (tokens + page_size - 1) / page_size;
}

__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {  // inclusive
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t x = __shfl_up(v, off, 64);
    if (lane >= off) v += x;
  }
  return v;
}

__global__ void __launch_bounds__(kTabThreads) batch_tables_kernel(const TabParams P) {
  extern __shared__ __align__(16) int64_t tab_smem[];
  __shared__ int64_t wsum[3][kTabWaves];
  __shared__ int s_fault[kTabWaves];
  __shared__ int64_t s_longest[kTabWaves];
  int64_t* row0 = tab_smem;               // first row of each request, [batch + 1]
  int64_t* take0 = tab_smem + P.batch + 1;  // first free-list entry of each request, [batch]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool first_wg = blockIdx.x == 0;

  int64_t rows_before = 0, take_before = 0, keys_before = 0, longest = 0;
  int fault = 0;
  if (first_wg && threadIdx.x == 0) {
    if (P.cu_q) put(P.cu_q, P.cu_64, 0, 0);
    if (P.cu_k) put(P.cu_k, P.cu_64, 0, 0);
  }
  for (int base = 0; base < P.batch; base += kTabThreads) {
    const int b = base + (int)threadIdx.x;
    int64_t c = 0, n = 0, need = 0;
    if (b < P.batch) {
      if (!request(P, b, &c, &n)) fault |= kBadLength;
      const int64_t total = pages_of(c + n, P.page_size);
      if (P.free_blocks) need = total - pages_of(c, P.page_size);
      if (total > P.bt_width && n > 0) fault |= kTableNarrow;
      longest = max(longest, c + n);
    }
    const int64_t ni = wave_scan(n, lane), qi = wave_scan(need, lane), ki = wave_scan(c + n, lane);
    if (lane == 63) {
      wsum[0][wave] = ni;
      wsum[1][wave] = qi;
      wsum[2][wave] = ki;
    }
    __syncthreads();
    int64_t at[3] = {rows_before, take_before, keys_before};
#pragma unroll
    for (int w = 0; w < kTabWaves; ++w) {
      if (w < wave) {
        at[0] += wsum[0][w];
        at[1] += wsum[1][w];
        at[2] += wsum[2][w];
      }
      rows_before += wsum[0][w];
      take_before += wsum[1][w];
      keys_before += wsum[2][w];
    }
    if (b < P.batch) {
      row0[b] = at[0] + ni - n;
      take0[b] = at[1] + qi - need;
      if (first_wg) {
        // an int32 total that does not fit is stored as the largest one, with its fault bit
        const int64_t most = P.cu_64 ? INT64_MAX : INT32_MAX;
        if (P.cu_q) put(P.cu_q, P.cu_64, b + 1, min(at[0] + ni, most));
        if (P.cu_k) put(P.cu_k, P.cu_64, b + 1, min(at[2] + ki, most));
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) row0[P.batch] = rows_before;
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

  const int64_t r_end = min(P.rows, ((int64_t)blockIdx.x + 1) * kRowsPerWG);
  for (int64_t r = (int64_t)blockIdx.x * kRowsPerWG + threadIdx.x; r < r_end; r += kTabThreads) {
    int64_t slot = -1, pos = 0, len = 0;
    if (r < rows_before) {
      int lo = 0, hi = P.batch - 1;  // last request whose first row is <= r: the one that has rows there
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (row0[mid] <= r) lo = mid; else hi = mid - 1;
      }
      int64_t c, n;
      request(P, lo, &c, &n);
      pos = c + r - row0[lo];
      len = pos + 1;
      const int64_t page = pos / P.page_size, off = pos - page * P.page_size;
      const int64_t old = pages_of(c, P.page_size);
      int64_t block = -1;
      if (page < P.bt_width) {
        int32_t* entry = P.tables + lo * P.bt_stride + page;
        if (!P.free_blocks || page < old) {
          block = *entry;
        } else {
          const int64_t f = head + take0[lo] + page - old;
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
  if (!status || (batch > 0 && (!cached_lens || !new_lens || !block_tables)) || (num_rows > 0 && !slots))
    return set_error(kInvalidArgument, "dsa_batch_tables: null pointer");
  const int64_t nwg = num_rows > 0 ? (num_rows - 1) / kRowsPerWG + 1 : 1;
  if (nwg > INT32_MAX) return set_error(kInvalidArgument, "dsa_batch_tables: too many rows");
  const TabParams P{cached_lens, new_lens, batch, block_tables, bt_stride, bt_width, page_size, free_blocks, num_free,
                    free_head, slots, slots_are_64, positions, positions_are_64, seq_lens, num_rows, cu_seqlens_q,
                    cu_seqlens_k, cu_is_64, status};
  const size_t smem = (2 * (size_t)batch + 1) * sizeof(int64_t);
  if (smem > 32 * 1024 && hipFuncSetAttribute((const void*)batch_tables_kernel,
                                              hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != hipSuccess)
    return set_error(kLaunchFailed, "dsa_batch_tables: cannot reserve %zu B of LDS", smem);
  hipLaunchKernelGGL(batch_tables_kernel, dim3((unsigned)nwg), dim3(kTabThreads), smem, (hipStream_t)stream, P);
  return check_launch("dsa_batch_tables");
}
