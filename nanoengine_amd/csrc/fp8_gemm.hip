// Products of fp8 matrices with a scale for each block of 128, for gfx950.
//
//   out[m, n] = sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k]
//
// a: activations [M, K], b: weights [N, K], both e4m3fn with K contiguous; scales float32,
// or powers of two as e8m0 bytes, which the matrix instruction applies itself.
//
// The products run on v_mfma_scale_f32_32x32x64_f8f6f4 with the weights as its rows, so that
// a lane ends up with one activation row's results for four neighbouring columns at a time.
// e8m0 scales are the instruction's own, and all of K runs into one accumulator. f32 scales take a
// second one: a block's sums times sa sb are added to the first by vector instructions.
//
// Three kernels share that: tiles staged through LDS; waves over K for up to 64 rows; and the
// sum of a product's parts where K is split. A cost fitted to measurements chooses (plan_of).
//
// Tiles: a workgroup's blocks of 128 of a and b go straight from memory into LDS, two or three
// blocks deep: while one is multiplied the others are on their way. A row's eight 16-byte pieces
// are stored in the order piece ^ (row / 2 % 8): 16 rows' reads of one piece fall on different banks
// (rows are half the banks' span apart; with row % 8 two of 16 met on each bank: 1e8 conflict
// cycles in 8192 x 8192 x 16384, now 2e6).
//
// What bounds it, measured: 8192 x 8192 x 16384 (e8m0) 735 to 780 us by card, 2.8 to 3.0 PFLOP/s, where the library's product
// with one scale a matrix takes 720 to 770 and one with a scale per 32 elements 1450. Products run in 79% of
// a SIMD's cycles, and the clock gives way under their power: without any copies it takes 698, with all data in L2 780
// of then 811, without scales 3% less; persistent workgroups, which close the gaps between tiles, gain nothing. Steps
// that brought it there from the first kernel's 1125: operands read ahead of their products 875, copies sent between
// products 840, four waves of 128 x 128 rather than eight of 128 x 64 811, a main loop without rare branches and masks
// 744. f32 scales: 8192^3 462 us against 387; with 64 x 64 a wave, whose sums join while the next tile's products run,
// 573, of which copies are 115 and the joining 80. (128 x 64 with all of its second accumulators does not fit the
// registers, 909.) Short K is bound by a tile's start and end (8192 x 24576 x 1536 298 us where its operations take
// 189); few tiles of long K by the steps of one tile (0.49 us for 128^3, one wave a SIMD) and the second launch: 333 x
// 2112 x 8192, four parts of K, 14 to 16 + 4 us.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "dsa_common.h"
#include "fp8_block.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

typedef float v16f __attribute__((ext_vector_type(16)));

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

// 16 bytes a lane from base + offset into LDS at lds + 16 * lane, without registers; the kernel
// waits for them itself (vmcnt).
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base),
               "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
// The same for the lanes in `mask` (every lane is active at the call).
__device__ __forceinline__ void dma16(const uint8_t* base, uint32_t offset, uint32_t lds, uint64_t mask) {
  asm volatile("s_mov_b64 exec, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\n\ts_mov_b64 exec, -1" ::"v"(offset),
               "s"(base), "s"(mask), "{m0}"(__builtin_amdgcn_readfirstlane(lds))
               : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void* p) { return (uint32_t)reinterpret_cast<uintptr_t>(p); }

// At most LEFT of this wave's loads are under way, and none of its LDS accesses. (A builtin: the compiler's own
// counting of what is under way takes note of it.)
template <int LEFT>
__device__ __forceinline__ void wait_loads() {
  static_assert(LEFT < 64, "the counter's range");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | (LEFT >> 4 << 14));
  asm volatile("" ::: "memory");
}

// The same, and then for every wave of the workgroup.
template <int LEFT>
__device__ __forceinline__ void meet() {
  wait_loads<LEFT>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

enum OutKind : int { kOutBf16 = 0, kOutF32 = 1 };

template <int KIND>
__device__ __forceinline__ uint32_t load_scale(const void* s, int64_t i) {
  return KIND == kScaleF32 ? static_cast<const uint32_t*>(s)[i] : (uint32_t)static_cast<const uint8_t*>(s)[i];
}

// 16 bytes of results from element `at` on, of which `left` lie inside the row.
template <int OUT>
__device__ __forceinline__ void store16(void* out, int64_t at, bool whole, int left, v4i v) {
  if (OUT == kOutBf16) {
    uint16_t* o = static_cast<uint16_t*>(out) + at;
    if (whole) *reinterpret_cast<v4i*>(o) = v;
    else
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left) o[j] = (uint16_t)((uint32_t)v[j >> 1] >> (16 * (j & 1)));
  } else {
    int* o = static_cast<int*>(out) + at;
    if (whole) *reinterpret_cast<v4i*>(o) = v;
    else
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < left) o[j] = v[j];
  }
}

template <int OUT>
__device__ __forceinline__ void store4(void* out, int64_t at, bool whole, int left, const float* v) {
  if (OUT == kOutF32) {
    store16<OUT>(out, at, whole, left,
                 (v4i){__float_as_int(v[0]), __float_as_int(v[1]), __float_as_int(v[2]), __float_as_int(v[3])});
    return;
  }
  uint16_t* o = static_cast<uint16_t*>(out) + at;
  const v2i p = {pack2(v[0], v[1]), pack2(v[2], v[3])};
  if (whole) *reinterpret_cast<v2i*>(o) = p;
  else
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) o[j] = (uint16_t)((uint32_t)p[j >> 1] >> (16 * (j & 1)));
}

constexpr int kMaxStride = 1 << 23;  // a tile's offsets are 32-bit
constexpr int kBand = 4;             // activation tiles of a band

// Activation scales of a tile lie in LDS in chunks, two at a time: 32 e8m0 or 16 f32 blocks (8 beside the widest
// tile's stages) of each row. Rows are an odd number of words apart, so that 32 rows' reads of one block fall on
// different banks.
template <int BM, int BN, int KIND>
constexpr int kScaleChunk = KIND == kScaleF32 && BM * BN < 256 * 256 ? 64 : 32;
template <int BM, int BN, int KIND>
constexpr int kScaleRow = kScaleChunk<BM, BN, KIND> + 4;

template <int BM, int BN, int STAGES, int KIND>
constexpr int gemm_smem() {
  return STAGES * (BM + BN) * kBlock + 2 * BM * kScaleRow<BM, BN, KIND>;
}

// 16 bytes of scales from element i of a row of n, at any address.
template <int KIND>
__device__ __forceinline__ v4i load_scale_piece(const void* row, int i, int n) {
  constexpr int kSize = KIND == kScaleF32 ? 4 : 1;
  const uint8_t* p = static_cast<const uint8_t*>(row) + (int64_t)i * kSize;
  uint64_t v[2] = {0, 0};
  if (i + 16 / kSize <= n) {
    __builtin_memcpy(v, p, 16);
  } else {
#pragma unroll 1
    for (int j = 0; j < 8; j += kSize) {  // an element of each half
      if (i + j / kSize < n) {
        uint32_t x = 0;
        __builtin_memcpy(&x, p + j, kSize);
        v[0] |= (uint64_t)x << (8 * j);
      }
      if (i + (j + 8) / kSize < n) {
        uint32_t x = 0;
        __builtin_memcpy(&x, p + 8 + j, kSize);
        v[1] |= (uint64_t)x << (8 * j);
      }
    }
  }
  return (v4i){(int)v[0], (int)(v[0] >> 32), (int)v[1], (int)(v[1] >> 32)};
}

// A tile of BM activation rows and BN weight rows; a wave takes WM x WN of it. STAGES blocks of both lie in
// LDS: one is multiplied, the others are on their way or wait.
//
// Operands are read from LDS a few products ahead of those that run. Where the reads
// of block s end and those of block s + 1 begin, the waves meet, once a block: all have read block
// s by then, and block s + 1 has landed; block s + STAGES is sent for in block s's place.
template <int BM, int BN, int WM, int WN, int STAGES, int KIND, int OUT>
__global__ void __launch_bounds__((BM / WM) * (BN / WN) * 64)
    __attribute__((amdgpu_waves_per_eu(WM * WN > 128 * 64 ? 1 : 2)))
fp8_gemm_kernel(const GemmParams P) {
  constexpr int kWaves = (BM / WM) * (BN / WN);
  constexpr int kMt = WM / 32, kNt = WN / 32;
  constexpr int kStage = (BM + BN) * kBlock;
  constexpr int kPerA = BM / 8 / kWaves, kPerB = BN / 8 / kWaves;  // instructions of a stage: eight rows each
  constexpr int kChunk = kScaleChunk<BM, BN, KIND>, kRow = kScaleRow<BM, BN, KIND>;
  constexpr int kScales = KIND == kScaleF32 ? kChunk / 4 : kChunk, kRowPieces = kChunk / 16;
  static_assert(kPerA * kWaves * 8 == BM && kPerB * kWaves * 8 == BN, "rows dealt out evenly");
  static_assert(kWaves % 2 == 0, "a wave's rows of a stage have one order of pieces");
  static_assert(kBlock % WN == 0, "one weight scale a wave");
  static_assert(STAGES == 2 || STAGES == 3, "one block on its way behind the next, or none");
  static_assert(64 % kScales == 0 && kScales >= 4, "weight scales are replaced where a chunk is");
  constexpr int kThreads = kWaves * 64, kPieces = (kRowPieces * BM + kThreads - 1) / kThreads;  // of a scale chunk, a thread
  static_assert(kRowPieces * BM % (kPieces * 64) == 0, "whole waves bring scales");
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Workgroups go to the eight XCDs in turn: each XCD takes a run of neighbouring tiles, in bands of four activation
  // tiles, so that the tiles at work beside one L2 share their rows. (Against tiles dealt out to the XCDs one by one,
  // 2048 x 8192 x 8192 takes 4% less and 333 x 8192 x 8192 40 us rather than 60.)
  const int tiles = P.mtiles * P.ntiles;
  const int xcd = blockIdx.x & 7, share = gridDim.x >> 3, rest = gridDim.x & 7;
  const int at = xcd * share + min(xcd, rest) + (blockIdx.x >> 3);
  const int split = at / tiles, tile = at - split * tiles;
  const int band = tile / (kBand * P.ntiles), in_band = tile - band * kBand * P.ntiles;
  const int wide = min(kBand, P.mtiles - kBand * band);
  const int m0 = (kBand * band + in_band % wide) * BM, n0 = in_band / wide * BN;
  const int kb0 = (int)((int64_t)P.kblocks * split / P.splits), kb1 = (int)((int64_t)P.kblocks * (split + 1) / P.splits);
  const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
  const int c32 = lane & 31, half = lane >> 5;

  // this lane's pieces of a stage, from the tile's first row on; rows past the matrix repeat its last one
  uint32_t off_a[kPerA], off_b[kPerB];
  const int piece = (lane & 7) ^ (4 * (wave & 1) + (lane >> 4));
  auto offset = [&](int i, int last, int64_t stride) {
    uint32_t v = (uint32_t)min(8 * (wave + i * kWaves) + (lane >> 3), last) * (uint32_t)stride + 16 * piece;
    asm volatile("" : "+v"(v));  // (one register, not the pair of a 64-bit product)
    return v;
  };
#pragma unroll
  for (int i = 0; i < kPerA; ++i) off_a[i] = offset(i, P.m - 1 - m0, P.a_stride);
#pragma unroll
  for (int i = 0; i < kPerB; ++i) off_b[i] = offset(i, P.n - 1 - n0, P.b_stride);
  const uint8_t* tile_a = P.a + (int64_t)m0 * P.a_stride;
  const uint8_t* tile_b = P.b + (int64_t)n0 * P.b_stride;
  // the lanes whose pieces of the last block lie inside K
  const int full = P.k / kBlock;  // whole blocks
  const uint64_t tail = __builtin_amdgcn_ballot_w64(16 * piece < P.k % kBlock);
  const uint32_t dst0 = lds_addr(smem) + wave * 1024;
  // copy i of block kb: the activations' first
  auto copy = [&](int kb, int buf, int i, auto... mask) {
    const uint32_t dst = dst0 + buf * kStage + i * kWaves * 1024;
    if (i < kPerA) dma16(tile_a + (int64_t)kb * kBlock, off_a[i < kPerA ? i : 0], dst, mask...);
    else dma16(tile_b + (int64_t)kb * kBlock, off_b[i < kPerA ? 0 : i - kPerA], dst, mask...);
  };
  // zeros where the last block lies past the end of K
  auto clear_tail = [&](int buf) {
    if (16 * piece >= P.k % kBlock) {
      uint8_t* z = smem + buf * kStage + wave * 1024 + lane * 16;
#pragma unroll
      for (int i = 0; i < kPerA + kPerB; ++i) *reinterpret_cast<v4i*>(z + i * kWaves * 1024) = (v4i){0, 0, 0, 0};
    }
  };
  auto issue = [&](int kb, int buf, int copies) {
    const uint64_t mask = kb < full ? ~0ull : tail;
#pragma unroll
    for (int i = 0; i < kPerA + kPerB; ++i)
      if (i < copies) copy(kb, buf, i, mask);
  };

  // activation scales: thread t brings piece t % kRowPieces of a chunk of row t / kRowPieces. (Its addresses are made
  // anew from an opaque copy of the thread's number: kept in registers they would be spilled.)
  uint8_t* scale_lds = smem + STAGES * kStage;
  const bool brings = kPieces * kThreads == kRowPieces * BM || (int)threadIdx.x < kRowPieces * BM;
  struct Chunk {
    v4i v[kPieces];
  };
  auto load_chunk = [&](int kb) {
    Chunk c;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int t = threadIdx.x + i * kThreads;
      asm volatile("" : "+v"(t));
      const int64_t row = (int64_t)min(m0 + t / kRowPieces, P.m - 1) * P.sa_stride;
      c.v[i] = load_scale_piece<KIND>(KIND == kScaleF32 ? (const void*)(static_cast<const uint32_t*>(P.sa) + row)
                                                        : (const void*)(static_cast<const uint8_t*>(P.sa) + row),
                                      kb + t % kRowPieces * (kScales / kRowPieces), P.kblocks);
    }
    return c;
  };
  auto keep_chunk = [&](const Chunk& c, int which) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      int t = threadIdx.x + i * kThreads;
      asm volatile("" : "+v"(t));
      uint32_t* d = reinterpret_cast<uint32_t*>(scale_lds + which * BM * kRow + t / kRowPieces * kRow + t % kRowPieces * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = (uint32_t)c.v[i][j];
    }
  };
  // the scale of this lane's row in activation tile j at block kb
  auto row_scale = [&](int step, int j) -> uint32_t {
    const uint8_t* p = scale_lds + ((step / kScales) & 1) * BM * kRow + (wm + 32 * j + c32) * kRow;
    return KIND == kScaleF32 ? reinterpret_cast<const uint32_t*>(p)[step % kScales] : (uint32_t)p[step % kScales];
  };
  // the wave's one weight scale a block, 64 blocks a lane each
  const int64_t sb_at = (int64_t)min((n0 + wn) / kBlock, (P.n - 1) / kBlock) * P.sb_stride;
  auto load_weight_scales = [&](int kb) { return load_scale<KIND>(P.sb, sb_at + min(kb + lane, P.kblocks - 1)); };

  v16f acc[kNt][kMt], part[kNt][kMt];  // (kByTile: one tile's part)
#pragma unroll
  for (int i = 0; i < kNt; ++i)
#pragma unroll
    for (int j = 0; j < kMt; ++j) acc[i][j] = (v16f){};

  // this lane's two 16-byte pieces of half h of a row: at0 ^ 64 h and that ^ 16
  const uint32_t at0 = c32 * kBlock + 16 * ((2 * half) ^ ((lane >> 1) & 7));
  auto operand = [&](int buf, int row, int h) {
    const uint8_t* rows = smem + (buf * kStage + row * kBlock);
    const v4i x = *reinterpret_cast<const v4i*>(rows + (at0 ^ (64 * h)));
    const v4i y = *reinterpret_cast<const v4i*>(rows + (at0 ^ (64 * h + 16)));
    return (v8i){x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };
  // A step's groups: half h of activation tile j times all weight tiles. Group g's activations lie in
  // slot g % kSlots and are read kAhead groups before; weights a half before.
  // (as far ahead as registers allow)
  constexpr bool kTight = kMt == 4 || (KIND == kScaleF32 && kMt == 2);
  // f32 scales and the widest tile: both halves of an activation tile follow one another, and its sums join the others
  // before the next tile's take their registers
  constexpr bool kByTile = KIND == kScaleF32 && kMt == 4;
  constexpr int kGroups = 2 * kMt, kAhead = kByTile ? 1 : kTight ? kMt - 1 : kMt;
  constexpr int kSlots = kByTile ? 2 : kTight ? kMt : kGroups;
  auto tile_of = [](int g) { return kByTile ? g / 2 : g % kMt; };
  auto half_of = [](int g) { return kByTile ? g % 2 : g / kMt; };
  v8i fa[kSlots], fb[2][kNt];
  // scales of this block, and of the next ones (replaced one by one behind their last use where tiles are read that late)
  constexpr bool kEach = kAhead < kMt;
  // Copies are sent between the products: a wave that sent all of its own at once would stand until they are taken.
  // Two meetings a block (kTwice): its weights' place is free early, its activations' at the second. Else the copies of
  // block s + STAGES are dealt out over the kSend products behind the meeting, the last of them in the next step.
  constexpr bool kTwice = kMt == 4;
  constexpr int kSlotsAll = kGroups * kNt, kMeetAt = (kGroups - kAhead) * kNt, kCopies = kPerA + kPerB;
  constexpr int kSend = STAGES > 2 ? kSlotsAll : kSlotsAll / 2, kSendHere = kSlotsAll - kMeetAt;
  constexpr int kCopiesHere = kSendHere >= kSend ? kCopies : kSendHere * kCopies / kSend;  // before the step ends
  uint32_t ca[kMt], na[kMt], cb, sb = 0, sb_next = 0;
  // f32 scales: a tile's sums over a block join the others while the next tile's products run
  constexpr bool kDelay = KIND == kScaleF32 && kMt > 1 && !kByTile;
  float join = 0.f;
  if (kDelay)
#pragma unroll
    for (int i = 0; i < kNt; ++i) part[i][kMt - 1] = (v16f){};
  auto join_tile = [&](int j, float f) {
#pragma unroll
    for (int i = 0; i < kNt; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] += part[i][kByTile ? 0 : j][r] * f;
  };

  const int steps = kb1 - kb0;
  if (steps > 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i)
      if (i < steps) issue(kb0 + i, i, i < STAGES - 1 || kTwice ? kCopies : kCopiesHere);
    if (kb0 == full) clear_tail(0);
    Chunk c0 = {}, c1 = {};
    sb = load_weight_scales(kb0);
    if (brings) {
      c0 = load_chunk(kb0);
      if (steps > kScales) c1 = load_chunk(kb0 + kScales);
      keep_chunk(c0, 0);
      keep_chunk(c1, 1);
    }
    asm volatile("" ::"v"(sb));  // (waited for here)
    meet<0>();
#pragma unroll
    for (int i = 0; i < kNt; ++i) fb[0][i] = operand(0, BM + wn + 32 * i, 0);
#pragma unroll
    for (int g = 0; g < kAhead; ++g) fa[g % kSlots] = operand(0, wm + 32 * tile_of(g), half_of(g));
#pragma unroll
    for (int j = 0; j < kMt; ++j) ca[j] = row_scale(0, j);
  }
  // What the epilogue needs is loaded, and waited for, before the loop: with a scalar load under way the
  // compiler would wait for every LDS read at each step's first product.
  void* out = P.out;
  int64_t out_stride = P.out_stride;
  asm volatile("" : "+s"(out), "+s"(out_stride));
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  Chunk next_chunk = {};
  int buf = 0;  // block s's place
  // One step: block s is multiplied, block s + STAGES sent for (and the rest of the one before).
  // LAST: one of them may be short, or not there.
  auto step = [&](int s, auto last) {
    constexpr bool LAST = decltype(last)::value;
    const int buf1 = buf + 1 < STAGES ? buf + 1 : 0, buf0 = buf > 0 ? buf - 1 : STAGES - 1, kb2 = kb0 + s + STAGES;
    const uint64_t mask = kb2 < min(kb1, full) ? ~0ull : kb2 < kb1 ? tail : 0ull;
    const uint64_t mask0 = kb2 - 1 < min(kb1, full) ? ~0ull : kb2 - 1 < kb1 ? tail : 0ull;
    auto send = [&](int i) {
      if constexpr (LAST) copy(kb2, buf, i, mask);
      else copy(kb2, buf, i);
    };
    auto send_rest = [&](int i) {
      if constexpr (LAST) copy(kb2 - 1, buf0, i, mask0);
      else copy(kb2 - 1, buf0, i);
    };
    cb = __builtin_amdgcn_readlane(sb, s % 64);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int h = half_of(g), j = tile_of(g), t = g + kAhead;
#pragma unroll
      for (int i = 0; i < kNt; ++i) {  // one product, and what is sent for meanwhile
        if (kTwice && g == 2 && i == 0) {
          // every wave has read the block's weights: those of block s + STAGES take their place
          asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        if (g == kGroups - kAhead && i == 0) {
          // this wave has read all of the block, and its share of the next has landed; past the barrier
          // that holds for all (behind the last block nothing has been sent: what is read then is not used).
          // The products before it stay before it: without a use there the compiler moves them past the branches.
#pragma unroll
          for (int x = 0; x < kNt; ++x)
#pragma unroll
            for (int y = 0; y < kMt; ++y) {
              if (WM * WN > 128 * 64) asm volatile("" : "+a"(acc[x][y]));
              else if (KIND == kScaleE8M0 || kByTile) asm volatile("" : "+v"(acc[x][y]));
              else asm volatile("" : "+v"(part[x][y]));
            }
          // The chunk of scales after the next: sent for at a chunk's first step, kept at its second.
          if (__builtin_expect((unsigned)(s + 1) % kScales < 3 && s + 1 >= kScales, 0)) {
            if (s % kScales == 0) {
              if (s % 64 == kScales % 64 && s + 64 - kScales < steps) sb_next = load_weight_scales(kb0 + s + 64 - kScales);
              if (s + kScales < steps && brings) next_chunk = load_chunk(kb0 + s + kScales);
            } else if (s % kScales == 1) {
              if (brings) keep_chunk(next_chunk, ((s / kScales) & 1) ^ 1);
              asm volatile("" ::"v"(sb_next));  // (waited for here, not where it is used)
            } else if (s % 64 == 63) {
              sb = sb_next;
            }
          }
          if (LAST && s + 1 < steps && kb0 + s + 1 == full) clear_tail(buf1);
          // the blocks behind the next may still be on their way
          if (kTwice) {
            if (LAST) wait_loads<0>();
            meet<kPerB>();
          } else if (LAST) {
            if (steps - 2 - s >= STAGES - 2) wait_loads<(STAGES - 2) * (kPerA + kPerB)>();
            else wait_loads<0>();
            meet<(STAGES - 2) * (kPerA + kPerB)>();
          } else {
            meet<(STAGES - 2) * (kPerA + kPerB)>();
          }
          if (!kEach) {
#pragma unroll
            for (int x = 0; x < kMt; ++x) na[x] = row_scale(s + 1, x);
          }
        }
        if constexpr (kTwice) {
          constexpr int kLate = kAhead < 2 ? 1 : 2;  // groups behind the meeting
          constexpr int kNowA = kPerA / (kLate * kNt), kNowB = kPerB / (2 * kNt);
          static_assert(kNowA * kLate * kNt == kPerA && kNowB * 2 * kNt == kPerB, "copies dealt out evenly");
          if (g / 2 == 1)
#pragma unroll
            for (int x = 0; x < kNowB; ++x) send(kPerA + ((g - 2) * kNt + i) * kNowB + x);
          if (g >= kGroups - kLate)
#pragma unroll
            for (int x = 0; x < kNowA; ++x) send(((g - kGroups + kLate) * kNt + i) * kNowA + x);
        } else {
          const int q = g * kNt + i, r = q >= kMeetAt ? q - kMeetAt : q + kSendHere;  // products since the meeting
#pragma unroll
          for (int x = 0; x < kCopies; ++x)
            if (r < kSend && x >= r * kCopies / kSend && x < (r + 1) * kCopies / kSend) {
              if (q >= kMeetAt) send(x);
              else send_rest(x);
            }
        }
        if (g == 0) fb[1][i] = operand(buf, BM + wn + 32 * i, 1);
        if (g == kGroups - kAhead) fb[0][i] = operand(buf1, BM + wn + 32 * i, 0);
        if (i == 0) {
          if (kByTile) {
            if (h == 0 && j + 1 < kMt) ca[j + 1] = row_scale(s, j + 1);
            if (g == kGroups - 1) na[0] = row_scale(s + 1, 0);
          } else if (kEach) {
            if (g >= kGroups - kAhead) ca[g - (kGroups - kAhead)] = row_scale(s + 1, g - (kGroups - kAhead));
            if (g == 0) ca[kMt - 1] = row_scale(s, kMt - 1);
          }
          fa[t % kSlots] = operand(t < kGroups ? buf : buf1, wm + 32 * tile_of(t % kGroups), half_of(t % kGroups));
        }
        __builtin_amdgcn_sched_barrier(0);
        if (KIND == kScaleE8M0)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[h][i], fa[g % kSlots], acc[i][j], 0, 0, 0, cb, 0,
                                                                      ca[j]);
        else
          part[i][kByTile ? 0 : j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
              fb[h][i], fa[g % kSlots], h ? part[i][kByTile ? 0 : j] : (v16f){}, 0, 0, 0, 127, 0, 127);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (kDelay && (g == 0 || h == 1)) {
        if (g == 0) join_tile(kMt - 1, join);
        else if (j > 0) join_tile(j - 1, join);
        if (h == 1) join = __uint_as_float(ca[j]) * __uint_as_float(cb);
        __builtin_amdgcn_sched_barrier(0);
      } else if (KIND == kScaleF32 && h == 1) {
        join_tile(j, __uint_as_float(ca[j]) * __uint_as_float(cb));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (kByTile) ca[0] = na[0];
    if (!kEach) {
#pragma unroll
      for (int j = 0; j < kMt; ++j) ca[j] = na[j];
    }
    buf = buf1;
  };
  const int plain = min(steps, full - kb0) - STAGES;  // steps that send for a whole block
  int s = 0;
  for (; s < plain; ++s) step(s, std::false_type{});
  for (; s < steps; ++s) step(s, std::true_type{});
  if (kDelay) join_tile(kMt - 1, join);

  // Lane (c32, half) holds row c32 of an activation tile, columns 8g + 4 half .. + 3 of a weight tile: 32 rows at a
  // time they change places in LDS (a part of its own for each wave), so that a store takes 16 bytes a lane and whole rows.
  // (From the registers, 8 bytes a lane and 32 rows to a store, 256 x 256 results took 10.8 us.)
  constexpr int kSize = OUT == kOutBf16 ? 2 : 4, kEach16 = 16 / kSize;
  constexpr int kPitch = WN * kSize + 16, kRowChunks = WN * kSize / 16;
  static_assert(kWaves * 32 * kPitch <= STAGES * kStage, "the stages' place");
  if (P.splits > 1) out = static_cast<float*>(out) + (int64_t)split * P.m * P.n;
  const bool aligned = !((reinterpret_cast<uintptr_t>(out) & 15) | (out_stride & (kEach16 - 1)));
  meet<0>();
  uint8_t* mine = smem + wave * 32 * kPitch;
#pragma unroll
  for (int j = 0; j < kMt; ++j) {
#pragma unroll
    for (int i = 0; i < kNt; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint8_t* d = mine + c32 * kPitch + (32 * i + 8 * g + 4 * half) * kSize;
        const v16f& v = acc[i][j];
        if (OUT == kOutBf16)
          *reinterpret_cast<v2i*>(d) = (v2i){pack2(v[4 * g], v[4 * g + 1]), pack2(v[4 * g + 2], v[4 * g + 3])};
        else
          *reinterpret_cast<v4f*>(d) = (v4f){v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
      }
    wait_loads<63>();  // (LDS only; the wave's own accesses are in order)
    auto row_of = [&](int x) { return (64 * x + lane) / kRowChunks; };
    auto col_of = [&](int x) { return (64 * x + lane) % kRowChunks * kEach16; };
    auto held = [&](int x) { return *reinterpret_cast<const v4i*>(mine + row_of(x) * kPitch + col_of(x) * kSize); };
    const int m = m0 + wm + 32 * j, n = n0 + wn;
    constexpr int kStores = 32 * kRowChunks / 64;
    if (aligned && n + WN <= P.n) {
      // Results are streamed past the L2, where they would take the place of rows that neighbouring tiles share (8192 x
      // 24576 x 1536 353 -> 318 us, f32 scales 504 -> 419; parts of K too, 333 x 2112 x
      // 8192 20.0 -> 19.3).
      uint8_t* to = static_cast<uint8_t*>(out) + ((int64_t)m * out_stride + n) * kSize;
#pragma unroll
      for (int x = 0; x < kStores; ++x)
        if (m + row_of(x) < P.m)
          __builtin_nontemporal_store(held(x), reinterpret_cast<v4i*>(to + (row_of(x) * out_stride + col_of(x)) * kSize));
    } else {
#pragma unroll 1
      for (int x = 0; x < kStores; ++x)
        if (m + row_of(x) < P.m && n + col_of(x) < P.n)
          store16<OUT>(out, (int64_t)(m + row_of(x)) * out_stride + n + col_of(x), aligned && n + col_of(x) + kEach16 <= P.n,
                       P.n - n - col_of(x), held(x));
    }
    wait_loads<63>();
  }
}

// Few rows: a workgroup takes 32 columns, its four or eight waves parts of K, each with two blocks of 128 of its own on
// their way into LDS in whole lines while a third is multiplied; the waves' sums meet in LDS, in order. No meetings of
// waves until then, no second launch: 1 x 8192 x 1536 in 4.0 us (by tiles 8.0), 32 x 576 x 1536 4.0 (7.5), 16 x 2112 x
// 8192 7.1 (10.8), 8 x 8192 x 8192 13.3 (15.4; its bytes take 13.0). What bounds it is the start (under 2 us beside the
// launch) and then memory, or what few CUs can fetch: 0.3 us a block of K for each of four waves. (Straight into
// registers a load touches 32 rows, and where these lie a power of two apart their lines crowd each other out of L1
// before the next load wants them: 16 x 2112 x 8192 15.4, 1 x 8192 x 1536 4.6.)
constexpr int kFew = 32;         // columns, and rows of one activation tile: there are one or two
constexpr int kFewBlocks = 16;   // of K, a wave at most
template <int TILES>
constexpr int kFewStage = (1 + TILES) * kFew * kBlock;  // a block of weights and of activations
template <int TILES>
constexpr int kFewWave = 2 * kFewStage<TILES> + kFewBlocks * TILES * kFew * 4;  // and the activations' scales

// The waves' sums of a workgroup's 32 columns, in order, to the result. Lane (c32, half) holds row c32, columns 8g + 4 half
// .. + 3.
template <int WAVES, int TILES, int OUT>
__device__ __forceinline__ void join_waves(const GemmParams& P, v4f* sums, const v16f* acc) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c32 = lane & 31, half = lane >> 5, n0 = blockIdx.x * kFew;
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      sums[(t * WAVES + wave) * 256 + g * 64 + lane] =
          (v4f){acc[t][4 * g], acc[t][4 * g + 1], acc[t][4 * g + 2], acc[t][4 * g + 3]};
  __syncthreads();
  const int n = n0 + 8 * wave + 4 * half;
  if (threadIdx.x >= 256 || n >= P.n) return;
  const bool aligned = !((reinterpret_cast<uintptr_t>(P.out) & (OUT == kOutBf16 ? 7 : 15)) | (P.out_stride & 3));
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    const int m = t * kFew + c32;
    if (m >= P.m) return;
    v4f v = sums[t * WAVES * 256 + threadIdx.x];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      const v4f x = sums[(t * WAVES + w) * 256 + threadIdx.x];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += x[j];
    }
    const float r[4] = {v[0], v[1], v[2], v[3]};
    store4<OUT>(P.out, (int64_t)m * P.out_stride + n, aligned && n + 4 <= P.n, P.n - n, r);
  }
}

template <int WAVES, int TILES, int KIND, int OUT>
__global__ void __launch_bounds__(WAVES * 64) fp8_gemm_few_kernel(const GemmParams P) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c32 = lane & 31, half = lane >> 5;
  const int n0 = blockIdx.x * kFew;
  const int kb0 = (int)((int64_t)P.kblocks * wave / WAVES), kb1 = (int)((int64_t)P.kblocks * (wave + 1) / WAVES);
  const int steps = kb1 - kb0, full = P.k / kBlock;
  constexpr int kStage = kFewStage<TILES>, kRows = TILES * kFew, kCopies = 4 + 4 * TILES;
  uint8_t* mine = smem + wave * kFewWave<TILES>;
  uint32_t* scales = reinterpret_cast<uint32_t*>(mine + 2 * kStage);

  // copy i brings rows 8i .. 8i + 7, pieces in the tiles' order; rows past the matrix repeat its last one
  const int piece0 = (lane & 7) ^ (lane >> 4), piece1 = piece0 ^ 4;
  uint32_t off_a[4 * TILES], off_b[4];
#pragma unroll
  for (int i = 0; i < 4 * TILES; ++i) {
    const int row = 8 * i + (lane >> 3), piece = i & 1 ? piece1 : piece0;
    off_a[i] = (uint32_t)min(row, P.m - 1) * (uint32_t)P.a_stride + 16 * piece;
    if (i < 4) off_b[i] = (uint32_t)min(row, P.n - 1 - n0) * (uint32_t)P.b_stride + 16 * piece;
  }
  const uint8_t* tile_b = P.b + (int64_t)n0 * P.b_stride;
  const uint64_t tail0 = __builtin_amdgcn_ballot_w64(16 * piece0 < P.k % kBlock);
  const uint64_t tail1 = __builtin_amdgcn_ballot_w64(16 * piece1 < P.k % kBlock);
  auto issue = [&](int s) {
    const int kb = kb0 + s, buf = s & 1;
    const uint32_t dst = lds_addr(mine) + buf * kStage;
    if (kb < full) {
#pragma unroll
      for (int i = 0; i < 4 * TILES; ++i) {
        if (i < 4) dma16(tile_b + (int64_t)kb * kBlock, off_b[i], dst + i * 1024);
        dma16(P.a + (int64_t)kb * kBlock, off_a[i], dst + 4096 + i * 1024);
      }
    } else {
      const v4i zero = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4 * TILES; ++i) {
        const uint64_t mask = i & 1 ? tail1 : tail0;
        if (i < 4) dma16(tile_b + (int64_t)kb * kBlock, off_b[i], dst + i * 1024, mask);
        dma16(P.a + (int64_t)kb * kBlock, off_a[i], dst + 4096 + i * 1024, mask);
      }
#pragma unroll
      for (int i = 0; i < kCopies; ++i)
        if (16 * (i & 1 ? piece1 : piece0) >= P.k % kBlock)
          *reinterpret_cast<v4i*>(mine + buf * kStage + i * 1024 + lane * 16) = zero;
    }
  };
  for (int s = 0; s < min(steps, 2); ++s) issue(s);
  // scales: of the activations in LDS, [block][row]; of the weights one a lane
  const int row = lane % kRows, first = lane / kRows;
  const int64_t sb_at = (int64_t)(n0 / kBlock) * P.sb_stride, sa_at = (int64_t)min(row, P.m - 1) * P.sa_stride;
  uint32_t sb = load_scale<KIND>(P.sb, sb_at + min(kb0 + lane, P.kblocks - 1));
  constexpr int kEach = 64 / kRows;  // blocks at a time
  uint32_t sa[kFewBlocks / kEach];
#pragma unroll
  for (int t = 0; t < kFewBlocks / kEach; ++t)
    sa[t] = load_scale<KIND>(P.sa, sa_at + min(kb0 + kEach * t + first, P.kblocks - 1));
#pragma unroll
  for (int t = 0; t < kFewBlocks / kEach; ++t) scales[(kEach * t + first) * kRows + row] = sa[t];
  asm volatile("" : "+v"(sb));  // (waited for here)
  wait_loads<0>();

  const uint32_t at0 = c32 * kBlock + 16 * ((2 * half) ^ ((lane >> 1) & 7));
  v16f acc[TILES] = {};
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) wait_loads<kCopies>();  // the next block may still be on its way
    else wait_loads<0>();
    const uint8_t* rows = mine + s % 2 * kStage;
    v8i fa[TILES][2], fb[2];
    auto operand = [&](int at) {
      const v4i p = *reinterpret_cast<const v4i*>(rows + at), q = *reinterpret_cast<const v4i*>(rows + (at ^ 16));
      return (v8i){p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      fb[h] = operand(at0 ^ (64 * h));
#pragma unroll
      for (int t = 0; t < TILES; ++t) fa[t][h] = operand((1 + t) * 4096 + (at0 ^ (64 * h)));
    }
    uint32_t ca[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) ca[t] = scales[s * kRows + t * kFew + c32];
    const uint32_t cb = __builtin_amdgcn_readlane(sb, s);
    wait_loads<63>();  // the block is in registers: its place is free
    if (s + 2 < steps) issue(s + 2);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      if (KIND == kScaleE8M0) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          acc[t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[h], fa[t][h], acc[t], 0, 0, 0, cb, 0, ca[t]);
      } else {
        v16f part = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
          part = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[h], fa[t][h], part, 0, 0, 0, 127, 0, 127);
        const float f = __uint_as_float(ca[t]) * __uint_as_float(cb);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] += part[r] * f;
      }
    }
  }
  __syncthreads();
  join_waves<WAVES, TILES, OUT>(P, reinterpret_cast<v4f*>(smem), acc);
}

// out = the sum of the splits' partial sums, in order; eight parts' loads in flight at once. They are read once, past the L2
// (333 x 2112 x 8192, cold, 19.6 -> 18.1 us); single waves spread evenly over the CUs (0.2 us).
constexpr int kSumThreads = 64;

template <int OUT>
__global__ void __launch_bounds__(kSumThreads)
fp8_gemm_sum_kernel(const float* __restrict__ part, int splits, int m, int n, void* __restrict__ out, int64_t out_stride) {
  // (few tiles are split: the results are far fewer than 2^32)
  const uint32_t per_row = (n + 3) / 4, i = blockIdx.x * kSumThreads + threadIdx.x, in_order = i / per_row;
  if (in_order >= (uint32_t)m) return;
  const int64_t row = in_order;
  const int c = (int)(i - in_order * per_row) * 4;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  const bool whole = n % 4 == 0;
  const float* p = part + row * n + c;
  const int64_t step = (int64_t)m * n;
  for (int s = 0; s < splits; s += 8) {
    v4f x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float* q = p + min(s + k, splits - 1) * step;
      if (whole) {
        x[k] = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(q));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[k][j] = q[min(c + j, n - 1) - c];
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s + k < splits) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += x[k][j];
      }
  }
  const bool aligned = !((reinterpret_cast<uintptr_t>(out) & (OUT == kOutBf16 ? 7 : 15)) | (out_stride & 3));
  store4<OUT>(out, row * out_stride + c, aligned && whole, n - c, v);
}

// The tiles there are, and what a product of G of them takes, in us: fitted to measurements of several hundred shapes (1 to
// 8192 rows, 64 to 24576 columns, 128 to 8192 deep). Over 360 others the choice takes 1.004 times the best form's time in the
// mean, above 64 rows 1.007, and 1.17 at worst.
//   n = ceil(G / CUs) tiles a CU, r = ceil(n / resident) of them after one another, steps blocks of K each:
//   base + n (per_tile + steps per_step) + r (per_round + steps per_round_step)
// Small tiles keep every CU and its memory path busy where there are few rows (1 x 8192 x 1536 by 32 x 64 tiles of
// three stages 7.7 us, of two 9.3); large ones read less from L2 per product (2048 x 8192 x 8192 by 256 x 256 104 us,
// by 128 x 128 143). The widest tile has four waves of 128 x 128, or eight of 128 x 64: these read more from LDS (8192^3 387
// and 394 us) but begin and end a tile sooner (8192 x 24576 x 1536 318 and 298). f32 scales leave room for the latter only.
struct Tile {
  int bm, bn, wm, wn, stages, resident;
  float base, per_step, per_round_step, per_tile, per_round;
};
constexpr Tile kTilesE8M0[] = {
    {32, 64, 32, 32, 3, 4, 3.0f, 0.05f, 0.20f, 1.25f, 0.f},   {64, 64, 32, 32, 3, 3, 2.85f, 0.11f, 0.12f, 1.1f, 1.1f},
    {64, 128, 32, 64, 3, 2, 3.0f, 0.20f, 0.10f, 1.4f, 1.4f},  {128, 128, 64, 64, 2, 2, 1.9f, 0.21f, 0.36f, 2.1f, 1.7f},
    {128, 128, 64, 64, 3, 1, 1.7f, 0.42f, 0.f, 4.8f, 0.f},    {256, 128, 64, 64, 2, 1, 0.8f, 0.86f, 0.f, 6.0f, 0.f},
    {256, 256, 128, 64, 2, 1, 0.f, 1.25f, 0.f, 10.1f, 0.f},   {256, 256, 128, 128, 2, 1, 0.f, 1.19f, 0.f, 12.2f, 0.f}};
constexpr Tile kTilesF32[] = {
    {32, 64, 32, 32, 3, 3, 2.3f, 0.04f, 0.28f, 1.2f, 0.f},    {64, 64, 32, 32, 3, 2, 2.6f, 0.08f, 0.235f, 1.35f, 0.f},
    {64, 128, 32, 64, 2, 2, 2.1f, 0.085f, 0.41f, 1.7f, 0.f},  {64, 128, 32, 64, 3, 1, 2.2f, 0.38f, 0.f, 0.f, 2.4f},
    {256, 128, 64, 64, 2, 1, 0.55f, 1.05f, 0.f, 5.9f, 0.f},   {256, 256, 128, 64, 2, 1, 0.f, 1.6f, 0.f, 9.0f, 0.f}};
template <int KIND>
constexpr int kTileCount = KIND == kScaleF32 ? sizeof(kTilesF32) / sizeof(Tile) : sizeof(kTilesE8M0) / sizeof(Tile);
template <int KIND, int I>
constexpr Tile kTile = KIND == kScaleF32 ? kTilesF32[I] : kTilesE8M0[I];
constexpr const Tile* tiles_of(int kind) { return kind == kScaleF32 ? kTilesF32 : kTilesE8M0; }
// A second launch adds up the parts of K: so much, and more by their MB.
constexpr float kSumBase = 2.9f, kSumPerMB[2] = {0.33f, 0.25f};

constexpr int kFewTile = -1;

struct Plan {
  int tile, splits;  // kFewTile: by the kernel for few rows, and its waves
};

Plan plan_of(int m, int n, int k, int kind, int cus) {
  const int kblocks = (k + kBlock - 1) / kBlock;
  // Few rows: the kernel of their own as far as a wave's scales reach. Up to 32: 1.4 times as fast as the best tile over 125
  // shapes (64 to 24576 columns, 128 to 8192 deep), by four waves, of which a CU holds two groups (32 x 8192 x 8192
  // 13.5 us, by eight 15.6), and by eight where K is too long for four. Up to 64 where every group has a CU at once (64 x
  // 8192 x 1536 6.2 us, by tiles 8.3; 64 x 24576 x 1536 14.8 and 11.3), and K is short or half of the CUs have one (64 x 576
  // x 8192 11.1 and 9.0).
  const int groups = (n - 1) / kFew + 1;
  if (m <= kFew && kblocks <= 8 * kFewBlocks) return {kFewTile, kblocks > 4 * kFewBlocks ? 8 : 4};
  if (m > kFew && m <= 2 * kFew && groups <= cus && kblocks <= 4 * kFewBlocks && (kblocks <= 32 || groups > cus / 2))
    return {kFewTile, 4};
  const Tile* tiles = tiles_of(kind);
  const int count = kind == kScaleF32 ? kTileCount<kScaleF32> : kTileCount<kScaleE8M0>;
  Plan best = {0, 1};
  double least = 1e300;
  for (int t = 0; t < count; ++t) {
    const Tile& T = tiles[t];
    const double all = ((m - 1) / T.bm + 1.0) * ((n - 1) / T.bn + 1.0);
    for (int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
      // parts of two blocks at least, and none where every CU has its tile
      if (splits > 1 && (2 * splits > kblocks || all * (splits - 1) > 2.0 * cus)) break;
      const double g = std::ceil(all * splits / cus), r = std::ceil(g / T.resident), steps = (kblocks - 1) / splits + 1;
      double us = T.base + g * (T.per_tile + steps * T.per_step) + r * (T.per_round + steps * T.per_round_step);
      if (splits > 1) us += kSumBase + kSumPerMB[kind] * 4e-6 * splits * m * n;
      if (us < least) {
        least = us;
        best = {t, splits};
      }
    }
  }
  return best;
}

size_t workspace_of(const Plan& p, int m, int n) {
  return p.tile != kFewTile && p.splits > 1 ? (size_t)p.splits * m * n * sizeof(float) : 0;
}

constexpr int kMaxDevices = 64;

// Compute units of the current device (asked for once: a call is a few us).
int device_cus(int dev) {
  static std::atomic<int> known[kMaxDevices];
  if (dev < 0 || dev >= kMaxDevices) return 256;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) return 256;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int current_device() {
  int dev = -1;
  return hipGetDevice(&dev) == hipSuccess ? dev : -1;
}

// A kernel's use of more LDS than 64 KB has to be asked for, once a device (`known`: those that were).
int allow_smem(const void* kern, int bytes, int dev, std::atomic<uint64_t>& known) {
  const uint64_t bit = dev >= 0 && dev < kMaxDevices ? 1ull << dev : 0;
  if (bytes <= 64 * 1024 || (known.load(std::memory_order_relaxed) & bit)) return kOk;
  const hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return set_error(kLaunchFailed, "dsa_fp8_gemm: %s", hipGetErrorString(e));
  known.fetch_or(bit, std::memory_order_relaxed);
  return kOk;
}

template <int KIND, int I, int OUT>
int launch_tile(GemmParams P, int dev, hipStream_t st) {
  constexpr Tile T = kTile<KIND, I>;
  constexpr int BM = T.bm, BN = T.bn, WM = T.wm, WN = T.wn, STAGES = T.stages;
  constexpr int kSmem = gemm_smem<BM, BN, STAGES, KIND>();
  static_assert(kSmem <= 160 * 1024, "LDS of a CU");
  auto kern = fp8_gemm_kernel<BM, BN, WM, WN, STAGES, KIND, OUT>;
  static std::atomic<uint64_t> known{0};
  const int rc = allow_smem(reinterpret_cast<const void*>(kern), kSmem, dev, known);
  if (rc != kOk) return rc;
  P.mtiles = (P.m - 1) / BM + 1;
  P.ntiles = (P.n - 1) / BN + 1;
  constexpr int kThreads = (BM / WM) * (BN / WN) * 64;
  const int64_t groups = (int64_t)P.mtiles * P.ntiles * P.splits;
  if (!launch_holds(groups, kThreads))
    return set_error(kUnsupported, "dsa_fp8_gemm: %lld tiles take 2^32 threads or more", (long long)groups);
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(kThreads), kSmem, st, P);
  return check_launch("dsa_fp8_gemm");
}

template <int WAVES, int TILES, int KIND, int OUT>
int launch_few(const GemmParams& P, int dev, hipStream_t st) {
  constexpr int kSmem = WAVES * kFewWave<TILES>;
  static_assert(kSmem <= 160 * 1024 && WAVES >= 4, "LDS of a CU, and 256 threads to join");
  const int64_t groups = (P.n - 1) / kFew + 1;
  if (!launch_holds(groups, WAVES * 64))
    return set_error(kUnsupported, "dsa_fp8_gemm: %d columns of few rows take 2^32 threads or more", P.n);
  auto kern = fp8_gemm_few_kernel<WAVES, TILES, KIND, OUT>;
  static std::atomic<uint64_t> known{0};
  const int rc = allow_smem(reinterpret_cast<const void*>(kern), kSmem, dev, known);
  if (rc != kOk) return rc;
  hipLaunchKernelGGL(kern, dim3((unsigned)groups), dim3(WAVES * 64), kSmem, st, P);
  return check_launch("dsa_fp8_gemm");
}

// The kernel of tile `tile`.
template <int KIND, int OUT, int I = 0>
int launch_one(int tile, const GemmParams& P, int dev, hipStream_t st) {
  if constexpr (I + 1 < kTileCount<KIND>) {
    if (tile != I) return launch_one<KIND, OUT, I + 1>(tile, P, dev, st);
  }
  return launch_tile<KIND, I, OUT>(P, dev, st);
}

template <int OUT>
int launch_plan(const Plan& p, int kind, const GemmParams& P, int dev, hipStream_t st) {
  if (p.tile == kFewTile) {
    if (kind == kScaleE8M0)
      return P.m > kFew        ? launch_few<4, 2, kScaleE8M0, OUT>(P, dev, st)
             : p.splits == 8 ? launch_few<8, 1, kScaleE8M0, OUT>(P, dev, st)
                             : launch_few<4, 1, kScaleE8M0, OUT>(P, dev, st);
    return P.m > kFew        ? launch_few<4, 2, kScaleF32, OUT>(P, dev, st)
           : p.splits == 8 ? launch_few<8, 1, kScaleF32, OUT>(P, dev, st)
                           : launch_few<4, 1, kScaleF32, OUT>(P, dev, st);
  }
  return kind == kScaleE8M0 ? launch_one<kScaleE8M0, OUT>(p.tile, P, dev, st) : launch_one<kScaleF32, OUT>(p.tile, P, dev, st);
}

template <int OUT>
void launch_sum(const void* part, int splits, int m, int n, void* out, int64_t out_stride, hipStream_t st) {
  const int64_t threads = (int64_t)m * ((n - 1) / 4 + 1);
  hipLaunchKernelGGL(fp8_gemm_sum_kernel<OUT>, dim3((unsigned)((threads + kSumThreads - 1) / kSumThreads)),
                     dim3(kSumThreads), 0, st, static_cast<const float*>(part), splits, m, n, out, out_stride);
}

}  // namespace
}  // namespace dsa

extern "C" {

size_t dsa_fp8_gemm_workspace_bytes(int m, int n, int k, int scale_kind) {
  using namespace dsa;
  if (m <= 0 || n <= 0 || k <= 0 || (scale_kind != kScaleF32 && scale_kind != kScaleE8M0)) return 0;
  return workspace_of(plan_of(m, n, k, scale_kind, device_cus(current_device())), m, n);
}

int dsa_fp8_gemm_plan(int m, int n, int k, int scale_kind, int cus, int* out) {
  using namespace dsa;
  if (m <= 0 || n <= 0 || k <= 0 || cus < 0 || (scale_kind != kScaleF32 && scale_kind != kScaleE8M0) || !out)
    return set_error(kInvalidArgument, "dsa_fp8_gemm_plan: bad arguments");
  const Plan p = plan_of(m, n, k, scale_kind, cus ? cus : device_cus(current_device()));
  if (p.tile == kFewTile) {
    const int few[5] = {m > kFew ? 2 * kFew : kFew, kFew, p.splits, 2, 1};
    std::copy(few, few + 5, out);
  } else {
    const Tile& T = tiles_of(scale_kind)[p.tile];
    const int tile[5] = {T.bm, T.bn, T.bm / T.wm * (T.bn / T.wn), T.stages, p.splits};
    std::copy(tile, tile + 5, out);
  }
  return kOk;
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
  if ((m > 1 && a_stride > kMaxStride) || (n > 1 && b_stride > kMaxStride))
    return set_error(kUnsupported, "dsa_fp8_gemm: rows more than %d bytes apart", kMaxStride);
  if ((scale_kind == kScaleF32 && ((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) & 3)) ||
      (reinterpret_cast<uintptr_t>(out) & (out_is_f32 ? 3 : 1)))
    return set_error(kInvalidArgument, "dsa_fp8_gemm: pointers must be aligned to their elements");
  const int dev = current_device();
  const Plan p = plan_of(m, n, k, scale_kind, device_cus(dev));
  const size_t need = workspace_of(p, m, n);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(kWorkspaceTooSmall, "dsa_fp8_gemm: workspace %zu bytes, %zu needed", workspace_bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 15))
    return set_error(kInvalidArgument, "dsa_fp8_gemm: the workspace must be 16-byte aligned");
  GemmParams P = {a, b, m > 1 ? a_stride : k, n > 1 ? b_stride : k, a_scale, b_scale, a_scale_stride, b_scale_stride,
                  m, n, k, kblocks, 0, 0, p.tile == kFewTile ? 1 : p.splits, out, out_stride};
  const hipStream_t st = (hipStream_t)stream;
  if (p.tile == kFewTile || p.splits == 1)
    return out_is_f32 ? launch_plan<kOutF32>(p, scale_kind, P, dev, st) : launch_plan<kOutBf16>(p, scale_kind, P, dev, st);
  P.out = workspace;
  P.out_stride = n;
  const int rc = launch_plan<kOutF32>(p, scale_kind, P, dev, st);
  if (rc != kOk) return rc;
  if (out_is_f32) launch_sum<kOutF32>(workspace, p.splits, m, n, out, out_stride, st);
  else launch_sum<kOutBf16>(workspace, p.splits, m, n, out, out_stride, st);
  return check_launch("dsa_fp8_gemm");
}

}  // extern "C"
