// Rotary positions of query heads and of the shared key, for gfx950.
//
//   (u, v) = (a cos - b sin, b cos + a sin)
// for the rot / 2 pairs (a, b) of a head at its token's position; pair p turns by the
// table's angle p. Pairs lie beside each other (2p, 2p + 1) or in halves (p, p + rot / 2),
// in the input and in the output each: a layout can change on the way. The output may be the
// input (a row belongs to lanes of one wave, which hold all of it before they write) or
// another tensor, such as the tail of the rows that the attention reads.
//
// A lane takes four pairs of a token (eight neighbouring lanes a line of 128 bytes of a head
// of 64) and turns them in HEADS heads with one read of their cosines and sines. f32
// arithmetic, one rounding to bf16. What bounds it is memory for many rows and the launch
// for few: 8192 tokens x 129 heads of 64 in rows of 192, 270 MB, in 59 us (4.5 TB/s; a plain copy
// of whole rows reaches 5.1); 4 tokens of 128 heads in 2.9 us, most of which is a launch.
#include "dsa_common.h"
#include "../../include/dsa_amd.h"

namespace dsa {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxRot = 512;  // a row within one wave
// From as many lanes as the card holds at a time (256 CUs of 2048), a lane takes four heads: the loads in flight that
// a lane's second turn would have given, and a quarter of the positions and angles read. 8192 tokens x 129 heads of
// 64: 65 us against 81 with one head a lane (two: 68, eight: 75; all with warm caches and before what load_pairs
// says); 1024 tokens: 9.2 and 9.9. Below, more lanes hide more: 128 tokens, 4.2 and 3.5.
constexpr int64_t kManyLanes = 256 * 2048;
constexpr int kManyHeads = 4;

struct RopeParams {
  const uint16_t* x[2];  // queries, keys (may be null: no heads)
  uint16_t* out[2];
  int64_t x_token[2], x_head[2], out_token[2], out_head[2];
  int heads[2];
  int64_t tokens;
  int rot;
  const float* table;
  int64_t table_rows;
  const void* positions;
  int wide;
  int lanes;       // a row's lanes: a power of two, four pairs each
  int lane_shift;
  int groups;      // groups of heads of a token: queries' ones, then the keys'
  int q_groups;
};

__device__ __forceinline__ float lo_f32(int v) { return __uint_as_float((uint32_t)v << 16); }
__device__ __forceinline__ float hi_f32(int v) { return __uint_as_float((uint32_t)v & 0xffff0000u); }

// The value of the other lane of two neighbours (both of them active).
__device__ __forceinline__ int neighbour(int v) { return __builtin_amdgcn_mov_dpp(v, 0xb1, 15, 15, true); }

// Pairs p .. p + 3 of a row (half = rot / 2 pairs). VEC: rot a multiple of eight, rows 16-byte aligned.
// Halves take 8 bytes a lane from each; where half is a multiple of eight, two neighbouring lanes share 16 of one half
// and 16 of the other (8192 tokens x 129 heads, stored so: 70 us against 73). Each element is read once, past the L2:
// 70 -> 59 (stores past it too: 63).
template <bool PAIRS, bool VEC>
__device__ __forceinline__ void load_pairs(const uint16_t* row, int p, int half, float* a, float* b) {
  if (VEC) {
    if (p >= half) return;
    if (PAIRS) {
      const v4i v = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(row + 2 * p));
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = lo_f32(v[j]), b[j] = hi_f32(v[j]);
    } else {
      v2i u, w;
      if (half % 8 == 0) {
        const bool odd = p & 4;
        const v4i own = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(row + (odd ? half + p - 4 : p)));
        const int got0 = neighbour(odd ? own[0] : own[2]), got1 = neighbour(odd ? own[1] : own[3]);
        u = odd ? (v2i){got0, got1} : (v2i){own[0], own[1]};
        w = odd ? (v2i){own[2], own[3]} : (v2i){got0, got1};
      } else {
        u = *reinterpret_cast<const v2i*>(row + p);
        w = *reinterpret_cast<const v2i*>(row + half + p);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        a[2 * j] = lo_f32(u[j]), a[2 * j + 1] = hi_f32(u[j]);
        b[2 * j] = lo_f32(w[j]), b[2 * j + 1] = hi_f32(w[j]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (p + j < half) {
        a[j] = bf16_to_f32(row[PAIRS ? 2 * (p + j) : p + j]);
        b[j] = bf16_to_f32(row[PAIRS ? 2 * (p + j) + 1 : half + p + j]);
      }
  }
}

template <bool PAIRS, bool VEC>
__device__ __forceinline__ void store_pairs(uint16_t* row, int p, int half, const float* u, const float* v) {
  if (VEC) {
    if (p >= half) return;
    if (PAIRS) {
      *reinterpret_cast<v4i*>(row + 2 * p) =
          (v4i){pack2(u[0], v[0]), pack2(u[1], v[1]), pack2(u[2], v[2]), pack2(u[3], v[3])};
    } else {
      const v2i x = {pack2(u[0], u[1]), pack2(u[2], u[3])}, y = {pack2(v[0], v[1]), pack2(v[2], v[3])};
      if (half % 8 == 0) {
        const bool odd = p & 4;
        const int got0 = neighbour(odd ? x[0] : y[0]), got1 = neighbour(odd ? x[1] : y[1]);
        *reinterpret_cast<v4i*>(row + (odd ? half + p - 4 : p)) =
            odd ? (v4i){got0, got1, y[0], y[1]} : (v4i){x[0], x[1], got0, got1};
      } else {
        *reinterpret_cast<v2i*>(row + p) = x;
        *reinterpret_cast<v2i*>(row + half + p) = y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (p + j < half) {
        const int w = pack2(u[j], v[j]);
        row[PAIRS ? 2 * (p + j) : p + j] = (uint16_t)w;
        row[PAIRS ? 2 * (p + j) + 1 : half + p + j] = (uint16_t)((uint32_t)w >> 16);
      }
  }
}

template <bool PAIRS, bool OUT_PAIRS, bool VEC, int HEADS>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams P) {
  // rows (a token's group of heads each) stay under 2^31: a 32-bit division
  const uint32_t at = (uint32_t)(((uint64_t)blockIdx.x * kRopeThreads + threadIdx.x) >> P.lane_shift);
  const uint32_t in_order = at / (uint32_t)P.groups;
  const int64_t token = in_order;
  if (token >= P.tokens) return;  // a row's lanes together
  int g = (int)(at - in_order * (uint32_t)P.groups);
  const int which = g >= P.q_groups;
  if (which) g -= P.q_groups;
  const int half = P.rot >> 1, p = 4 * (threadIdx.x & (P.lanes - 1));
  const int heads = P.heads[which];
  const uint16_t* x = P.x[which] + token * P.x_token[which];
  uint16_t* out = P.out[which] + token * P.out_token[which];

  float a[HEADS][4], b[HEADS][4], cos[4], sin[4];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = g * HEADS + i;
    if (h < heads) load_pairs<PAIRS, VEC>(x + h * P.x_head[which], p, half, a[i], b[i]);
  }
  int64_t pos = P.wide ? static_cast<const int64_t*>(P.positions)[token]
                       : (int64_t)static_cast<const int32_t*>(P.positions)[token];
  pos = pos < 0 ? 0 : pos >= P.table_rows ? P.table_rows - 1 : pos;
  const float* row = P.table + pos * P.rot;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int i = VEC ? (p < half ? p + j : j) : p + j < half ? p + j : 0;
    cos[j] = row[i];
    sin[j] = row[half + i];
  }
  asm volatile("" ::: "memory");  // where the output is the input: rows are read before they are written
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = g * HEADS + i;
    if (h >= heads) break;
    float u[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[j] = a[i][j] * cos[j] - b[i][j] * sin[j];
      v[j] = b[i][j] * cos[j] + a[i][j] * sin[j];
    }
    store_pairs<OUT_PAIRS, VEC>(out + h * P.out_head[which], p, half, u, v);
  }
}

template <int HEADS>
int launch_rope(RopeParams P, bool pairs, bool out_pairs, bool vec, hipStream_t st) {
  P.q_groups = (P.heads[0] + HEADS - 1) / HEADS;
  P.groups = P.q_groups + (P.heads[1] + HEADS - 1) / HEADS;
  const int64_t groups = (P.tokens * P.groups * P.lanes + kRopeThreads - 1) / kRopeThreads;
  if (!launch_holds(groups, kRopeThreads))
    return set_error(kUnsupported, "dsa_rope: %lld tokens of %d heads take 2^32 threads or more", (long long)P.tokens,
                     P.heads[0] + P.heads[1]);
  const dim3 grid((unsigned)groups), block(kRopeThreads);
#define DSA_ROPE(A, B, V) hipLaunchKernelGGL((rope_kernel<A, B, V, HEADS>), grid, block, 0, st, P)
  if (pairs && out_pairs) { if (vec) DSA_ROPE(true, true, true); else DSA_ROPE(true, true, false); }
  else if (pairs) { if (vec) DSA_ROPE(true, false, true); else DSA_ROPE(true, false, false); }
  else if (out_pairs) { if (vec) DSA_ROPE(false, true, true); else DSA_ROPE(false, true, false); }
  else { if (vec) DSA_ROPE(false, false, true); else DSA_ROPE(false, false, false); }
#undef DSA_ROPE
  return check_launch("dsa_rope");
}

// Rows of rot elements that do not share any: heads within a token's step or tokens within a head's.
bool rope_apart(int64_t tokens, int64_t token, int64_t heads, int64_t head, int rot) {
  if (heads == 0) return true;
  if (tokens <= 1 || heads <= 1) return (tokens <= 1 || token >= rot) && (heads <= 1 || head >= rot);
  return (head >= rot && token >= (heads - 1) * head + rot) || (token >= rot && head >= (tokens - 1) * token + rot);
}

// In place, every row is where it was.
bool rope_in_place(const void* x, int64_t tokens, int64_t token, int64_t heads, int64_t head, const void* out, int64_t out_token,
                   int64_t out_head) {
  return heads == 0 || x != out || ((tokens <= 1 || token == out_token) && (heads <= 1 || head == out_head));
}

bool rope_aligned(const void* p, int64_t token, int64_t head) {
  return !p || (!(reinterpret_cast<uintptr_t>(p) & 15) && !(token & 7) && !(head & 7));
}

}  // namespace
}  // namespace dsa

extern "C" int dsa_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads, void* q_out,
                        int64_t q_out_token_stride, int64_t q_out_head_stride, const void* k, int64_t k_token_stride,
                        int64_t k_head_stride, int k_heads, void* k_out, int64_t k_out_token_stride,
                        int64_t k_out_head_stride, int64_t num_tokens, int rot_dim, const float* cos_sin_cache,
                        int64_t cache_positions, const void* positions, int pos_is_64, int interleaved,
                        int out_interleaved, void* stream) {
  using namespace dsa;
  if (num_tokens < 0 || num_tokens > INT32_MAX || q_heads < 0 || k_heads < 0 || q_heads > 65536 || k_heads > 65536)
    return set_error(kInvalidArgument, "dsa_rope: bad sizes");
  if (rot_dim < 2 || (rot_dim & 1)) return set_error(kInvalidArgument, "dsa_rope: rot_dim %d must be even", rot_dim);
  if (rot_dim > kMaxRot) return set_error(kUnsupported, "dsa_rope: rot_dim %d (at most %d)", rot_dim, kMaxRot);
  if (num_tokens == 0 || q_heads + k_heads == 0) return kOk;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !cos_sin_cache || !positions)
    return set_error(kInvalidArgument, "dsa_rope: null pointer");
  if (cache_positions < 1) return set_error(kInvalidArgument, "dsa_rope: empty cos_sin_cache");
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k) |
        reinterpret_cast<uintptr_t>(k_out)) & 1) ||
      (reinterpret_cast<uintptr_t>(cos_sin_cache) & 3) || (reinterpret_cast<uintptr_t>(positions) & (pos_is_64 ? 7 : 3)))
    return set_error(kInvalidArgument, "dsa_rope: pointers must be aligned to their elements");
  if (!rope_apart(num_tokens, q_out_token_stride, q_heads, q_out_head_stride, rot_dim) ||
      !rope_apart(num_tokens, k_out_token_stride, k_heads, k_out_head_stride, rot_dim))
    return set_error(kInvalidArgument, "dsa_rope: output rows overlap");
  if (!rope_in_place(q, num_tokens, q_token_stride, q_heads, q_head_stride, q_out, q_out_token_stride, q_out_head_stride) ||
      !rope_in_place(k, num_tokens, k_token_stride, k_heads, k_head_stride, k_out, k_out_token_stride, k_out_head_stride))
    return set_error(kInvalidArgument, "dsa_rope: in place, rows need the same strides");
  int lanes = 1, shift = 0;
  while (lanes * 8 < rot_dim) lanes <<= 1, ++shift;
  RopeParams P = {{static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k)},
                  {static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_out)},
                  {q_token_stride, k_token_stride},
                  {q_head_stride, k_head_stride},
                  {q_out_token_stride, k_out_token_stride},
                  {q_out_head_stride, k_out_head_stride},
                  {q_heads, k_heads},
                  num_tokens, rot_dim, cos_sin_cache, cache_positions, positions, pos_is_64, lanes, shift, 0, 0};
  const bool vec = rot_dim % 8 == 0 && rope_aligned(q_heads ? q : nullptr, q_token_stride, q_head_stride) &&
                   rope_aligned(q_heads ? q_out : nullptr, q_out_token_stride, q_out_head_stride) &&
                   rope_aligned(k_heads ? k : nullptr, k_token_stride, k_head_stride) &&
                   rope_aligned(k_heads ? k_out : nullptr, k_out_token_stride, k_out_head_stride);
  if (num_tokens * (q_heads + k_heads) >= INT32_MAX - kRopeThreads)
    return set_error(kUnsupported, "dsa_rope: 2^31 heads of all tokens or more");
  const bool many = num_tokens * (q_heads + k_heads) * lanes >= kManyLanes;
  return many ? launch_rope<kManyHeads>(P, interleaved, out_interleaved, vec, (hipStream_t)stream)
              : launch_rope<1>(P, interleaved, out_interleaved, vec, (hipStream_t)stream);
}
