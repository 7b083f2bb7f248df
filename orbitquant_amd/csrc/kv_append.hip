// New tokens' keys and values into the 4-bit cache, the key normed and turned to its position on the way, and the queries with them.
// (No counterpart in the reference, which has no cache.)
#include "qk_rotary.h"
#include "qk_rotary_calls.h"

namespace oq {
namespace {

// Where a lane's sixteen values of a vector are (its part p of D / 16):
//   IN_A_ROW   16 p .. 16 p + 15, which are eight pairs of neighbours
//   IN_HALVES  8 p .. and D / 2 + 8 p .., which are eight pairs of halves where all of the head is turned (or nothing is)
//   THROUGH_LDS  a key's as its pairs are, and then in a row: the pairs' halves are not where the transform wants them
// So no key waits for a lane that has its other half, but where only a part of a head is turned.
enum KvLayout { IN_A_ROW, IN_HALVES, THROUGH_LDS };

template <int DT, int LAYOUT>
__device__ __forceinline__ void load_vector(const void *p, int64_t at, int part, int dim, bool wide, float (&y)[16]) {
  load8<DT>(p, at + (LAYOUT == IN_HALVES ? 8 : 16) * part, wide, y);
  load8<DT>(p, at + (LAYOUT == IN_HALVES ? dim / 2 + 8 * part : 16 * part + 8), wide, y + 8);
}

// The workgroups of kv_write (one head of sixteen tokens each), whose keys go through the norm and the rotation first, and behind them
// those of the queries.  A wavefront has keys or values, never both.  MI355X, 8192 tokens, 32 query heads on 8 of 128, bf16, 181 MB: 38.3 us, 4.7 TB/s (a copy
// of as many bytes 35); vector instructions issue in 89 % of the cycles, twenty a value.  One token 4.4 us, of them some 2 the launch.
// In fp16 38.5, in fp32 70 (331 MB); half of the head turned, through LDS, 41, 40 and 73.
// Pieces are of eight values or of one.  Where four at a time would do (parts of four pairs and not of eight, vectors that begin on eight bytes) they go one by one, four times as long:
// 72 of 128 dimensions turned as halves 157 us, all of them from bf16 vectors that begin on eight bytes 130.  (qk_norm_rotary, which has pieces of four, 37 and 34 us.)
template <int D, int DT, int LAYOUT, int PIECE>
__global__ __launch_bounds__(kv_write_threads(D)) void kv_append_kernel(KvAppendArgs a) {
  constexpr int E = 16, L = D / E, THREADS = kv_write_threads(D);
  constexpr int AT_ONCE = THREADS / L, PASSES = 2 * kKvGroup / AT_ONCE;
  __shared__ KvPlace places[kKvGroup];
  __shared__ uint32_t bytes[kKvGroup][D / 8 + 1];
  __shared__ __attribute__((aligned(16))) float turned[LAYOUT == THROUGH_LDS ? kKvGroup : 1][LAYOUT == THROUGH_LDS ? D + 4 : 1];
  if (blockIdx.x >= a.kv_blocks) {
    qk_block<DT, L, qk_form(LAYOUT == IN_A_ROW, L, PIECE), PIECE, true, THREADS>(a.how, a.q, 0, a.write.tokens, D, blockIdx.x - a.kv_blocks);
    return;
  }
  const KvWriteArgs &w = a.write;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), part = qk_part_of<L>(lane);
  const int head = blockIdx.x % w.cache.heads;
  const int64_t first = static_cast<int64_t>(blockIdx.x / w.cache.heads) * kKvGroup;
  float y[PASSES][E];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int base = p * AT_ONCE + wave * (64 / L), vector = base + qk_vector_of<L>(lane);
    const int64_t token = min(first + (vector & (kKvGroup - 1)), w.tokens - 1);
    if (base >= kKvGroup) {
      load_vector<DT, LAYOUT>(w.v, token * w.v_token_stride + head * w.v_head_stride, part, D, w.v_wide, y[p]);
    } else {
      const int64_t at = token * w.k_token_stride + head * w.k_head_stride;
      float u[8], v[8], wu[8], wv[8];
      constexpr int FORM = LAYOUT == IN_A_ROW ? QK_NEIGHBOURS : QK_HALVES, STRIPE = qk_stripe(DT);
      QkTurn<L, FORM, STRIPE> turn;
      QkWeight<L, FORM, PIECE, STRIPE, true> weight;
      const int position = turn.request(a.how, token);
      QkRaw<DT, L, FORM, PIECE, STRIPE, true> raw;
      raw.request(w.k, at, part, D, a.how);
      weight.request(a.how, 1, part, D);
      turn.load(a.how, token, position, part);
      weight.pairs(a.how, 1, wu, wv);
      raw.pairs(u, v);
      qk_apply(a.how, wu, wv, turn, u, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[p][LAYOUT == IN_A_ROW ? 2 * i : i] = u[i];
        y[p][LAYOUT == IN_A_ROW ? 2 * i + 1 : 8 + i] = v[i];
      }
      if constexpr (LAYOUT == THROUGH_LDS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int2 d = qk_pair(8 * part + i, D, a.how);
          turned[vector][d.x] = u[i];
          turned[vector][d.y] = v[i];
        }
      }
    }
  }
  const uint2 *signs = reinterpret_cast<const uint2 *>(w.cache.signs);
  const uint2 low = signs[LAYOUT == IN_HALVES ? part : 2 * part], high = signs[LAYOUT == IN_HALVES ? D / 16 + part : 2 * part + 1];
  const uint32_t words[4] = {low.x, low.y, high.x, high.y};
  group_places<D>(places, w.cache, w.slots, first, w.tokens, head);
  __syncthreads();
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int base = p * AT_ONCE + wave * (64 / L), vector = base + qk_vector_of<L>(lane), token = vector & (kKvGroup - 1);
    if constexpr (LAYOUT == THROUGH_LDS) {
      if (base < kKvGroup) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
          const float4 v = *reinterpret_cast<const float4 *>(&turned[vector][E * part + i]);
          y[p][i] = v.x; y[p][i + 1] = v.y; y[p][i + 2] = v.z; y[p][i + 3] = v.w;
        }
      }
    }
    times_signs(y[p], words);
    kv_butterflies<D, E, LAYOUT == IN_HALVES>(y[p], lane);
    uint16_t scale;
    uint32_t codes[2];
    kv_encode<D>(y[p], scale, codes);
    const int at_low = LAYOUT == IN_HALVES ? part : 2 * part, at_high = LAYOUT == IN_HALVES ? D / 16 + part : 2 * part + 1;  // dwords of a vector
    const bool there = places[token].slot >= 0;
    const int64_t at = places[token].key;
    if (base >= kKvGroup) {
      bytes[token][at_low] = codes[0];
      bytes[token][at_high] = codes[1];
      if (there && part == 0) w.cache.v_scales[at] = scale;
    } else if (there) {
      uint32_t *const to = reinterpret_cast<uint32_t *>(w.cache.k_codes) + at * (D / 8);
      if constexpr (LAYOUT == IN_HALVES) {
        to[at_low] = codes[0];
        to[at_high] = codes[1];
      } else {
        reinterpret_cast<uint2 *>(to)[part] = make_uint2(codes[0], codes[1]);
      }
      if (part == 0) w.cache.k_scales[at] = scale;
    }
  }
  __syncthreads();
  store_values<D, THREADS>(w.cache, places, bytes);
}

template <int D, int DT, int LAYOUT>
void launch(const KvAppendArgs &a, hipStream_t stream) {
  const dim3 grid(a.kv_blocks + a.q_blocks), block(kv_write_threads(D));
  if (a.how.piece == 8) launch_kernel(kv_append_kernel<D, DT, LAYOUT, 8>, grid, block, 0, stream, a);
  else launch_kernel(kv_append_kernel<D, DT, LAYOUT, 1>, grid, block, 0, stream, a);
}
template <int D, int DT>
void launch(const KvAppendArgs &a, hipStream_t stream) {
  if (a.how.interleaved) launch<D, DT, IN_A_ROW>(a, stream);
  else if (a.how.half == 0 || a.how.half == D / 2) launch<D, DT, IN_HALVES>(a, stream);
  else launch<D, DT, THROUGH_LDS>(a, stream);
}
template <int D>
void launch(const KvAppendArgs &a, int dtype, hipStream_t stream) {
  if (dtype == OQ_F32) launch<D, OQ_F32>(a, stream);
  else if (dtype == OQ_F16) launch<D, OQ_F16>(a, stream);
  else launch<D, OQ_BF16>(a, stream);
}

}  // namespace

int kv_append_dispatch(const KvAppendArgs &a, int dim, int dtype, hipStream_t stream) {
  if (dim == 64) launch<64>(a, dtype, stream);
  else if (dim == 128) launch<128>(a, dtype, stream);
  else launch<256>(a, dtype, stream);
  return check_launch("kv_append");
}

}  // namespace oq
