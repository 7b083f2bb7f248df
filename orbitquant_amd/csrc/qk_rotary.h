// Norms of queries and keys for each head, with the rotary positions in the same pass.
//
// A head's D values are D/2 pairs (x0, x1): dimensions 2p and 2p+1 (interleaved), or p and p + R/2 of the first R dimensions and
// p and p + (D-R)/2 of the rest.
//   s = sum of x^2 over the head;  r = 1 / sqrt(s / D + eps);  y = (x r) w
//   of the first R/2 pairs:  (y0, y1) -> (y0 c - y1 s', y1 c + y0 s')          c, s': the position's row of the tables
// in fp32, every product and sum rounded by itself, whatever the inputs' type: the value is rounded once, when it is stored (or, a key on its
// way into the 4-bit cache, when it becomes a code).  s is added up in one order everywhere: the two squares of a pair, then pairs 4, 2, 1
// apart of each eight, then eights 1, 2, 4, ... apart, zeros behind the last pair.  So a key's codes do not depend on the launch that made them.
//
// A lane holds eight pairs, `L` = 1, 2, 4, ... 32 lanes a head: both values of every pair are in one lane, the rotation needs no other, and
// the sums need log2(L) exchanges.  Bound by memory: 32760 tokens, 40 heads of 128 for queries and keys each, bf16, 1.36 GB, 249 us (neighbours 252, as many
// bytes in fp32 245), 5.4 TB/s, where a copy of the library reaches 5.2; vector instructions issue in 72 % of the cycles.  Few tokens by latency, 3.1 us for one.
// (Converted as they were fetched, head by head, 352 us; four heads a lane 260.)
#pragma once

#include "kv_rows.h"

namespace oq {

// Where the entry points' tensors are.
struct QkNormRotary {
  const float *cos, *sin;      // [rows, half]
  const int32_t *positions;    // NULL: token t is at t
  int64_t rows;
  int half;                    // R / 2; 0: nothing is turned
  bool table_wide;             // eight entries begin on 16 bytes
  const void *weight[2];       // of queries and of keys; NULL: ones
  int weight_dtype;
  int piece;                   // values fetched at once, of all that is fetched: 8, 4 or 1
  bool norm, interleaved;
  float eps, by_dim;           // by_dim: 1 / D
};

struct QkSide {  // queries, or keys
  const void *x;
  void *out;                   // [tokens, heads, D]
  int64_t token_stride, head_stride;
  int heads, groups, each;     // groups of `each` heads: kQkHeads or 1
  uint32_t magic;              // of a division by `groups`: ceil(2^32 / groups)
};

// Heads of a token that a lane takes, which share its entries of the tables and the weights; where there are few, one: what a wavefront then waits
// for is its own instructions (one token, 32 heads and 8, 5.2 -> 3.1 us; 1024 tokens are as fast either way).
constexpr int kQkHeads = 2;
constexpr int64_t kQkAlone = 1 << 14;  // heads of all tokens

template <int L>
__device__ __forceinline__ int qk_part_of(int lane) {
  if constexpr (L <= 2) return lane & (L - 1);
  else return kv_part_of<8 * L>(lane);
}
template <int L>
__device__ __forceinline__ int qk_vector_of(int lane) {
  if constexpr (L <= 2) return lane / L;
  else return kv_vector_of<8 * L>(lane);
}

// Which of a head's pairs a lane has (its part of L), and how they are fetched.
//   QK_HALVES      eight in a row, whose first and whose second values lie in a row
//   QK_NEIGHBOURS  eight in a row, sixteen values in a row
//   QK_STRIPES     the same pairs dealt out to the lanes sixteen bytes at a time, so that what all lanes fetch or store at once lies in a row (sixteen values a
//                  lane in a row: as many bytes in fp32 326 us instead of 258)
enum QkForm { QK_HALVES, QK_NEIGHBOURS, QK_STRIPES };
constexpr int qk_form(bool interleaved, int lanes, int piece) { return !interleaved ? QK_HALVES : lanes >= 4 && piece == 8 ? QK_STRIPES : QK_NEIGHBOURS; }
constexpr int qk_stripe(int dt) { return dt == OQ_F32 ? 4 : 8; }  // values

// The i-th pair of a lane; STRIPE: values of a stripe.
template <int L, int FORM, int STRIPE>
__device__ __forceinline__ int qk_pair_of(int part, int i) {
  if constexpr (FORM == QK_STRIPES) return STRIPE / 2 * (L * (i / (STRIPE / 2)) + part) + i % (STRIPE / 2);
  else return 8 * part + i;
}

// Plus what the lane has whose part differs in bit BIT.
template <int L, int BIT>
__device__ __forceinline__ float qk_exchange_sum(float x) {
  constexpr int SWAPS = L == 8 ? 1 : L >= 16 ? 2 : 0, FIRST = L == 32 ? 3 : 2;  // the swaps of lane groups are the last exchanges
  if constexpr ((1 << BIT) >= L) {
    return x;
  } else if constexpr (BIT >= FIRST) {
    constexpr int X = BIT - FIRST == SWAPS - 1 ? 32 : 16;
    const kv_u32x2 both = kv_swap<X>(__float_as_uint(x), __float_as_uint(x));
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
  } else {
    constexpr int CTRL = BIT == 0 ? kDppXor1 : BIT == 1 ? kDppXor2 : kDppXor8;
    return x + __uint_as_float(kv_dpp<CTRL>(__float_as_uint(x)));
  }
}

// Of a head's squares, in the order above.
template <int L, int FORM, int STRIPE>
__device__ __forceinline__ float qk_square_sum(const float (&a)[8], const float (&b)[8]) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = a[i] * a[i] + b[i] * b[i];
  if constexpr (FORM == QK_STRIPES && STRIPE == 8) {  // pairs 4 apart are in the next lane
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = qk_exchange_sum<L, 0>(s[i]);
#pragma unroll
    for (int c = 0; c < 8; c += 4) {
      s[c] = (s[c] + s[c + 2]) + (s[c + 1] + s[c + 3]);
      s[c] = qk_exchange_sum<L, 4>(qk_exchange_sum<L, 3>(qk_exchange_sum<L, 2>(qk_exchange_sum<L, 1>(s[c]))));
    }
    return s[0] + s[4];
  } else if constexpr (FORM == QK_STRIPES) {  // 4 and 2 apart in other lanes
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = qk_exchange_sum<L, 0>(qk_exchange_sum<L, 1>(s[i]));
#pragma unroll
    for (int c = 0; c < 8; c += 2) s[c] = qk_exchange_sum<L, 4>(qk_exchange_sum<L, 3>(qk_exchange_sum<L, 2>(s[c] + s[c + 1])));
    return (s[0] + s[2]) + (s[4] + s[6]);
  } else {
#pragma unroll
    for (int d = 4; d > 0; d /= 2) {
#pragma unroll
      for (int i = 0; i < d; ++i) s[i] = s[i] + s[i + d];
    }
    return qk_exchange_sum<L, 4>(qk_exchange_sum<L, 3>(qk_exchange_sum<L, 2>(qk_exchange_sum<L, 1>(qk_exchange_sum<L, 0>(s[0])))));
  }
}

// The dimensions of pair p.
__device__ __forceinline__ int2 qk_pair(int p, int dim, const QkNormRotary &how) {
  if (how.interleaved) return make_int2(2 * p, 2 * p + 1);
  if (how.half == 0) return make_int2(p, p + dim / 2);
  return p < how.half ? make_int2(p, p + how.half) : make_int2(p + how.half, p + dim / 2);
}

// How a lane's pairs are fetched: PIECE = 8 or 4 values at once, where the first dimensions of the head's parts and its vectors allow it, or one by one.
constexpr int qk_piece_words(int dt, int piece) { return dt == OQ_F32 ? piece : (piece + 1) / 2; }
template <int DT, int PIECE>
__device__ __forceinline__ void qk_fetch(const void *p, int64_t at, uint32_t *w) {
  if constexpr (PIECE == 1) {
    if constexpr (DT == OQ_F32) w[0] = static_cast<const uint32_t *>(p)[at];
    else w[0] = static_cast<const uint16_t *>(p)[at];
  } else {
    constexpr int WORDS = qk_piece_words(DT, PIECE);
    const char *from = static_cast<const char *>(p) + at * (DT == OQ_F32 ? 4 : 2);
    if constexpr (WORDS == 2) {
      const uint2 v = *reinterpret_cast<const uint2 *>(from);
      w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = reinterpret_cast<const uint4 *>(from)[i / 4];
        w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
      }
    }
  }
}

// Sixteen values as they come, requested for all of a lane's heads before the first is looked at.  (STRIPE is the tensors', whatever these values' type.)
// FULL: the lanes have nothing behind the last pair (D = 16 L).
template <int DT, int L, int FORM, int PIECE, int STRIPE, bool FULL>
struct QkRaw {
  static constexpr int AT_ONCE = FORM == QK_STRIPES ? STRIPE : PIECE;
  static constexpr int EACH = qk_piece_words(DT, AT_ONCE), PIECES = 16 / AT_ONCE;
  uint32_t w[PIECES * EACH];

  // Halves: the first values of the eight pairs, then the second ones; otherwise pair by pair.  Zeros behind the last pair.
  __device__ __forceinline__ void request(const void *x, int64_t at, int part, int dim, const QkNormRotary &how) {
    if constexpr (!FULL) {
#pragma unroll
      for (int i = 0; i < PIECES * EACH; ++i) w[i] = 0;
    }
#pragma unroll
    for (int c = 0; c < PIECES; ++c) {
      if constexpr (FORM == QK_HALVES) {
        const int pair = 8 * part + c % (PIECES / 2) * AT_ONCE;
        const int2 d = qk_pair(pair, dim, how);
        if (FULL || 2 * pair < dim) qk_fetch<DT, AT_ONCE>(x, at + (c < PIECES / 2 ? d.x : d.y), w + c * EACH);
      } else {
        const int d = FORM == QK_STRIPES ? STRIPE * (L * c + part) : 16 * part + AT_ONCE * c;
        if (FULL || d < dim) qk_fetch<DT, AT_ONCE>(x, at + d, w + c * EACH);
      }
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (DT == OQ_F32) return __uint_as_float(w[i]);
    else if constexpr (AT_ONCE == 1) return dyn_bits_to_f32(w[i], DT);
    else if constexpr (DT == OQ_BF16) return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return f16_bits_to_f32(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1))));
  }
  __device__ __forceinline__ void pairs(float (&a)[8], float (&b)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = value(FORM == QK_HALVES ? i : 2 * i);
      b[i] = value(FORM == QK_HALVES ? 8 + i : 2 * i + 1);
    }
  }
};

// A norm's weights, as they come and as numbers.  (Their type is looked at twice: what is converted where it is requested is waited for there.)
template <int L, int FORM, int PIECE, int STRIPE, bool FULL>
struct QkWeight {
  QkRaw<OQ_F32, L, FORM, PIECE, STRIPE, FULL> wide;
  QkRaw<OQ_BF16, L, FORM, PIECE, STRIPE, FULL> narrow;
  __device__ __forceinline__ void request(const QkNormRotary &how, int side, int part, int dim) {
    const void *const w = how.weight[side];
    if (w == nullptr) return;
    if (how.weight_dtype == OQ_F32) wide.request(w, 0, part, dim, how);
    else narrow.request(w, 0, part, dim, how);
  }
  __device__ __forceinline__ void pairs(const QkNormRotary &how, int side, float (&a)[8], float (&b)[8]) const {
    if (how.weight[side] == nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 1.0f;
    } else if (how.weight_dtype == OQ_F32) {
      wide.pairs(a, b);
    } else if (how.weight_dtype == OQ_BF16) {
      narrow.pairs(a, b);
    } else {
      QkRaw<OQ_F16, L, FORM, PIECE, STRIPE, FULL> half;
#pragma unroll
      for (int i = 0; i < narrow.PIECES * narrow.EACH; ++i) half.w[i] = narrow.w[i];
      half.pairs(a, b);
    }
  }
};

// A token's row of the tables, eight entries of a lane.  A negative position (a token of no request) turns nothing, one behind the tables makes NaN;
// both read a row that exists, so that no load is in a branch of some lanes.
template <int L, int FORM, int STRIPE>
struct QkTurn {
  float c[8], s[8];
  uint32_t turned;  // a bit for each pair that is
  bool broken;
  // Of a token: requested first, since loads come back in order and the tables' wait for it.
  static __device__ __forceinline__ int request(const QkNormRotary &how, int64_t token) {
    int position = 0;
    if (how.positions != nullptr) position = how.positions[token];
    __builtin_amdgcn_sched_barrier(0);
    return position;
  }
  __device__ __forceinline__ void load(const QkNormRotary &how, int64_t token, int position, int part) {
    constexpr int IN_ROW = FORM == QK_STRIPES ? STRIPE / 2 : 8;  // pairs
    turned = 0;
    broken = false;
    if (how.half == 0) return;
    const int64_t row = how.positions != nullptr ? position : token;
#pragma unroll
    for (int i = 0; i < 8; i += IN_ROW) turned |= ((1u << min(max(how.half - qk_pair_of<L, FORM, STRIPE>(part, i), 0), IN_ROW)) - 1u) << i;
    turned = row >= 0 ? turned : 0;
    broken = row >= how.rows;
    if (how.rows == 0) return;
    const int64_t at = min(max(row, static_cast<int64_t>(0)), how.rows - 1) * how.half;
#pragma unroll
    for (int i = 0; i < 8; i += IN_ROW) {
      if (how.table_wide) {
        const int64_t from = at + min(qk_pair_of<L, FORM, STRIPE>(part, i), how.half - IN_ROW);
#pragma unroll
        for (int e = 0; e < IN_ROW; e += IN_ROW < 4 ? 2 : 4) {
          if constexpr (IN_ROW < 4) {
            const float2 x = *reinterpret_cast<const float2 *>(how.cos + from), y = *reinterpret_cast<const float2 *>(how.sin + from);
            c[i] = x.x; c[i + 1] = x.y; s[i] = y.x; s[i + 1] = y.y;
          } else {
            const float4 x = *reinterpret_cast<const float4 *>(how.cos + from + e), y = *reinterpret_cast<const float4 *>(how.sin + from + e);
            c[i + e] = x.x; c[i + e + 1] = x.y; c[i + e + 2] = x.z; c[i + e + 3] = x.w;
            s[i + e] = y.x; s[i + e + 1] = y.y; s[i + e + 2] = y.z; s[i + e + 3] = y.w;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < IN_ROW; ++e) {
          const int64_t from = at + min(qk_pair_of<L, FORM, STRIPE>(part, i + e), how.half - 1);
          c[i + e] = how.cos[from];
          s[i + e] = how.sin[from];
        }
      }
    }
  }
};

template <int L, int FORM, int STRIPE>
__device__ __forceinline__ void qk_apply(const QkNormRotary &how, const float (&wa)[8], const float (&wb)[8], const QkTurn<L, FORM, STRIPE> &turn, float (&a)[8], float (&b)[8]) {
  if (how.norm) {
    const float r = 1.0f / sqrtf(qk_square_sum<L, FORM, STRIPE>(a, b) * how.by_dim + how.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = a[i] * r * wa[i];
      b[i] = b[i] * r * wb[i];
    }
  }
  if (how.half == 0) return;
  if (turn.turned == 0xffu && !turn.broken) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = a[i] * turn.c[i] - b[i] * turn.s[i];
      b[i] = b[i] * turn.c[i] + a[i] * turn.s[i];
      a[i] = u;
    }
    return;
  }
  if (turn.broken) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = turn.turned >> i & 1 ? NAN : a[i];
      b[i] = turn.turned >> i & 1 ? NAN : b[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = a[i] * turn.c[i] - b[i] * turn.s[i], v = b[i] * turn.c[i] + a[i] * turn.s[i];
    a[i] = turn.turned >> i & 1 ? u : a[i];
    b[i] = turn.turned >> i & 1 ? v : b[i];
  }
}

template <int DT, int PIECE>
__device__ __forceinline__ void qk_put(void *p, int64_t at, const float *y) {
  if constexpr (PIECE == 8) {
    store8<DT>(p, at, y);
  } else if constexpr (PIECE == 1) {
    store_from_f32<DT>(p, at, y[0]);
  } else if constexpr (DT == OQ_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(p) + at) = make_float4(y[0], y[1], y[2], y[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = DT == OQ_F16 ? f32_to_f16_bits(y[2 * i]) | static_cast<uint32_t>(f32_to_f16_bits(y[2 * i + 1])) << 16
                          : f32_to_bf16_bits(y[2 * i]) | static_cast<uint32_t>(f32_to_bf16_bits(y[2 * i + 1])) << 16;
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + at) = make_uint2(w[0], w[1]);
  }
}
template <int DT, int L, int FORM, int PIECE, int STRIPE, bool FULL>
__device__ __forceinline__ void qk_store_pairs(void *out, int64_t at, int part, int dim, const QkNormRotary &how, const float (&a)[8], const float (&b)[8]) {
  if constexpr (FORM == QK_HALVES) {
#pragma unroll
    for (int i = 0; i < 8; i += PIECE) {
      const int pair = 8 * part + i;
      const int2 d = qk_pair(pair, dim, how);
      if (FULL || 2 * pair < dim) {
        qk_put<DT, PIECE>(out, at + d.x, a + i);
        qk_put<DT, PIECE>(out, at + d.y, b + i);
      }
    }
  } else {
    constexpr int AT_ONCE = FORM == QK_STRIPES ? STRIPE : PIECE;
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[2 * i] = a[i];
      v[2 * i + 1] = b[i];
    }
#pragma unroll
    for (int i = 0; i < 16; i += AT_ONCE) {
      const int d = FORM == QK_STRIPES ? STRIPE * (L * (i / STRIPE) + part) : 16 * part + i;
      if (FULL || d < dim) qk_put<DT, AT_ONCE>(out, at + d, v + i);
    }
  }
}

// Workgroup `block` of a side: HEADS heads of a token for every L lanes.
template <int DT, int L, int FORM, int PIECE, bool FULL, int THREADS, int HEADS>
__device__ __forceinline__ void qk_heads_block(const QkNormRotary &how, const QkSide &side, int which, int64_t tokens, int dim, uint32_t block) {
  constexpr int UNITS = THREADS / L, STRIPE = qk_stripe(DT);
  const int lane = threadIdx.x & 63, part = qk_part_of<L>(lane);
  const uint32_t first = block * UNITS, local = (threadIdx.x >> 6) * (64 / L) + qk_vector_of<L>(lane);
  const uint32_t groups = side.groups, row = first / groups, n = first - row * groups + local;  // (n < groups + 256: the product by the reciprocal is exact)
  const uint32_t down = groups == 1 ? n : __umulhi(n, side.magic);
  const int64_t token = static_cast<int64_t>(row) + down;
  const int head = static_cast<int>(n - down * groups) * HEADS;
  if (token >= tokens) return;  // (all of a unit's lanes)
  QkRaw<DT, L, FORM, PIECE, STRIPE, FULL> raw[HEADS];
  float wa[8], wb[8];
  QkTurn<L, FORM, STRIPE> turn;
  QkWeight<L, FORM, PIECE, STRIPE, FULL> weight;
  const int position = turn.request(how, token);
  const int64_t at = token * side.token_stride;
#pragma unroll
  for (int h = 0; h < HEADS; ++h) raw[h].request(side.x, at + min(head + h, side.heads - 1) * side.head_stride, part, dim, how);
  weight.request(how, which, part, dim);
  turn.load(how, token, position, part);
  weight.pairs(how, which, wa, wb);
#pragma unroll
  for (int h = 0; h < HEADS; ++h) {
    if (h > 0 && head + h >= side.heads) break;
    float a[8], b[8];
    raw[h].pairs(a, b);
    qk_apply(how, wa, wb, turn, a, b);
    qk_store_pairs<DT, L, FORM, PIECE, STRIPE, FULL>(side.out, (token * side.heads + head + h) * dim, part, dim, how, a, b);
  }
}
template <int DT, int L, int FORM, int PIECE, bool FULL, int THREADS>
__device__ __forceinline__ void qk_block(const QkNormRotary &how, const QkSide &side, int which, int64_t tokens, int dim, uint32_t block) {
  if (side.each == 1) qk_heads_block<DT, L, FORM, PIECE, FULL, THREADS, 1>(how, side, which, tokens, dim, block);
  else qk_heads_block<DT, L, FORM, PIECE, FULL, THREADS, kQkHeads>(how, side, which, tokens, dim, block);
}

}  // namespace oq
