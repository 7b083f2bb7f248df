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
// A lane holds eight pairs, `L` = 1, 2, 4, ... 32 lanes a head: both halves of every pair are in one lane, the rotation needs no other, and
// the sums need log2(L) exchanges.
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
  bool weight_wide;
  bool norm, interleaved;
  float eps, by_dim;           // by_dim: 1 / D
};

struct QkSide {  // queries, or keys
  const void *x;
  void *out;                   // [tokens, heads, D]
  int64_t token_stride, head_stride;
  int heads, groups;           // groups of kQkHeads heads
  uint32_t magic;              // of a division by `groups`: ceil(2^32 / groups)
  bool wide;                   // eight values begin on 16 bytes, in x and in out
};

constexpr int kQkHeads = 4;    // of a token a lane, which share its entries of the tables and the weights

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

template <int X>
__device__ __forceinline__ float qk_swap_sum(float x) {
  const kv_u32x2 both = kv_swap<X>(__float_as_uint(x), __float_as_uint(x));
  return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}
template <int CTRL>
__device__ __forceinline__ float qk_dpp_sum(float x) { return x + __uint_as_float(kv_dpp<CTRL>(__float_as_uint(x))); }

// Of a head's squares, in the order above.
template <int L>
__device__ __forceinline__ float qk_square_sum(const float (&a)[8], const float (&b)[8]) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = a[i] * a[i] + b[i] * b[i];
#pragma unroll
  for (int d = 4; d > 0; d /= 2) {
#pragma unroll
    for (int i = 0; i < d; ++i) s[i] = s[i] + s[i + d];
  }
  float sum = s[0];
  if constexpr (L >= 2) sum = qk_dpp_sum<kDppXor1>(sum);
  if constexpr (L >= 4) sum = qk_dpp_sum<kDppXor2>(sum);
  if constexpr (L == 32) sum = qk_dpp_sum<kDppXor8>(sum);
  if constexpr (L >= 16) sum = qk_swap_sum<16>(sum);
  if constexpr (L >= 8) sum = qk_swap_sum<32>(sum);
  return sum;
}

// The dimensions of pair p.
__device__ __forceinline__ int2 qk_pair(int p, int dim, const QkNormRotary &how) {
  if (how.interleaved) return make_int2(2 * p, 2 * p + 1);
  if (how.half == 0) return make_int2(p, p + dim / 2);
  return p < how.half ? make_int2(p, p + how.half) : make_int2(p + how.half, p + dim / 2);
}

// Eight values that begin on 16 bytes, of a type that is known when the call comes.
__device__ __forceinline__ void qk_load8(const void *p, int dtype, int64_t at, bool wide, float *y) {
  if (dtype == OQ_F32) load8<OQ_F32>(p, at, wide, y);
  else if (dtype == OQ_F16) load8<OQ_F16>(p, at, wide, y);
  else load8<OQ_BF16>(p, at, wide, y);
}

// A lane's pairs 8 * part .. of the vector at `at`; `load`: eight values in a row, or one.
template <typename Load8, typename Load1>
__device__ __forceinline__ void qk_load_pairs(int part, int dim, const QkNormRotary &how, bool wide, float (&a)[8], float (&b)[8], const Load8 &eight, const Load1 &one) {
  if (wide) {
    const bool there = 16 * part < dim;
    if (how.interleaved) {
      float v[16];
      if (there) {
        eight(16 * part, v);
        eight(16 * part + 8, v + 8);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = there ? v[2 * i] : 0.0f;
        b[i] = there ? v[2 * i + 1] : 0.0f;
      }
    } else {
      const int2 at = qk_pair(8 * part, dim, how);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.0f;
      if (there) {
        eight(at.x, a);
        eight(at.y, b);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = 8 * part + i;
      const int2 at = qk_pair(p, dim, how);
      a[i] = 2 * p < dim ? one(at.x) : 0.0f;
      b[i] = 2 * p < dim ? one(at.y) : 0.0f;
    }
  }
}

template <int DT>
__device__ __forceinline__ void qk_load_vector(const void *x, int64_t at, int part, int dim, const QkNormRotary &how, bool wide, float (&a)[8], float (&b)[8]) {
  qk_load_pairs(part, dim, how, wide, a, b, [&](int d, float *y) { load8<DT>(x, at + d, true, y); }, [&](int d) { return load_as_f32<DT>(x, at + d); });
}
__device__ __forceinline__ void qk_load_weight(const QkNormRotary &how, int side, int part, int dim, float (&a)[8], float (&b)[8]) {
  const void *const w = how.weight[side];
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = b[i] = 1.0f;
  } else {
    qk_load_pairs(part, dim, how, how.weight_wide, a, b, [&](int d, float *y) { qk_load8(w, how.weight_dtype, d, true, y); },
                  [&](int d) { return load_dyn_f32(w, how.weight_dtype, d); });
  }
}

// A token's row of the tables, eight entries of a lane.  A negative position (a token of no request) turns nothing, one behind the tables makes NaN.
struct QkTurn {
  float c[8], s[8];
  bool turns;
  __device__ __forceinline__ void load(const QkNormRotary &how, int64_t token, int part) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = 1.0f;
      s[i] = 0.0f;
    }
    turns = false;
    if (how.half == 0) return;
    const int64_t row = how.positions != nullptr ? how.positions[token] : token;
    if (row < 0) return;
    turns = true;
    if (row >= how.rows) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = NAN;
      return;
    }
    const int64_t at = row * how.half + 8 * part;
    if (how.table_wide) {
      if (8 * part < how.half) {
        load8<OQ_F32>(how.cos, at, true, c);
        load8<OQ_F32>(how.sin, at, true, s);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (8 * part + i < how.half) {
          c[i] = how.cos[at + i];
          s[i] = how.sin[at + i];
        }
      }
    }
  }
};

template <int L>
__device__ __forceinline__ void qk_apply(const QkNormRotary &how, int part, const float (&wa)[8], const float (&wb)[8], const QkTurn &turn, float (&a)[8], float (&b)[8]) {
  if (how.norm) {
    const float r = 1.0f / sqrtf(qk_square_sum<L>(a, b) * how.by_dim + how.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = a[i] * r * wa[i];
      b[i] = b[i] * r * wb[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float u = a[i] * turn.c[i] - b[i] * turn.s[i], v = b[i] * turn.c[i] + a[i] * turn.s[i];
    const bool turned = turn.turns && 8 * part + i < how.half;  // (what is not may be an infinity, which a sine of zero does not leave alone)
    a[i] = turned ? u : a[i];
    b[i] = turned ? v : b[i];
  }
}

template <int DT>
__device__ __forceinline__ void qk_store_vector(void *out, int64_t at, int part, int dim, const QkNormRotary &how, bool wide, const float (&a)[8], const float (&b)[8]) {
  if (wide) {
    if (16 * part >= dim) return;
    if (how.interleaved) {
      float v[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[2 * i] = a[i];
        v[2 * i + 1] = b[i];
      }
      store8<DT>(out, at + 16 * part, v);
      store8<DT>(out, at + 16 * part + 8, v + 8);
    } else {
      const int2 d = qk_pair(8 * part, dim, how);
      store8<DT>(out, at + d.x, a);
      store8<DT>(out, at + d.y, b);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = 8 * part + i;
      if (2 * p < dim) {
        const int2 d = qk_pair(p, dim, how);
        store_from_f32<DT>(out, at + d.x, a[i]);
        store_from_f32<DT>(out, at + d.y, b[i]);
      }
    }
  }
}

// Workgroup `block` of a side: four heads of a token for every L lanes.
template <int DT, int L, int THREADS>
__device__ __forceinline__ void qk_block(const QkNormRotary &how, const QkSide &side, int which, int64_t tokens, int dim, uint32_t block) {
  constexpr int UNITS = THREADS / L;
  const int lane = threadIdx.x & 63, part = qk_part_of<L>(lane);
  const uint32_t first = block * UNITS, local = (threadIdx.x >> 6) * (64 / L) + qk_vector_of<L>(lane);
  const uint32_t groups = side.groups, row = first / groups, n = first - row * groups + local;  // (n < groups + 256: the product by the reciprocal is exact)
  const uint32_t down = groups == 1 ? n : __umulhi(n, side.magic);
  const int64_t token = static_cast<int64_t>(row) + down;
  const int head = static_cast<int>(n - down * groups) * kQkHeads;
  const bool there = token < tokens;
  float a[kQkHeads][8], b[kQkHeads][8], wa[8], wb[8];
  QkTurn turn;
  if (there) {
    const int64_t at = token * side.token_stride;
#pragma unroll
    for (int h = 0; h < kQkHeads; ++h) qk_load_vector<DT>(side.x, at + min(head + h, side.heads - 1) * side.head_stride, part, dim, how, side.wide, a[h], b[h]);
    turn.load(how, token, part);
    qk_load_weight(how, which, part, dim, wa, wb);
  }
#pragma unroll
  for (int h = 0; h < kQkHeads; ++h) {
    if (h > 0 && head + h >= side.heads) break;  // (a unit's lanes agree, and their sums are theirs)
    qk_apply<L>(how, part, wa, wb, turn, a[h], b[h]);
    if (there) qk_store_vector<DT>(side.out, (token * side.heads + head + h) * dim, part, dim, how, side.wide, a[h], b[h]);
  }
}

}  // namespace oq
