// The 4-bit key/value cache: layout, and the arithmetic that a vector goes through on its way in and out.
//
// A token's key or value of one head, x[D] (D = 64, 128 or 256), is held in the rotated space y = H(signs * x), H the
// unnormalised Walsh-Hadamard transform, as one bf16 scale a and D codes of four bits: E2M1, whose values
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 (and a sign) gfx950 converts to a pair of fp16 values, exactly, in one instruction a byte.  The
// rotation makes the entries of a vector nearly Gaussian whatever its outliers are, so one scale a vector is enough;
// H is its own inverse but for the factor D, a power of two, so that no normalisation is rounded.
//
//   k_codes  [pages, heads, page, D/2]   byte j: dimension 2j in the low half, 2j+1 in the high half
//   v_codes  [pages, heads, D/2, page]   the same bytes with a page's tokens side by side: the product with the weights
//                                        runs along the tokens, and its matrix operand wants a lane's values along them
//   k_scales, v_scales  bf16 [pages, heads, page]
#pragma once

#include "oq_common.h"

namespace oq {

struct KvCache {
  uint8_t *k_codes, *v_codes;
  uint16_t *k_scales, *v_scales;
  const int8_t *signs;
  int64_t pages;
  int heads, page_shift;  // page = 1 << page_shift tokens
};

constexpr int kKvMaxRequests = 8192;  // of one oq_kv_assign: its two running sums and the lengths sit in LDS
constexpr int kKvMinPage = 16, kKvMaxPage = 1024;

// E values of a vector a lane (8 or 16): element E * part + i in lane `part` of the vector's D / E.  The parts' bits are lane bits
// whose exchanges are vector instructions: 0 and 1 (quad permutes), 3 (a rotation of the row by eight; of 32 lanes only), 4 (of sixteen and more) and 5 (of eight; swaps
// of lane groups); the other lane bits tell the wavefront's vectors apart.
template <int D, int E = 8>
__device__ __forceinline__ int kv_part_of(int lane) {
  if constexpr (D / E == 4) return lane & 3;
  else if constexpr (D / E == 8) return (lane & 3) | (lane >> 5) << 2;
  else if constexpr (D / E == 16) return (lane & 3) | (lane >> 4) << 2;
  else return (lane & 3) | (lane >> 3) << 2;
}
template <int D, int E = 8>
__device__ __forceinline__ int kv_vector_of(int lane) {
  if constexpr (D / E == 4) return lane >> 2;
  else if constexpr (D / E == 8) return (lane >> 2) & 7;
  else if constexpr (D / E == 16) return (lane >> 2) & 3;
  else return (lane >> 2) & 1;
}

// Sums over the lanes up to each: within rows of sixteen, then from row to row.
__device__ __forceinline__ int kv_sums(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

template <int CTRL>
__device__ __forceinline__ uint32_t kv_dpp(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, 0xf, 0xf, true));
}
constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e, kDppXor8 = 0x128;  // quad permutes, and a row rotated by eight
typedef uint32_t kv_u32x2 __attribute__((ext_vector_type(2)));

template <int X>  // 16 or 32
__device__ __forceinline__ kv_u32x2 kv_swap(uint32_t a, uint32_t b) {
  if constexpr (X == 16) return __builtin_amdgcn_permlane16_swap(a, b, false, false);
  else return __builtin_amdgcn_permlane32_swap(a, b, false, false);
}

// The butterflies between lanes X apart, two registers at a time: a swap of lane groups puts the two operands of
// every result into one lane, and a second one the results back.
template <int X>
__device__ __forceinline__ void kv_lane_butterfly(float &a, float &b) {
  const kv_u32x2 in = kv_swap<X>(__float_as_uint(a), __float_as_uint(b));
  const float x = __uint_as_float(in[0]), y = __uint_as_float(in[1]);
  const kv_u32x2 out = kv_swap<X>(__float_as_uint(x + y), __float_as_uint(x - y));
  a = __uint_as_float(out[0]);
  b = __uint_as_float(out[1]);
}

template <int CTRL, int E>
__device__ __forceinline__ void kv_dpp_butterflies(float (&y)[E], bool upper) {
  const float sign = upper ? -1.0f : 1.0f;  // other + y below, other - y above, one rounding
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = fmaf(y[i], sign, __uint_as_float(kv_dpp<CTRL>(__float_as_uint(y[i]))));
}

// One add or subtract for each output and stage, distances 1, 2, 4, ... in this order: the results are those of any other
// schedule of the same butterflies.
// HALVES: of sixteen values a lane has elements 8 * part + i and D / 2 + 8 * part + i, and their distance, the last, between registers.
template <int D, int E, bool HALVES = false>
__device__ __forceinline__ void kv_butterflies(float (&y)[E], int lane) {
  constexpr int LANES = D / E;
  static_assert(!HALVES || E == 16, "two eights");
#pragma unroll
  for (int d = 1; d < (HALVES ? E / 2 : E); d *= 2) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if ((i & d) == 0) {
        const float a = y[i], b = y[i + d];
        y[i] = a + b;
        y[i + d] = a - b;
      }
    }
  }
  kv_dpp_butterflies<kDppXor1>(y, lane & 1);
  kv_dpp_butterflies<kDppXor2>(y, lane & 2);
  if constexpr (LANES == 32) kv_dpp_butterflies<kDppXor8>(y, lane & 8);
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    if constexpr (LANES >= 16) kv_lane_butterfly<16>(y[i], y[i + 1]);
    if constexpr (LANES >= 8) kv_lane_butterfly<32>(y[i], y[i + 1]);
  }
  if constexpr (HALVES) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const float a = y[i], b = y[i + E / 2];
      y[i] = a + b;
      y[i + E / 2] = a - b;
    }
  }
}

// Scale (bf16 bits) and the lane's codes (element i in bits 4 (i % 8) of dword i / 8) of a rotated vector.
//   a = bf16(max|y| * fp32(1/6)), 0 below the smallest normal number; code = E2M1 nearest to y * (1 / a), ties to even
// A vector with an infinity or a NaN in it gets the scale NaN and codes of zero: what attends to it becomes NaN.
template <int D, int E>
__device__ __forceinline__ void kv_encode(const float (&y)[E], uint16_t &scale_bits, uint32_t (&codes)[E / 8]) {
  // The largest magnitude as bits: a NaN is above infinity, infinity above every number.  As signed numbers the bits of positive values are in
  // order, as unsigned ones those of negative values above all others: two maxima, and one sign cleared.
  constexpr int LANES = D / E;
  int positive = 0;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    positive = max(positive, __float_as_int(y[i]));
    any = max(any, __float_as_uint(y[i]));
  }
  uint32_t top = max(static_cast<uint32_t>(positive), any & 0x7fffffffu);
  top = max(top, kv_dpp<kDppXor1>(top));
  top = max(top, kv_dpp<kDppXor2>(top));
  if constexpr (LANES == 32) top = max(top, kv_dpp<kDppXor8>(top));
  if constexpr (LANES >= 16) {
    const kv_u32x2 both = kv_swap<16>(top, top);
    top = max(both[0], both[1]);
  }
  if constexpr (LANES >= 8) {
    const kv_u32x2 both = kv_swap<32>(top, top);
    top = max(both[0], both[1]);
  }
  const bool broken = top >= 0x7f800000u;
  uint16_t a = f32_to_bf16_bits(__uint_as_float(top) * (1.0f / 6.0f));
  if (a < 0x0080u) a = 0;
  scale_bits = broken ? 0x7fc0u : a;
  const float inv = a != 0 && !broken ? 1.0f / bf16_bits_to_f32(a) : 0.0f;
#pragma unroll
  for (int w = 0; w < E / 8; ++w) {
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[8 * w] * inv, y[8 * w + 1] * inv, 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[8 * w + 2] * inv, y[8 * w + 3] * inv, 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[8 * w + 4] * inv, y[8 * w + 5] * inv, 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[8 * w + 6] * inv, y[8 * w + 7] * inv, 1.0f, 3);
    codes[w] = broken ? 0u : q;
  }
}

typedef _Float16 kv_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_f16x8 __attribute__((ext_vector_type(8)));

// Eight codes of a dword as fp16 values, in order.
__device__ __forceinline__ kv_f16x8 kv_decode8(uint32_t w) {
  const kv_f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1);
  const kv_f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3);
  return kv_f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace oq
