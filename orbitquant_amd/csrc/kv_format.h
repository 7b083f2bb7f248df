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

// Eight values of a vector a lane, the vector's D / 8 lanes side by side: element 8 * lane + i.  Butterfly distances 1, 2
// and 4 are the lane's own registers, the larger ones exchanges with lane ^ (distance / 8).  One add or subtract for each
// output and stage: the results do not depend on the schedule.
template <int D>
__device__ __forceinline__ void kv_butterflies(float (&y)[8], int lane) {
#pragma unroll
  for (int d = 1; d < 8; d *= 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if ((i & d) == 0) {
        const float a = y[i], b = y[i + d];
        y[i] = a + b;
        y[i + d] = a - b;
      }
    }
  }
#pragma unroll
  for (int d = 1; d < D / 8; d *= 2) {
    const bool upper = (lane & d) != 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_xor(y[i], d, 64);
      y[i] = upper ? other - y[i] : y[i] + other;
    }
  }
}

// Scale (bf16 bits) and the lane's eight codes (a dword, element i in bits 4i) of a rotated vector.
//   a = bf16(max|y| * fp32(1/6)), 0 below the smallest normal number; code = E2M1 nearest to y * (1 / a), ties to even
// A vector with an infinity or a NaN in it gets the scale NaN and codes of zero: what attends to it becomes NaN.
template <int D>
__device__ __forceinline__ uint32_t kv_encode(const float (&y)[8], uint16_t &scale_bits) {
  uint32_t top = 0;  // as bits: a NaN is above infinity, infinity above every number
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
#pragma unroll
  for (int d = 1; d < D / 8; d *= 2) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), d, 64)));
  if (top >= 0x7f800000u) {
    scale_bits = 0x7fc0u;
    return 0;
  }
  uint16_t a = f32_to_bf16_bits(__uint_as_float(top) * (1.0f / 6.0f));
  if (a < 0x0080u) a = 0;
  scale_bits = a;
  const float inv = a != 0 ? 1.0f / bf16_bits_to_f32(a) : 0.0f;
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[0] * inv, y[1] * inv, 1.0f, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[2] * inv, y[3] * inv, 1.0f, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[4] * inv, y[5] * inv, 1.0f, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, y[6] * inv, y[7] * inv, 1.0f, 3);
  return q;
}

typedef float kv_f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_f16x8 __attribute__((ext_vector_type(8)));

// Eight codes of a dword as fp16 values, in order.
__device__ __forceinline__ kv_f16x8 kv_decode8(uint32_t w) {
  const kv_f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1);
  const kv_f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3);
  return kv_f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace oq
