// Vectors of sixteen tokens of one head on their way into and out of the 4-bit cache.
#pragma once

#include "kv_cache.h"

namespace oq {

template <int DT>
__device__ __forceinline__ void load8(const void *p, int64_t at, bool wide, float *y) {
  if (wide) {
    if constexpr (DT == OQ_F32) {
      const float4 lo = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at)[0], hi = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at)[1];
      y[0] = lo.x; y[1] = lo.y; y[2] = lo.z; y[3] = lo.w; y[4] = hi.x; y[5] = hi.y; y[6] = hi.z; y[7] = hi.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
      const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = dyn_bits_to_f32((v[i / 2] >> (16 * (i & 1))) & 0xffffu, DT);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = load_as_f32<DT>(p, at + i);
  }
}

template <int DT>
__device__ __forceinline__ void store8(void *p, int64_t at, const float *y) {  // 16-byte aligned
  if constexpr (DT == OQ_F32) {
    reinterpret_cast<float4 *>(static_cast<float *>(p) + at)[0] = make_float4(y[0], y[1], y[2], y[3]);
    reinterpret_cast<float4 *>(static_cast<float *>(p) + at)[1] = make_float4(y[4], y[5], y[6], y[7]);
  } else {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = DT == OQ_F16 ? f32_to_f16_bits(y[2 * i]) : f32_to_bf16_bits(y[2 * i]);
      const uint32_t hi = DT == OQ_F16 ? f32_to_f16_bits(y[2 * i + 1]) : f32_to_bf16_bits(y[2 * i + 1]);
      v[i] = lo | hi << 16;
    }
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + at) = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

template <int E>
__device__ __forceinline__ void times_signs(float (&y)[E], const uint32_t (&words)[E / 4]) {
#pragma unroll
  for (int i = 0; i < E; ++i) y[i] = __uint_as_float(__float_as_uint(y[i]) ^ ((words[i / 4] << (24 - 8 * (i & 3))) & 0x80000000u));
}

// Where the workgroup's tokens are: `slot` -1 for nothing to do, `key` the vector among those of k_codes and the scales, `value` the
// first byte of its column in v_codes.
struct KvPlace {
  int64_t slot, key, value;
};
template <int D>
__device__ __forceinline__ void group_places(KvPlace (&places)[kKvGroup], const KvCache &cache, const int64_t *from, int64_t first, int64_t tokens, int head) {
  if (threadIdx.x < kKvGroup) {
    const int shift = cache.page_shift;
    int64_t slot = -1;
    if (first + threadIdx.x < tokens) slot = from[first + threadIdx.x];
    if (slot < 0 || slot >= cache.pages << shift) slot = -1;
    const int64_t block = max(slot, static_cast<int64_t>(0)) >> shift, in_page = slot & ((1 << shift) - 1);
    places[threadIdx.x] = {slot, ((block * cache.heads + head) << shift) + in_page, (((block * cache.heads + head) * (D / 2)) << shift) + in_page};
  }
}

// Whether four tokens' bytes of a row are one dword.
__device__ __forceinline__ int64_t slot_of(int64_t slot) { return slot; }
__device__ __forceinline__ int64_t slot_of(const KvPlace &place) { return place.slot; }
template <typename Token>
__device__ __forceinline__ bool in_a_row(const Token *tokens, int page_shift) {
  const int64_t s = slot_of(tokens[0]);
  return s >= 0 && slot_of(tokens[1]) == s + 1 && slot_of(tokens[2]) == s + 2 && slot_of(tokens[3]) == s + 3 && (s >> page_shift) == ((s + 3) >> page_shift);
}

// The values' bytes of the workgroup's tokens into their rows, one dword where four of them lie side by side.
template <int D, int THREADS>
__device__ __forceinline__ void store_values(const KvCache &cache, const KvPlace (&places)[kKvGroup], const uint32_t (&bytes)[kKvGroup][D / 8 + 1]) {
  const int shift = cache.page_shift;
  for (int i = threadIdx.x; i < (D / 2) * (kKvGroup / 4); i += THREADS) {
    const int row = i / (kKvGroup / 4), t = i % (kKvGroup / 4) * 4;
    uint32_t four[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) four[k] = reinterpret_cast<const uint8_t *>(bytes[t + k])[row];
    uint8_t *const at_row = cache.v_codes + (static_cast<int64_t>(row) << shift);
    if (in_a_row(places + t, shift)) {
      const uint32_t word = four[0] | four[1] << 8 | four[2] << 16 | four[3] << 24;
      __builtin_memcpy(at_row + places[t].value, &word, 4);  // (a page's tokens may begin anywhere)
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (places[t + k].slot >= 0) at_row[places[t + k].value] = static_cast<uint8_t>(four[k]);
      }
    }
  }
}

}  // namespace oq
