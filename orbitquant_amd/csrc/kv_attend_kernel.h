// Attention over the 4-bit key/value cache.
//
//   s[i, t] = scale * q_i . k^_t = (scale / D) * (H (signs * q_i)) . (a_t c_t)          c: the codes' values, a: their scale
//   o_i     = sum_t e^(s[i, t] - m_i) v^_t / l_i = signs * H (sum_t e^(s[i, t] - m_i) b_t c'_t) / (D l_i)
//
// so a query is rotated once, the output is rotated back once, and in between the codes are used as they are: neither keys nor
// values are ever rotated back.  Query i of a request that holds `length` tokens, new of them now, stands at position length -
// new + i and sees the positions up to its own (causal), the last `window` of them if there is a window.
//
// A wavefront holds tiles of sixteen query rows (a row: one token and one of the `group` heads that share a key head) and walks
// the keys in steps of 64.  Both products run transposed, keys and dimensions as the matrix instruction's rows, queries as
// its columns:
//   S^T = K Q^T:  lane (n = lane & 15, g = lane >> 4) of the A operand holds key row n and D / 4 dimensions from g * D / 4 on:
//                 one contiguous piece of the cache.  Row n of tile k is key 16 * (n >> 2) + 4 * k + (n & 3) of the step.
//   the result:   lane (n, g) has query n and keys 16 * g + 4 * k + r, r = 0..3: sixteen keys in a row over the four tiles.
//   O^T = V^T P^T: the B operand wants query n and eight keys a lane, and any order of the keys does as long as V has the
//                 same: lane (n, g) has just the sixteen it needs, so the weights go from one product to the other inside their
//                 registers.  V^T's lane (n, g) reads the bytes of dimensions 32 j + 2 n, 32 j + 2 n + 1 and the tokens
//                 16 g .. 16 g + 15, sixteen bytes, whose halves are regrouped by token pair.
// So pages may be as small as sixteen tokens.
//
// Precision.  The codes are exact in fp16.  A rotated query is scaled by a power of two to use fp16's range and rounded to its
// eleven bits, and so are the weights e^(s - R) b_t; SPLIT 1 (fp16 inputs) keeps a second fp16 part of the query, SPLIT 2 (fp32
// inputs) of both, which leaves 22 bits.  Sums, maxima and exponentials are fp32.
// The reference R of a row is not its maximum: it is raised when a weight could pass 2^15, to where the largest is about 2^10.
// Rows are so rescaled a few times in all, no maximum is exchanged between lanes in between, and the fp16 weights have 24
// binary digits below their largest before they lose any.  R holds the exponent of the largest value scale too (b_t is
// anything), bounded so that l stays finite.
//
// Two kernels.  Few rows (single tokens, at most kKvFewRows of a request): four wavefronts share the keys of sixteen rows, every
// one decodes for itself, and the launch is bound by the cache's bytes.  Many rows (a prompt): the wavefronts have rows of
// their own and the same keys, which they decode once for all of them into LDS; bound by the vector instructions around the
// products.
#pragma once

#include "kv_cache.h"

namespace oq {

typedef float kv_f32x4 __attribute__((ext_vector_type(4)));

constexpr float kKvNothing = -1.0e30f;  // R of a row that has seen no key
constexpr int kKvFewRows = 64;          // rows of a request that the first kernel takes
constexpr int kKvManyRows = 128;        // rows of a workgroup of the second

// Tiles in front of request r when its rows begin at `row`: enough for every request's last, unfilled tile.
__host__ __device__ inline int64_t kv_tile_base(int64_t row, int64_t r) { return row / kKvManyRows + r; }

__device__ __forceinline__ float kv_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// D / 4 values a lane.  Every pair of dimensions that differ in one bit meets once: which bits are registers and which lanes
// does not matter.
template <int D>
__device__ __forceinline__ void kv_rotate_lane(float (&y)[D / 4]) {
#pragma unroll
  for (int d = 1; d < D / 4; d *= 2) {
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      if ((i & d) == 0) {
        const float a = y[i], b = y[i + d];
        y[i] = a + b;
        y[i + d] = a - b;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < D / 4; i += 2) kv_lane_butterfly<16>(y[i], y[i + 1]);
#pragma unroll
  for (int i = 0; i < D / 4; i += 2) kv_lane_butterfly<32>(y[i], y[i + 1]);
}

// Over the four lanes that hold a row (lane & 15 the same).
template <typename Op>
__device__ __forceinline__ float kv_over_groups(float x, Op op) {
  const kv_u32x2 a = kv_swap<16>(__float_as_uint(x), __float_as_uint(x));
  x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const kv_u32x2 b = kv_swap<32>(__float_as_uint(x), __float_as_uint(x));
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float kv_max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float kv_sum_of(float a, float b) { return a + b; }

// A run of rows of one request.
struct KvRows {
  int request, start, fresh, length;  // its first token in q, its queries, its cached tokens
  int first, rows;                    // the run
  int last_key;
  __device__ __forceinline__ int position(int token) const { return length - fresh + token; }
};

__device__ __forceinline__ int kv_start_of(const KvAttendArgs &a, int request) {  // the tokens behind the last request's are a request of their own, without keys
  return request <= a.requests ? min(max(a.starts[request], 0), static_cast<int>(a.tokens)) : static_cast<int>(a.tokens);
}

__device__ __forceinline__ void kv_keys_of(const KvAttendArgs &a, KvRows &r) {
  r.length = r.request < a.requests ? max(a.lengths[r.request], 0) : 0;
  const int64_t reach = static_cast<int64_t>(a.table_width) << a.cache.page_shift;  // what lies behind the table is not there
  r.last_key = static_cast<int>(min(static_cast<int64_t>(r.length), reach)) - 1;
}

// What rows [first, first + rows) of the run see: some row the keys lowest..highest, every row the keys all_low..all_high.
struct KvSpan {
  int lowest, highest, all_low, all_high;
};
__device__ __forceinline__ KvSpan kv_span_of(const KvAttendArgs &a, const KvRows &r, int first, int rows) {
  const int from = r.position(first / a.group), to = r.position((first + rows - 1) / a.group);
  KvSpan s;
  s.highest = a.causal ? min(to, r.last_key) : r.last_key;
  s.all_high = a.causal ? min(from, r.last_key) : r.last_key;
  s.lowest = a.window != 0 ? max(from - a.window + 1, 0) : 0;
  s.all_low = a.window != 0 ? max(to - a.window + 1, 0) : 0;
  return s;
}

__device__ __forceinline__ int kv_page_at(const KvAttendArgs &a, const int32_t *table, int key) {  // -1: not there
  const int column = key >> a.cache.page_shift;
  const int page = column < a.table_width ? table[column] : -1;
  return page < a.cache.pages ? page : -1;
}

// One row a lane (n = lane & 15; the four lanes of a row have a quarter of its dimensions each).
struct KvRow {
  int token, head, low, high;  // token -1: none
};
__device__ __forceinline__ KvRow kv_row_of(const KvAttendArgs &a, const KvRows &r, int kv_head, int row, bool there) {
  const int i = row / a.group;
  KvRow k;
  k.token = there ? r.start + i : -1;
  k.head = kv_head * a.group + row - i * a.group;
  const int position = r.position(i);
  k.high = there ? (a.causal ? min(position, r.last_key) : r.last_key) : -1;
  k.low = a.window != 0 ? max(position - a.window + 1, 0) : 0;
  return k;
}

template <int D>
__device__ __forceinline__ void kv_load_query(const KvAttendArgs &a, const KvRow &row, int g, float (&y)[D / 4]) {
  if (row.token >= 0) {
    const int64_t at = row.token * a.q_token_stride + row.head * a.q_head_stride + g * (D / 4);
    if (a.q_wide && a.q_dtype != OQ_F32) {
#pragma unroll
      for (int i = 0; i < D / 4; i += 8) {
        const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + at + i);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i + e] = dyn_bits_to_f32((w[e / 2] >> (16 * (e & 1))) & 0xffffu, a.q_dtype);
      }
    } else if (a.q_wide) {
#pragma unroll
      for (int i = 0; i < D / 4; i += 4) {
        const float4 v = *reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at + i);
        y[i] = v.x; y[i + 1] = v.y; y[i + 2] = v.z; y[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) y[i] = load_dyn_f32(a.q, a.q_dtype, at + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < D / 4; ++i) y[i] = 0.0f;
  }
}

// Rotates a row's quarter; gives the largest magnitude of the row.
template <int D>
__device__ __forceinline__ float kv_rotate_query(const KvAttendArgs &a, int g, float (&y)[D / 4]) {
#pragma unroll
  for (int i = 0; i < D / 4; ++i) y[i] *= static_cast<float>(a.cache.signs[g * (D / 4) + i]);
  kv_rotate_lane<D>(y);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(y[i]));
  return kv_over_groups(top, kv_max_of);
}

// The power of two 2^-exponent puts `top` into [2^10, 2^11).
__device__ __forceinline__ int kv_query_exponent(float top) {
  return top > 0.0f && top < INFINITY ? min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10, -110), 117) : 0;
}
__device__ __forceinline__ float kv_power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// Two fp16 parts of a pair of numbers.  The first is cut off, by an instruction of its own: the conversion that rounds is merged into
// the product before it here and not there, where it rounds once instead of twice, and a remainder taken from the one does not belong to
// the other (one number in four thousand, an error of 2^-11 of it).
__device__ __forceinline__ void kv_two_parts(float x, float y, _Float16 &x0, _Float16 &y0, _Float16 &x1, _Float16 &y1) {
  const kv_f16x2 cut = __builtin_bit_cast(kv_f16x2, __builtin_amdgcn_cvt_pkrtz(x, y));
  x0 = cut[0]; y0 = cut[1];
  x1 = static_cast<_Float16>(x - static_cast<float>(x0));
  y1 = static_cast<_Float16>(y - static_cast<float>(y0));
}

template <int D, int SPLIT>
__device__ __forceinline__ void kv_query_parts(const float (&y)[D / 4], float down, kv_f16x8 (&q)[D / 32], kv_f16x8 (&rest)[SPLIT > 0 ? D / 32 : 1]) {
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float u = y[8 * c + e] * down, v = y[8 * c + e + 1] * down;
      if constexpr (SPLIT > 0) {
        _Float16 u0, v0, u1, v1;
        kv_two_parts(u, v, u0, v0, u1, v1);
        q[c][e] = u0; q[c][e + 1] = v0;
        rest[c][e] = u1; rest[c][e + 1] = v1;
      } else {
        q[c][e] = static_cast<_Float16>(u);
        q[c][e + 1] = static_cast<_Float16>(v);
      }
    }
  }
}

// Scores become weights, for one tile of sixteen rows and the sixteen keys of a lane.
struct KvState {
  float ref, sum;
  float limit;  // of a score above R: kKvNothing until the row has seen a key, so that the first one sets R
  __device__ __forceinline__ void begin() { ref = 0.0f; sum = 0.0f; limit = kKvNothing; }
  __device__ __forceinline__ float reference() const { return limit < 0.0f ? kKvNothing : ref; }
};

// x: scores minus R.  Raises R where a weight could pass 2^15, O along with it.
template <int D>
__device__ __forceinline__ void kv_keep_in_range(float (&x)[16], float top_exponent, KvState &st, kv_f32x4 (&o)[D / 16]) {
  float best = fmaxf(x[0], x[1]);
#pragma unroll
  for (int i = 2; i < 16; i += 2) best = fmaxf(best, fmaxf(x[i], x[i + 1]));
  best += top_exponent;
  if (__builtin_amdgcn_ballot_w64(best > st.limit) != 0) {
    best = kv_over_groups(best, kv_max_of);
    const bool raise = best > st.limit;
    const float up = raise ? best - 10.0f : 0.0f, by = kv_exp2(fminf(-up, 0.0f));  // (down only where nothing is summed up yet)
    st.ref += up;
    st.sum *= by;
    st.limit = raise ? 15.0f : st.limit;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[j] *= by;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] -= up;
  }
}

// Weights as the B operand: entries of tiles 2 * half and 2 * half + 1 side by side.
template <int SPLIT>
__device__ __forceinline__ void kv_weights(const float (&x)[16], const float (&vs)[16], float &sum, kv_f16x8 (&p)[2], kv_f16x8 (&rest)[SPLIT > 1 ? 2 : 1]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 8 * half + r;
      const float e0 = kv_exp2(x[i]), e1 = kv_exp2(x[i + 4]);
      sum += e0;
      sum += e1;
      const float w0 = e0 * vs[i], w1 = e1 * vs[i + 4];
      if constexpr (SPLIT > 1) {
        _Float16 a0, b0, a1, b1;
        kv_two_parts(w0, w1, a0, b0, a1, b1);
        p[half][2 * r] = a0; p[half][2 * r + 1] = b0;
        rest[half][2 * r] = a1; rest[half][2 * r + 1] = b1;
      } else {
        p[half][2 * r] = static_cast<_Float16>(w0);
        p[half][2 * r + 1] = static_cast<_Float16>(w1);
      }
    }
  }
}

// Keys that a row does not see, or that are not there.  A weight of 0 does not undo a scale that is NaN: where a value's is, the
// rows that see it get theirs through the score; what lies behind the last key may be anything.
__device__ __forceinline__ float kv_masked_score(float x, float vs, int key, bool there, const KvRow &row) {
  const bool seen = there && key <= row.high && key >= row.low;
  return seen ? (vs != vs ? NAN : x) : -INFINITY;
}

__device__ __forceinline__ float kv_exponent_above(const float (&vs)[16]) {  // every scale is below 2^this
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(vs[i]));
  return static_cast<float>(min(max(static_cast<int>(top >> 23) - 126, -80), 80));
}

// Sixteen token bytes of two dimensions -> the A operands of the even and the odd one, tiles 2 * half and 2 * half + 1 side by side.
__device__ __forceinline__ void kv_decode_values(uint32_t x, uint32_t y, kv_f16x8 &even, kv_f16x8 &odd) {
  even = kv_decode8((x & 0x0f0f0f0fu) | ((y & 0x0f0f0f0fu) << 4));
  odd = kv_decode8(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u));
}

// A row's result: rotated back, and stored as the output, or as a part of it.
template <int D>
__device__ __forceinline__ void kv_finish(const KvAttendArgs &a, const KvRow &row, int g, int part, const KvState &st, const kv_f32x4 (&o)[D / 16]) {
  const float l = kv_over_groups(st.sum, kv_sum_of);
  const bool parts = a.parts > 1;
  const float by = parts ? 1.0f / D : l != 0.0f ? (1.0f / D) / l : 0.0f;  // (no key: zeros)
  // dimension 32 j + 8 g + 2 r + parity is in o[2 j + parity][r]
  float y[D / 4];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      y[8 * j + 2 * r] = o[2 * j][r] * by;
      y[8 * j + 2 * r + 1] = o[2 * j + 1][r] * by;
    }
  }
  kv_rotate_lane<D>(y);
  if (row.token < 0) return;
  const int64_t index = static_cast<int64_t>(row.token) * a.heads + row.head;
  const int64_t in_parts = static_cast<int64_t>(part) * a.tokens * a.heads + index;
#pragma unroll
  for (int j = 0; j < D / 32; ++j) {
    const uint2 sign = *reinterpret_cast<const uint2 *>(a.cache.signs + 32 * j + 8 * g);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(__float_as_uint(y[8 * j + e]) ^ (((e < 4 ? sign.x : sign.y) << (24 - 8 * (e & 3))) & 0x80000000u));
    const int at = 32 * j + 8 * g;
    if (parts || a.q_dtype == OQ_F32) {
      float *to = parts ? a.part_out + in_parts * D + at : static_cast<float *>(a.out) + index * D + at;
      reinterpret_cast<float4 *>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4 *>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        w[e] = a.q_dtype == OQ_F16 ? f32_to_f16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_f16_bits(v[2 * e + 1])) << 16
                                   : f32_to_bf16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16;
      }
      *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + index * D + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (g != 0) return;
  if (parts) a.part_stats[in_parts] = make_float2(st.reference(), l);
  else if (a.lse != nullptr) a.lse[index] = l != 0.0f ? (st.ref + __builtin_amdgcn_logf(l)) * 0.693147180559945f : -INFINITY;
}

// A step's keys, scales and values as they come from the cache, for a wavefront that decodes all of them.
template <int D>
struct KvRaw {
  uint32_t k[4][D / 32];
  uint4 v[D / 32], k_scale[2], v_scale[2];
  bool here;  // the page of the lane's sixteen keys is there
};
struct KvPages {  // of key rows (n >> 2) and of values and scales (g)
  int k, v;
};
__device__ __forceinline__ KvPages kv_pages_of(const KvAttendArgs &a, const int32_t *table, int n, int g, int step) {
  return {kv_page_at(a, table, step * 64 + 16 * (n >> 2)), kv_page_at(a, table, step * 64 + 16 * g)};
}
template <int D>
__device__ __forceinline__ void kv_request_keys(const KvAttendArgs &a, int kv_head, int n, int g, int s, const KvPages &page, KvRaw<D> &to) {
  constexpr int W = D / 32;
  const int shift = a.cache.page_shift, in_page = (1 << shift) - 1;
  const int64_t k_block = static_cast<int64_t>(max(page.k, 0)) * a.cache.heads + kv_head, v_block = static_cast<int64_t>(max(page.v, 0)) * a.cache.heads + kv_head;
  const uint32_t *from = reinterpret_cast<const uint32_t *>(a.cache.k_codes) + ((k_block << shift) + ((s * 64 + 16 * (n >> 2)) & in_page) + (n & 3)) * (D / 8) + g * W;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (W == 2) {
      const uint2 v = *reinterpret_cast<const uint2 *>(from + 4 * t * (D / 8));
      to.k[t][0] = v.x; to.k[t][1] = v.y;
    } else {
#pragma unroll
      for (int w = 0; w < W; w += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(from + 4 * t * (D / 8) + w);
        to.k[t][w] = v.x; to.k[t][w + 1] = v.y; to.k[t][w + 2] = v.z; to.k[t][w + 3] = v.w;
      }
    }
  }
  const int64_t scales = (v_block << shift) + ((s * 64 + 16 * g) & in_page);
  const uint4 *k_from = reinterpret_cast<const uint4 *>(a.cache.k_scales + scales), *v_from = reinterpret_cast<const uint4 *>(a.cache.v_scales + scales);
  to.k_scale[0] = k_from[0]; to.k_scale[1] = k_from[1];
  to.v_scale[0] = v_from[0]; to.v_scale[1] = v_from[1];
  to.here = page.v >= 0;
}
template <int D>
__device__ __forceinline__ void kv_request_values(const KvAttendArgs &a, int kv_head, int n, int g, int s, const KvPages &page, KvRaw<D> &to) {
  const int shift = a.cache.page_shift;
  const int64_t block = static_cast<int64_t>(max(page.v, 0)) * a.cache.heads + kv_head;
  const uint8_t *from = a.cache.v_codes + ((block * (D / 2) + n) << shift) + ((s * 64 + 16 * g) & ((1 << shift) - 1));
#pragma unroll
  for (int j = 0; j < D / 32; ++j) to.v[j] = *reinterpret_cast<const uint4 *>(from + (static_cast<int64_t>(16 * j) << shift));
}
template <int D>
__device__ __forceinline__ void kv_request(const KvAttendArgs &a, int kv_head, int n, int g, int s, const KvPages &page, KvRaw<D> &to) {
  kv_request_keys<D>(a, kv_head, n, g, s, page, to);
  kv_request_values<D>(a, kv_head, n, g, s, page, to);
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// Sixteen rows a workgroup; its four wavefronts take every fourth step of the part's keys and are joined through LDS.  A step's
// keys, scales and values (8.4 KB at D = 128) are requested DEPTH of the wavefront's steps ahead, into the registers of the ones just used.
template <int D, int SPLIT>
__global__ __launch_bounds__(256, 2) void kv_attend_few_kernel(KvAttendArgs a) {
  constexpr int W = D / 32;  // dwords of codes that a lane has of a key, and matrix instructions along the dimensions
  constexpr int DEPTH = D == 256 ? 1 : 2;  // (of heads of 256 two steps do not fit the registers)
  __shared__ float join[2][D / 4 + 2][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kv_head = blockIdx.x % a.cache.heads, part = blockIdx.y;
  const int tile = blockIdx.x / a.cache.heads;

  KvRows r;
  r.request = tile / a.few_tiles;
  r.first = (tile - r.request * a.few_tiles) * 16;
  r.start = r.request;
  r.fresh = 1;
  if (a.starts != nullptr) {
    r.start = kv_start_of(a, r.request);
    r.fresh = max(kv_start_of(a, r.request + 1) - r.start, 0);
    if (static_cast<int64_t>(r.fresh) * a.group > kKvFewRows) return;
  }
  r.rows = min(r.fresh * a.group - r.first, 16);
  if (r.rows <= 0) return;
  kv_keys_of(a, r);
  const KvSpan span = kv_span_of(a, r, r.first, r.rows);
  int step = (span.lowest >> 6) + part * a.part_steps;
  int end = span.highest >= span.lowest ? (span.highest >> 6) + 1 : 0;
  if (part + 1 < a.parts) end = min(end, step + a.part_steps);
  step += wave;

  const int32_t *table = a.table + r.request * a.table_stride;
  KvRaw<D> raw[DEPTH];
  KvPages pages[DEPTH];  // of the steps that are requested next
  // the first steps are on their way while the queries are rotated
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) {
    if (step + 4 * i < end) kv_request<D>(a, kv_head, n, g, step + 4 * i, kv_pages_of(a, table, n, g, step + 4 * i), raw[i]);
  }
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) pages[i] = kv_pages_of(a, table, n, g, step + 4 * (DEPTH + i));

  const KvRow row = kv_row_of(a, r, kv_head, r.first + n, n < r.rows);
  kv_f16x8 q[W], q_rest[SPLIT > 0 ? W : 1];
  float factor;
  {
    float y[D / 4];
    kv_load_query<D>(a, row, g, y);
    const int exponent = kv_query_exponent(kv_rotate_query<D>(a, g, y));
    factor = a.scale * (1.44269504088896f / D) * kv_power_of_two(exponent);
    kv_query_parts<D, SPLIT>(y, kv_power_of_two(-exponent), q, q_rest);
  }

  KvState st;
  st.begin();
  kv_f32x4 o[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) o[j] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const auto take_step = [&](int s, KvRaw<D> &now, KvPages &next) {
    const bool more = s + 4 * DEPTH < end;
    float x[16], vs[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      kv_f32x4 score = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const kv_f16x8 codes = kv_decode8(now.k[k][c]);
        if constexpr (SPLIT > 0) score = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q_rest[c], score, 0, 0, 0);
        score = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q[c], score, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * k + i] = score[i];
    }
    {
      const uint32_t kw[8] = {now.k_scale[0].x, now.k_scale[0].y, now.k_scale[0].z, now.k_scale[0].w, now.k_scale[1].x, now.k_scale[1].y, now.k_scale[1].z, now.k_scale[1].w};
      const uint32_t vw[8] = {now.v_scale[0].x, now.v_scale[0].y, now.v_scale[0].z, now.v_scale[0].w, now.v_scale[1].x, now.v_scale[1].y, now.v_scale[1].z, now.v_scale[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[2 * i] = fmaf(x[2 * i], __uint_as_float(kw[i] << 16) * factor, -st.ref);
        x[2 * i + 1] = fmaf(x[2 * i + 1], __uint_as_float(kw[i] & 0xffff0000u) * factor, -st.ref);
        vs[2 * i] = __uint_as_float(vw[i] << 16);
        vs[2 * i + 1] = __uint_as_float(vw[i] & 0xffff0000u);
      }
    }
    const bool here = now.here;
    if (more) kv_request_keys<D>(a, kv_head, n, g, s + 4 * DEPTH, next, now);
    const int first = s * 64;
    if (first + 63 > span.all_high || first < span.all_low || __builtin_amdgcn_ballot_w64(!here) != 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = first + 16 * g + i;
        const bool there = here && key <= r.last_key;
        x[i] = kv_masked_score(x[i], vs[i], key, there, row);
        vs[i] = there && vs[i] == vs[i] ? vs[i] : 0.0f;
      }
    }
    kv_keep_in_range<D>(x, kv_exponent_above(vs), st, o);
    kv_f16x8 p[2], p_rest[SPLIT > 1 ? 2 : 1];
    kv_weights<SPLIT>(x, vs, st.sum, p, p_rest);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t w[4] = {now.v[j].x, now.v[j].y, now.v[j].z, now.v[j].w};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        kv_f16x8 even, odd;
        kv_decode_values(w[2 * half], w[2 * half + 1], even, odd);
        if constexpr (SPLIT > 1) {
          o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p_rest[half], o[2 * j], 0, 0, 0);
          o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p_rest[half], o[2 * j + 1], 0, 0, 0);
        }
        o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p[half], o[2 * j], 0, 0, 0);
        o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p[half], o[2 * j + 1], 0, 0, 0);
      }
    }
    if (more) kv_request_values<D>(a, kv_head, n, g, s + 4 * DEPTH, next, now);
    next = kv_pages_of(a, table, n, g, s + 8 * DEPTH);
  };
  for (; step < end; step += 4 * DEPTH) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (step + 4 * i < end) take_step(step + 4 * i, raw[i], pages[i]);
    }
  }
  st.ref = st.reference();

  // the four wavefronts: neighbours first, then the two pairs, in this order
  const auto give = [&](int place) {
    join[place][0][lane] = st.ref;
    join[place][1][lane] = st.sum;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) join[place][2 + 4 * j + i][lane] = o[j][i];
    }
  };
  const auto take = [&](int place) {
    const float theirs = join[place][0][lane], both = fmaxf(st.ref, theirs);
    const float mine = kv_exp2(st.ref - both), other = kv_exp2(theirs - both);
    st.ref = both;
    st.sum = fmaf(st.sum, mine, join[place][1][lane] * other);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = fmaf(o[j][i], mine, join[place][2 + 4 * j + i][lane] * other);
    }
  };
  if (wave & 1) give(wave >> 1);
  __syncthreads();
  if ((wave & 1) == 0) take(wave >> 1);
  __syncthreads();
  if (wave == 2) give(1);
  __syncthreads();
  if (wave != 0) return;
  take(1);
  st.limit = 1.0f;  // (what R says is all there is to know now)
  kv_finish<D>(a, row, g, part, st, o);
}

// ---- many rows -----------------------------------------------------------------------------------------------------
// 128 rows a workgroup, 16 * RT a wavefront, all on the same keys.  Decoding a step costs as many vector instructions as the softmax
// of 32 rows: each wavefront decodes a part of it into LDS, in the order of the operands (conflict-free on both sides), for the next step while
// this one's products run; one barrier a step.
template <int D>
constexpr int kv_many_waves() { return D == 256 ? 8 : 4; }

template <int D, int SPLIT>
__global__ __launch_bounds__(64 * kv_many_waves<D>(), 2) void kv_attend_many_kernel(KvAttendArgs a) {
  constexpr int WAVES = kv_many_waves<D>(), RT = kKvManyRows / 16 / WAVES;
  constexpr int C = D / 32;
  constexpr int KD = D * 2 / (16 * WAVES), VD = KD;  // dwords of a step's keys and values that a lane decodes
  struct Step {
    kv_f16x8 k[4][C][64];         // [tile][dimensions][lane]
    kv_f16x8 v[D / 32][2][2][64]; // [dimensions][half of the keys][even, odd][lane]
    float ks[64], vs[64];         // times the scale of the scores; as it is
  };
  extern __shared__ char lds[];
  Step *steps = reinterpret_cast<Step *>(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kv_head = blockIdx.x % a.cache.heads, part = blockIdx.y;
  const int tile = a.many_tiles - 1 - static_cast<int>(blockIdx.x / a.cache.heads);  // a prompt's last rows see the most keys: they begin first

  KvRows r;
  {
    int low = 0, high = a.requests + 1;
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (kv_tile_base(static_cast<int64_t>(kv_start_of(a, mid)) * a.group, mid) <= tile) low = mid; else high = mid;
    }
    r.request = low;
    r.start = kv_start_of(a, low);
    r.fresh = max(kv_start_of(a, low + 1) - r.start, 0);
    const int64_t first = (tile - kv_tile_base(static_cast<int64_t>(r.start) * a.group, low)) * kKvManyRows, all = static_cast<int64_t>(r.fresh) * a.group;
    if (first >= all || all <= a.few_rows) return;
    r.first = static_cast<int>(first);
    r.rows = static_cast<int>(min(all - first, static_cast<int64_t>(kKvManyRows)));
  }
  kv_keys_of(a, r);
  const KvSpan span = kv_span_of(a, r, r.first, r.rows);
  int step = (span.lowest >> 6) + part * a.part_steps;
  int end = span.highest >= span.lowest ? (span.highest >> 6) + 1 : 0;
  if (part + 1 < a.parts) end = min(end, step + a.part_steps);

  // what this wavefront decodes: keys of one tile, all or half of their dimensions; values of one j, both halves of the keys or one
  const int shift = a.cache.page_shift;
  const int32_t *table = a.table + r.request * a.table_stride;
  const int k_tile = WAVES == 8 ? wave >> 1 : wave, k_from = WAVES == 8 ? (wave & 1) * KD : 0;
  const int v_j = VD == 2 ? wave >> 1 : wave, v_from = VD == 2 ? wave & 1 : 0;
  uint32_t k_raw[KD], v_raw[VD], scale_raw = 0;
  const auto load = [&](int s, int page_k, int page_v) {
    const int64_t k_block = static_cast<int64_t>(max(page_k, 0)) * a.cache.heads + kv_head, v_block = static_cast<int64_t>(max(page_v, 0)) * a.cache.heads + kv_head;
    const int in_page = (1 << shift) - 1;
    const uint32_t *k_at = reinterpret_cast<const uint32_t *>(a.cache.k_codes) +
                           ((k_block << shift) + ((s * 64 + 16 * (n >> 2)) & in_page) + 4 * k_tile + (n & 3)) * (D / 8) + g * (D / 32) + k_from;
    const uint8_t *v_at = a.cache.v_codes + ((v_block * (D / 2) + 16 * v_j + n) << shift) + ((s * 64 + 16 * g) & in_page) + 8 * v_from;
    if constexpr (KD == 2) {
      const uint2 k = *reinterpret_cast<const uint2 *>(k_at), v = *reinterpret_cast<const uint2 *>(v_at);
      k_raw[0] = k.x; k_raw[1] = k.y; v_raw[0] = v.x; v_raw[1] = v.y;
    } else {
      const uint4 k = *reinterpret_cast<const uint4 *>(k_at), v = *reinterpret_cast<const uint4 *>(v_at);
      k_raw[0] = k.x; k_raw[1] = k.y; k_raw[2] = k.z; k_raw[3] = k.w; v_raw[0] = v.x; v_raw[1] = v.y; v_raw[2] = v.z; v_raw[3] = v.w;
    }
    if (wave < 2) scale_raw = (wave == 0 ? a.cache.k_scales : a.cache.v_scales)[(v_block << shift) + ((s * 64 + 16 * g) & in_page) + n];
  };
  int page_v = -1, next_k = -1, next_v = -1, later_k = -1, later_v = -1;  // of the step that is computed (v: whether its keys are there), requested, and after it
  if (step < end) {
    const int page_k = kv_page_at(a, table, step * 64 + 16 * (n >> 2));
    page_v = kv_page_at(a, table, step * 64 + 16 * g);
    next_k = kv_page_at(a, table, (step + 1) * 64 + 16 * (n >> 2));
    next_v = kv_page_at(a, table, (step + 1) * 64 + 16 * g);
    load(step, page_k, page_v);
  }

  KvRow row[RT];
  kv_f16x8 q[RT][C], q_rest[RT][SPLIT > 0 ? C : 1];
  float factor;
  {
    float y[RT][D / 4], top = 0.0f;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int at = (wave * RT + t) * 16 + n;
      row[t] = kv_row_of(a, r, kv_head, r.first + at, at < r.rows);
      kv_load_query<D>(a, row[t], g, y[t]);
      const float own_top = kv_rotate_query<D>(a, g, y[t]);
      top = own_top < INFINITY ? fmaxf(top, own_top) : top;  // (a broken row is its own affair)
    }
    // one power of two for the workgroup's rows: its factor goes into the keys' scales
#pragma unroll
    for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
    float *tops = steps[1].ks;  // (the first step decodes into steps[0])
    if (lane == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, tops[w]);
    const int exponent = kv_query_exponent(top);
    factor = a.scale * (1.44269504088896f / D) * kv_power_of_two(exponent);
#pragma unroll
    for (int t = 0; t < RT; ++t) kv_query_parts<D, SPLIT>(y[t], kv_power_of_two(-exponent), q[t], q_rest[t]);
  }
  const int wave_first = wave * RT * 16, wave_rows = min(r.rows - wave_first, RT * 16);  // rows of this wavefront, if any
  const KvSpan own = kv_span_of(a, r, r.first + min(wave_first, r.rows - 1), max(wave_rows, 1));

  const auto decode = [&](Step &to) {
#pragma unroll
    for (int i = 0; i < KD; ++i) to.k[k_tile][k_from + i][lane] = kv_decode8(k_raw[i]);
#pragma unroll
    for (int i = 0; i < VD / 2; ++i) {
      kv_f16x8 even, odd;
      kv_decode_values(v_raw[2 * i], v_raw[2 * i + 1], even, odd);
      to.v[v_j][v_from + i][0][lane] = even;
      to.v[v_j][v_from + i][1][lane] = odd;
    }
    const float scale = __uint_as_float(scale_raw << 16);  // of key 16 * g + n: lane
    if (wave == 0) to.ks[lane] = scale * factor;
    else if (wave == 1) to.vs[lane] = scale;
  };

  KvState st[RT];
  kv_f32x4 o[RT][D / 16];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    st[t].begin();
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[t][j] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  if (step < end) {
    decode(steps[0]);
    if (step + 1 < end) load(step + 1, next_k, next_v);
    later_k = kv_page_at(a, table, (step + 2) * 64 + 16 * (n >> 2));
    later_v = kv_page_at(a, table, (step + 2) * 64 + 16 * g);
  }
  for (int now = 0; step < end; ++step, now ^= 1) {
    __syncthreads();  // this step is decoded, and nobody reads the one before it any more
    const Step &from = steps[now];
    const bool here = page_v >= 0;
    if (step + 1 < end) {
      decode(steps[now ^ 1]);
      if (step + 2 < end) load(step + 2, later_k, later_v);
    }
    page_v = next_v; next_k = later_k; next_v = later_v;
    later_k = kv_page_at(a, table, (step + 3) * 64 + 16 * (n >> 2));
    later_v = kv_page_at(a, table, (step + 3) * 64 + 16 * g);
    const int first = step * 64;
    if (wave_rows <= 0 || first > own.highest || first + 63 < own.lowest) continue;

    float x[RT][16], vs[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      kv_f32x4 s[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const kv_f16x8 codes = from.k[k][c][lane];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if constexpr (SPLIT > 0) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q_rest[t][c], s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q[t][c], s[t], 0, 0, 0);
        }
      }
      const kv_f32x4 ks = *reinterpret_cast<const kv_f32x4 *>(&from.ks[16 * g + 4 * k]), v = *reinterpret_cast<const kv_f32x4 *>(&from.vs[16 * g + 4 * k]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vs[4 * k + i] = v[i];
#pragma unroll
        for (int t = 0; t < RT; ++t) x[t][4 * k + i] = fmaf(s[t][i], ks[i], -st[t].ref);
      }
    }
    if (first + 63 > own.all_high || first < own.all_low || __builtin_amdgcn_ballot_w64(!here) != 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = first + 16 * g + i;
        const bool there = here && key <= r.last_key;
#pragma unroll
        for (int t = 0; t < RT; ++t) x[t][i] = kv_masked_score(x[t][i], vs[i], key, there, row[t]);
        vs[i] = there && vs[i] == vs[i] ? vs[i] : 0.0f;
      }
    }
    const float top_exponent = kv_exponent_above(vs);
    kv_f16x8 p[RT][2], p_rest[RT][SPLIT > 1 ? 2 : 1];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      kv_keep_in_range<D>(x[t], top_exponent, st[t], o[t]);
      kv_weights<SPLIT>(x[t], vs, st[t].sum, p[t], p_rest[t]);
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const kv_f16x8 even = from.v[j][half][0][lane], odd = from.v[j][half][1][lane];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          if constexpr (SPLIT > 1) {
            o[t][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p_rest[t][half], o[t][2 * j], 0, 0, 0);
            o[t][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p_rest[t][half], o[t][2 * j + 1], 0, 0, 0);
          }
          o[t][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p[t][half], o[t][2 * j], 0, 0, 0);
          o[t][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p[t][half], o[t][2 * j + 1], 0, 0, 0);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) kv_finish<D>(a, row[t], g, part, st[t], o[t]);
}

template <int D>
constexpr size_t kv_many_lds() { return 2 * (4 * (D / 32) * 64 * 16 + (D / 32) * 4 * 64 * 16 + 512); }

template <int D, int SPLIT>
bool kv_attend_launch(const KvAttendArgs &a, hipStream_t stream) {
  const unsigned heads = static_cast<unsigned>(a.cache.heads), parts = static_cast<unsigned>(a.parts);
  if (a.many_tiles > 0) {
    if (!reserve_dynamic_lds(reinterpret_cast<const void *>(kv_attend_many_kernel<D, SPLIT>), kv_many_lds<D>())) return false;
    launch_kernel(kv_attend_many_kernel<D, SPLIT>, dim3(heads * a.many_tiles, parts), dim3(64 * kv_many_waves<D>()), kv_many_lds<D>(), stream, a);
  }
  if (a.few_requests > 0) launch_kernel(kv_attend_few_kernel<D, SPLIT>, dim3(heads * a.few_requests * a.few_tiles, parts), dim3(256), 0, stream, a);
  return true;
}

}  // namespace oq
