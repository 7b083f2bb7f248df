// Attention over the 4-bit key/value cache.
//
//   s[i, t] = scale * q_i . k^_t = (scale / D) * (H (signs * q_i)) . (a_t c_t)          c: the codes' values, a: their scale
//   o_i     = sum_t e^(s[i, t] - m_i) v^_t / l_i = signs * H (sum_t e^(s[i, t] - m_i) b_t c'_t) / (D l_i)
//
// so a query is rotated once, the output is rotated back once, and in between the codes are used as they are: neither keys nor values are ever
// rotated back.  Query i of a request that holds `length` tokens, new of them now, stands at position length - new + i and sees the
// positions up to its own (causal), the last `window` of them if there is a window.
//
// A wavefront holds RT tiles of sixteen query rows (a row: one token and one of the `group` heads that share a key head) and
// walks the keys in steps of 64.  Both products run transposed, keys and dimensions as the matrix instruction's rows,
// queries as its columns:
//   S^T = K Q^T:  lane (n = lane & 15, g = lane >> 4) of the A operand holds key row n and D / 4 dimensions from g * D / 4 on:
//                 one contiguous piece of the cache.  Row n of tile a is key 16 * (n >> 2) + 4 * a + (n & 3) of the step.
//   the result:   lane (n, g) has query n and keys 16 * g + 4 * a + r, r = 0..3: sixteen keys in a row over the four tiles.
//   O^T = V^T P^T: the B operand wants query n and eight keys a lane, and any order of the keys does as long as V has the
//                 same: lane (n, g) has just the sixteen it needs, so the weights go from one product to the other inside their
//                 registers.  V^T's lane (n, g) reads the bytes of dimensions 32 j + 2 n, 32 j + 2 n + 1 and the tokens
//                 16 g .. 16 g + 15, sixteen bytes, whose halves are regrouped by token pair.
// So there is no LDS and no barrier on the way; pages may be as small as sixteen tokens.
//
// Precision.  The codes are exact in fp16.  A rotated query is scaled by a power of two to use fp16's range and rounded to its eleven bits, and so are
// the weights e^(s - R) b_t; SPLIT 1 (fp16 inputs) keeps a second fp16 part of the query, SPLIT 2 (fp32 inputs) of both, which
// leaves 22 bits.  Sums, maxima and exponentials are fp32.
// The reference R of a row is not its maximum: it is raised when a weight could pass 2^15, to where the largest is about 2^10.  Rows are so rescaled a
// few times in all, no maximum is exchanged between lanes in between, and the fp16 weights have 24 binary digits below their
// largest before they lose any.  R holds the exponent of the largest value scale too (b_t is anything), bounded so that l stays finite.
#pragma once

#include "kv_cache.h"

namespace oq {

typedef float kv_f32x4 __attribute__((ext_vector_type(4)));

constexpr float kKvNothing = -1.0e30f;  // R of a row that has seen no key: e^(-inf - R) is 0, any key raises it

// Row tiles of a workgroup: four wavefronts with RT * 16 rows each.  A tile with few rows has its wavefronts share the keys instead.
template <int RT>
constexpr int kv_tile_rows() { return 64 * RT; }

// Tiles in front of request r when its rows begin at `row`: enough for every request's last, unfilled tile.
__host__ __device__ inline int64_t kv_tile_base(int64_t row, int64_t r, int tile_rows) { return row / tile_rows + r; }

template <int D>
__device__ __forceinline__ void kv_rotate_lane(float (&y)[D / 4], int lane) {  // D / 4 dimensions a lane from (lane >> 4) * D / 4 on
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
  for (int x = 16; x < 64; x *= 2) {
    const bool upper = (lane & x) != 0;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      const float other = __shfl_xor(y[i], x, 64);
      y[i] = upper ? other - y[i] : y[i] + other;
    }
  }
}

__device__ __forceinline__ float kv_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <int D, int RT, int SPLIT>
__global__ __launch_bounds__(256, 2) void kv_attend_kernel(KvAttendArgs a) {
  constexpr int C = D / 32;                 // matrix instructions along the dimensions
  constexpr int W = D / 32;                 // dwords of codes a lane has of a key
  constexpr int kOutRegs = RT * (D / 4);
  __shared__ float join[2][kOutRegs + 2 * RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kv_head = blockIdx.x % a.cache.heads, part = blockIdx.y;  // neighbours in the grid: heads of the same rows
  const int tile = a.tiles - 1 - static_cast<int>(blockIdx.x / a.cache.heads);  // a prompt's last rows see the most keys: they begin first

  // which rows
  int request, first_row, rows, start, length, fresh;
  if (a.starts == nullptr) {
    const int each = (a.group + kv_tile_rows<RT>() - 1) / kv_tile_rows<RT>();
    request = tile / each;
    first_row = (tile - request * each) * kv_tile_rows<RT>();
    start = request;
    fresh = 1;
  } else {
    const int tokens = static_cast<int>(a.tokens);
    const auto start_of = [&](int r) { return min(max(a.starts[r], 0), tokens); };
    int low = 0, high = a.requests + 1;     // the rows behind the last request's are a request of their own, without keys
    while (high - low > 1) {
      const int mid = (low + high) >> 1;
      if (kv_tile_base(static_cast<int64_t>(start_of(mid)) * a.group, mid, kv_tile_rows<RT>()) <= tile) low = mid; else high = mid;
    }
    request = low;
    start = start_of(request);
    fresh = max((request < a.requests ? start_of(request + 1) : tokens) - start, 0);
    const int64_t ahead = tile - kv_tile_base(static_cast<int64_t>(start) * a.group, request, kv_tile_rows<RT>());
    first_row = static_cast<int>(min(ahead * kv_tile_rows<RT>(), static_cast<int64_t>(0x7fffffff)));
  }
  if (first_row >= static_cast<int64_t>(fresh) * a.group) return;
  rows = min(static_cast<int>(min(static_cast<int64_t>(fresh) * a.group - first_row, static_cast<int64_t>(kv_tile_rows<RT>()))), kv_tile_rows<RT>());
  length = request < a.requests ? max(a.lengths[request], 0) : 0;
  const int64_t reach = static_cast<int64_t>(a.table_width) << a.cache.page_shift;  // what lies behind the table is not there
  const int last_key = static_cast<int>(min(static_cast<int64_t>(length), reach)) - 1;

  // rows and keys of this wavefront
  const int sets = (rows + 16 * RT - 1) / (16 * RT);        // of RT tiles
  const int sharing = sets == 1 ? 4 : sets == 2 ? 2 : 1;    // wavefronts on the same rows
  const int set = wave / sharing, rank = wave - set * sharing;
  int token[RT], head[RT], low[RT], high[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int in_tile = (set * RT + t) * 16 + n, row = first_row + in_tile;
    const int i = row / a.group;
    token[t] = in_tile < rows ? start + i : -1;
    head[t] = kv_head * a.group + row - i * a.group;
    const int position = length - fresh + i;
    high[t] = in_tile < rows ? (a.causal ? min(position, last_key) : last_key) : -1;
    low[t] = a.window != 0 ? max(position - a.window + 1, 0) : 0;
  }
  const int first_i = first_row / a.group, last_i = (first_row + rows - 1) / a.group;
  const int highest = a.causal ? min(length - fresh + last_i, last_key) : last_key;
  const int lowest = a.window != 0 ? max(length - fresh + first_i - a.window + 1, 0) : 0;
  // every row of the tile sees the keys in between
  const int all_high = a.causal ? min(length - fresh + first_i, last_key) : last_key;
  const int all_low = a.window != 0 ? max(length - fresh + last_i - a.window + 1, 0) : 0;
  int step = (lowest >> 6) + part * a.part_steps;
  int end = highest >= lowest ? (highest >> 6) + 1 : 0;
  if (part + 1 < a.parts) end = min(end, step + a.part_steps);

  // queries, rotated, as the B operand
  kv_f16x8 q[RT][C], q_rest[SPLIT > 0 ? RT : 1][C];
  float factor[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float y[D / 4];
    if (token[t] >= 0) {
      const int64_t at = token[t] * a.q_token_stride + head[t] * a.q_head_stride + g * (D / 4);
      if (a.q_wide && a.q_dtype != OQ_F32) {
#pragma unroll
        for (int i = 0; i < D / 4; i += 8) {
          const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + at + i);
          const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 8; ++e) y[i + e] = dyn_bits_to_f32((w[e / 2] >> (16 * (e & 1))) & 0xffffu, a.q_dtype);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i) y[i] = load_dyn_f32(a.q, a.q_dtype, at + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) y[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < D / 4; ++i) y[i] *= static_cast<float>(a.cache.signs[g * (D / 4) + i]);
    kv_rotate_lane<D>(y, lane);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(y[i]));
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // a power of two that puts the largest entry into [2^10, 2^11)
    const int exponent = top > 0.0f && top < INFINITY ? min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10, -110), 117) : 0;
    const float down = __uint_as_float(static_cast<uint32_t>(127 - exponent) << 23);
    factor[t] = a.scale * (1.44269504088896f / D) * __uint_as_float(static_cast<uint32_t>(127 + exponent) << 23);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = y[8 * c + e] * down;
        q[t][c][e] = static_cast<_Float16>(v);
        if constexpr (SPLIT > 0) q_rest[t][c][e] = static_cast<_Float16>(v - static_cast<float>(q[t][c][e]));
      }
    }
  }

  kv_f32x4 o[RT][D / 16];
  float sum[RT], ref[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    sum[t] = 0.0f;
    ref[t] = kKvNothing;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) o[t][j] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const int shift = a.cache.page_shift;
  const int32_t *table = a.table + request * a.table_stride;
  const auto page_at = [&](int key) {  // -1: not there
    const int column = key >> shift;
    const int page = column < a.table_width ? table[column] : -1;
    return page < a.cache.pages ? page : -1;
  };
  uint32_t k_raw[4][W];
  uint4 v_raw[D / 32], k_scale[2], v_scale[2];
  const auto load_keys = [&](int s, int page) {
    const int64_t block = static_cast<int64_t>(max(page, 0)) * a.cache.heads + kv_head;
    const int place = (s * 64 + 16 * (n >> 2)) & ((1 << shift) - 1);
    const uint32_t *from = reinterpret_cast<const uint32_t *>(a.cache.k_codes) + ((block << shift) + place + (n & 3)) * (D / 8) + g * W;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(from + 4 * t * (D / 8));
        k_raw[t][0] = v.x; k_raw[t][1] = v.y;
      } else {
#pragma unroll
        for (int w = 0; w < W; w += 4) {
          const uint4 v = *reinterpret_cast<const uint4 *>(from + 4 * t * (D / 8) + w);
          k_raw[t][w] = v.x; k_raw[t][w + 1] = v.y; k_raw[t][w + 2] = v.z; k_raw[t][w + 3] = v.w;
        }
      }
    }
  };
  const auto load_values = [&](int s, int page) {
    const int64_t block = static_cast<int64_t>(max(page, 0)) * a.cache.heads + kv_head;
    const int place = (s * 64 + 16 * g) & ((1 << shift) - 1);
    const uint8_t *from = a.cache.v_codes + ((block * (D / 2) + n) << shift) + place;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) v_raw[j] = *reinterpret_cast<const uint4 *>(from + (static_cast<int64_t>(16 * j) << shift));
  };
  const auto load_scales = [&](int s, int page) {
    const int64_t block = static_cast<int64_t>(max(page, 0)) * a.cache.heads + kv_head;
    const int place = (s * 64 + 16 * g) & ((1 << shift) - 1);
    const uint4 *k_from = reinterpret_cast<const uint4 *>(a.cache.k_scales + (block << shift) + place);
    const uint4 *v_from = reinterpret_cast<const uint4 *>(a.cache.v_scales + (block << shift) + place);
    k_scale[0] = k_from[0]; k_scale[1] = k_from[1];
    v_scale[0] = v_from[0]; v_scale[1] = v_from[1];
  };

  if (set < sets) {
    step += rank;
    int page_k = -1, page_v = -1, next_k = -1, next_v = -1;
    if (step < end) {
      page_k = page_at(step * 64 + 16 * (n >> 2));
      page_v = page_at(step * 64 + 16 * g);
      load_keys(step, page_k);
      load_scales(step, page_v);
      load_values(step, page_v);
      next_k = page_at((step + sharing) * 64 + 16 * (n >> 2));
      next_v = page_at((step + sharing) * 64 + 16 * g);
    }
    for (; step < end; step += sharing) {
      const int ahead = min(step + sharing, end - 1);  // (the last step asks for itself or an earlier one again)
      const bool more = step + sharing < end;
      // scores
      kv_f32x4 s[RT][4];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int k = 0; k < 4; ++k) s[t][k] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
          const kv_f16x8 codes = kv_decode8(k_raw[k][c]);
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            if constexpr (SPLIT > 0) s[t][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q_rest[t][c], s[t][k], 0, 0, 0);
            s[t][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q[t][c], s[t][k], 0, 0, 0);
          }
        }
      }
      float ks[16], vs[16];
      uint32_t top_scale = 0;
      {
        const uint32_t kw[8] = {k_scale[0].x, k_scale[0].y, k_scale[0].z, k_scale[0].w, k_scale[1].x, k_scale[1].y, k_scale[1].z, k_scale[1].w};
        const uint32_t vw[8] = {v_scale[0].x, v_scale[0].y, v_scale[0].z, v_scale[0].w, v_scale[1].x, v_scale[1].y, v_scale[1].z, v_scale[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          ks[2 * i] = __uint_as_float(kw[i] << 16);
          ks[2 * i + 1] = __uint_as_float(kw[i] & 0xffff0000u);
          vs[2 * i] = __uint_as_float(vw[i] << 16);
          vs[2 * i + 1] = __uint_as_float(vw[i] & 0xffff0000u);
        }
      }
      const int here_v = page_v;
      if (more) {
        load_keys(ahead, next_k);
        load_scales(ahead, next_v);
      }
      // masks: only where the step has keys that some row does not see, or that are not there
      const int first = step * 64;
      const bool masked = first + 63 > all_high || first < all_low || __builtin_amdgcn_ballot_w64(here_v < 0) != 0;
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = first + 16 * g + i;
          const bool there = key <= last_key && here_v >= 0;
          // A weight of 0 does not undo a scale that is NaN.  Where a value's is, the rows that see it get theirs through the
          // score; what lies behind the last key may be anything.
          const bool broken = vs[i] != vs[i];
          if (broken || !there) vs[i] = 0.0f;
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            const bool seen = there && key <= high[t] && key >= low[t];
            const float score = broken ? NAN : s[t][i >> 2][i & 3] * (ks[i] * factor[t]);
            s[t][i >> 2][i & 3] = seen ? score : -INFINITY;
          }
        }
      } else {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i >> 2][i & 3] *= ks[i] * factor[t];
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top_scale = max(top_scale, __float_as_uint(vs[i]));
      const float top_exponent = static_cast<float>(min(max(static_cast<int>(top_scale >> 23) - 126, -80), 80));  // b_t < 2^this
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        float best = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          best = fmaxf(best, s[t][i >> 2][i & 3]);
        }
        best += top_exponent;
        if (__builtin_amdgcn_ballot_w64(best - ref[t] > 15.0f) != 0) {
          best = fmaxf(best, __shfl_xor(best, 16, 64));
          best = fmaxf(best, __shfl_xor(best, 32, 64));
          const float to = fmaxf(ref[t], best - 10.0f), by = kv_exp2(ref[t] - to);
          ref[t] = to;
          sum[t] *= by;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) o[t][j] *= by;
        }
      }
      kv_f16x8 p[RT][2], p_rest[SPLIT > 1 ? RT : 1][2];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = kv_exp2(s[t][i >> 2][i & 3] - ref[t]);
          sum[t] += e;
          const float w = e * vs[i];
          const int half = i >> 3, at = 2 * (i & 3) + ((i >> 2) & 1);  // tiles 2 * half and 2 * half + 1 side by side
          p[t][half][at] = static_cast<_Float16>(w);
          if constexpr (SPLIT > 1) p_rest[t][half][at] = static_cast<_Float16>(w - static_cast<float>(p[t][half][at]));
        }
      }
      // outputs
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint32_t w[4] = {v_raw[j].x, v_raw[j].y, v_raw[j].z, v_raw[j].w};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x = w[2 * half], y = w[2 * half + 1];
          const kv_f16x8 even = kv_decode8((x & 0x0f0f0f0fu) | ((y & 0x0f0f0f0fu) << 4));
          const kv_f16x8 odd = kv_decode8(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u));
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
      if (more) load_values(ahead, next_v);
      page_v = next_v;
      next_k = page_at((step + 2 * sharing) * 64 + 16 * (n >> 2));
      next_v = page_at((step + 2 * sharing) * 64 + 16 * g);
    }
  }

  // the wavefronts that shared the keys: neighbours first, then the two pairs, in this order
  const auto give = [&](int place) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      join[place][2 * t][lane] = ref[t];
      join[place][2 * t + 1][lane] = sum[t];
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) join[place][2 * RT + (t * (D / 16) + j) * 4 + r][lane] = o[t][j][r];
      }
    }
  };
  const auto take = [&](int place) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float theirs = join[place][2 * t][lane], both = fmaxf(ref[t], theirs);
      const float mine = kv_exp2(ref[t] - both), other = kv_exp2(theirs - both);
      ref[t] = both;
      sum[t] = sum[t] * mine + join[place][2 * t + 1][lane] * other;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[t][j][r] = o[t][j][r] * mine + join[place][2 * RT + (t * (D / 16) + j) * 4 + r][lane] * other;
      }
    }
  };
  if (sharing > 1) {
    if (rank & 1) give(wave >> 1);
    __syncthreads();
    if ((rank & 1) == 0) take(wave >> 1);
    if (sharing == 4) {
      __syncthreads();
      if (rank == 2) give(1);
      __syncthreads();
      if (rank == 0) take(1);
    }
  }
  if (rank != 0 || set >= sets) return;

#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float l = sum[t];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const float by = l != 0.0f ? (1.0f / D) / l : 0.0f;  // (no key: zeros)
    // dimension 32 j + 8 g + 2 r + parity is in o[2 j + parity][r]
    float y[D / 4];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[8 * j + 2 * r] = o[t][2 * j][r] * by;
        y[8 * j + 2 * r + 1] = o[t][2 * j + 1][r] * by;
      }
    }
    kv_rotate_lane<D>(y, lane);  // (its order of the dimensions over lanes and registers does not matter: every pair of bits takes part once)
    if (token[t] < 0) continue;
    const int64_t row = static_cast<int64_t>(token[t]) * a.heads + head[t];
    const float log_sum = l != 0.0f ? (ref[t] + __builtin_amdgcn_logf(l)) * 0.693147180559945f : -INFINITY;
    if (a.parts > 1) {
      const int64_t at = static_cast<int64_t>(part) * a.tokens * a.heads + row;
      float *to = a.part_out + at * D + 8 * g;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint2 sign = *reinterpret_cast<const uint2 *>(a.cache.signs + 32 * j + 8 * g);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ((e < 4 ? sign.x : sign.y) >> (8 * (e & 3) + 7)) & 1 ? -y[8 * j + e] : y[8 * j + e];
        reinterpret_cast<float4 *>(to + 32 * j)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(to + 32 * j)[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
      if (g == 0) a.part_lse[at] = log_sum;
      continue;
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint2 sign = *reinterpret_cast<const uint2 *>(a.cache.signs + 32 * j + 8 * g);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = ((e < 4 ? sign.x : sign.y) >> (8 * (e & 3) + 7)) & 1 ? -y[8 * j + e] : y[8 * j + e];
      const int64_t at = row * D + 32 * j + 8 * g;
      if (a.q_dtype == OQ_F32) {
        reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at)[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = a.q_dtype == OQ_F16 ? f32_to_f16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_f16_bits(v[2 * e + 1])) << 16
                                     : f32_to_bf16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16;
        }
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    if (a.lse != nullptr && g == 0) a.lse[row] = log_sum;
  }
}

template <int D, int RT, int SPLIT>
void kv_attend_launch(const KvAttendArgs &a, hipStream_t stream) {
  launch_kernel(kv_attend_kernel<D, RT, SPLIT>, dim3(static_cast<unsigned>(a.cache.heads) * a.tiles, static_cast<unsigned>(a.parts)), dim3(256), 0,
                stream, a);
}

}  // namespace oq
