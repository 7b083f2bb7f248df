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
// Precision.  The codes are exact in fp16.  A rotated query is scaled by a power of two to use fp16's range (its own, or one that it shares
// with rows of about its size) and rounded to its eleven bits, and so are the weights e^(s - R) b_t; SPLIT 1 (fp16 inputs) keeps a second fp16 part of the query, SPLIT 2 (fp32
// inputs) of both, which leaves 22 bits.  Sums, maxima and exponentials are fp32.
// The reference R of a row is not its maximum: it is raised when a weight could pass 2^15, to where the largest is about 2^10.
// Rows are so rescaled a few times in all, no maximum is exchanged between lanes in between, and the fp16 weights have 24
// binary digits below their largest before they lose any.  R holds the exponent of the weightiest keys' value
// scales too (b_t is anything, from 2^-80 on: below it R stays, so that l stays finite; above 2^112 l, whose weights are then
// 2^-102 and less, has fewer than 24 digits before an fp32 ends).
//
// Two kernels.  Few rows (single tokens, at most kKvFewRows of a request): four wavefronts share the keys of sixteen rows, every
// one decodes for itself, and the launch is bound by the cache's bytes.  Many rows (a prompt): the wavefronts have rows of
// their own and the same keys, which they decode once for all of them into LDS; bound by the vector instructions around the
// products.
#pragma once

#include <type_traits>

#include "kv_cache.h"

namespace oq {

typedef float kv_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv_u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 kv_bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kKvNothing = -3.402823466e38f;  // R of a row that has seen no key: below every score
constexpr int kKvFewRows = 64;          // rows of a request that the first kernel takes
constexpr int kKvManyRows = 128;        // rows of a workgroup of the second
constexpr int kKvCutTiles = 384;        // tiles of a launch of the second that is cut, at most

// Tiles in front of request r when its rows begin at `row`: enough for every request's last, unfilled tile.
__host__ __device__ inline int64_t kv_tile_base(int64_t row, int64_t r) { return row / kKvManyRows + r; }

__device__ __forceinline__ float kv_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^(x / 2).  A sum of weights is taken to another reference in two steps of this: with value scales from 2^-80 to 2^127 in it the references are further
// apart than the exponents of an fp32 reach, the sums themselves are not.
__device__ __forceinline__ float kv_half_power(float x) { return kv_exp2(0.5f * x); }

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

typedef short kv_i16x2 __attribute__((ext_vector_type(2)));
constexpr int kDppHalfMirror = 0x141, kDppMirror = 0x140;  // of eight lanes, of sixteen
template <int CTRL>
__device__ __forceinline__ kv_i16x2 kv_dpp_max(kv_i16x2 x) {
  return __builtin_elementwise_max(x, __builtin_bit_cast(kv_i16x2, kv_dpp<CTRL>(__builtin_bit_cast(uint32_t, x))));
}
__device__ __forceinline__ kv_i16x2 kv_row_max(kv_i16x2 x) {  // of sixteen lanes
  return kv_dpp_max<kDppMirror>(kv_dpp_max<kDppHalfMirror>(kv_dpp_max<kDppXor2>(kv_dpp_max<kDppXor1>(x))));
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

__device__ __forceinline__ int kv_length_of(const KvAttendArgs &a, int request) { return request < a.requests ? max(a.lengths[request], 0) : 0; }
__device__ __forceinline__ void kv_keys_of(const KvAttendArgs &a, KvRows &r, int length) {
  r.length = length;
  const int64_t reach = static_cast<int64_t>(a.table_width) << a.cache.page_shift;  // what lies behind the table is not there
  r.last_key = static_cast<int>(min(static_cast<int64_t>(r.length), reach)) - 1;
}
__device__ __forceinline__ void kv_keys_of(const KvAttendArgs &a, KvRows &r) { kv_keys_of(a, r, kv_length_of(a, r.request)); }

__device__ __forceinline__ int kv_low_of(const KvAttendArgs &a, int position) {  // the first key that a query there sees (no sum passes 32 bits: positions may be negative)
  return a.window != 0 && position >= a.window ? position - a.window + 1 : 0;
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
  s.lowest = kv_low_of(a, from);
  s.all_low = kv_low_of(a, to);
  return s;
}

// Tile i of a launch: its rows, false where there are none.
__device__ __forceinline__ bool kv_few_tile(const KvAttendArgs &a, int i, KvRows &r) {
  r.request = i / a.few_tiles;
  r.first = (i - r.request * a.few_tiles) * 16;
  r.start = r.request;
  r.fresh = 1;
  if (a.starts != nullptr) {
    r.start = kv_start_of(a, r.request);
    r.fresh = max(kv_start_of(a, r.request + 1) - r.start, 0);
    if (static_cast<int64_t>(r.fresh) * a.group > kKvFewRows) return false;
  }
  r.rows = min(r.fresh * a.group - r.first, 16);
  if (r.rows <= 0) return false;
  kv_keys_of(a, r);
  return true;
}

// The request that tile i belongs to; start_of(r): where its tokens begin.
template <typename Starts>
__device__ __forceinline__ int kv_request_of(const KvAttendArgs &a, int i, const Starts &start_of) {
  int low = 0, high = a.requests + 1;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (kv_tile_base(static_cast<int64_t>(start_of(mid)) * a.group, mid) <= i) low = mid; else high = mid;
  }
  return low;
}

// Its rows, r.request, r.start and r.fresh known.
__device__ __forceinline__ bool kv_rows_of(const KvAttendArgs &a, int i, KvRows &r) {
  const int64_t first = (i - kv_tile_base(static_cast<int64_t>(r.start) * a.group, r.request)) * kKvManyRows, all = static_cast<int64_t>(r.fresh) * a.group;
  if (first >= all || all <= a.few_rows) return false;
  r.first = static_cast<int>(first);
  r.rows = static_cast<int>(min(all - first, static_cast<int64_t>(kKvManyRows)));
  return true;
}

__device__ __forceinline__ bool kv_many_tile(const KvAttendArgs &a, int i, KvRows &r) {
  r.request = kv_request_of(a, i, [&](int request) { return kv_start_of(a, request); });
  r.start = kv_start_of(a, r.request);
  r.fresh = max(kv_start_of(a, r.request + 1) - r.start, 0);
  if (!kv_rows_of(a, i, r)) return false;
  kv_keys_of(a, r);
  return true;
}

template <bool MANY>
__device__ __forceinline__ bool kv_tile(const KvAttendArgs &a, int i, KvRows &r) {
  if constexpr (MANY) return kv_many_tile(a, i, r);
  else return kv_few_tile(a, i, r);
}

__device__ __forceinline__ int kv_steps_of(const KvSpan &span) {  // one for a tile without keys: somebody writes its zeros
  return span.highest >= span.lowest ? (span.highest >> 6) - (span.lowest >> 6) + 1 : 1;
}
__device__ __forceinline__ int kv_counted_steps(const KvSpan &span) { return min(kv_steps_of(span), 1 << 22); }  // sums of some hundred tiles stay below 2^31

// A workgroup's part of a tile.
struct KvPart {
  KvRows rows;
  int tile, index, count;  // of the tile's parts
  int place;               // of the part among those of cut tiles
  __device__ __forceinline__ int from(int steps, int i) const { return steps / count * i + min(steps % count, i); }  // where part i begins
};
__device__ __forceinline__ int kv_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int kv_from_lane(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }

__device__ __forceinline__ int kv_longer(int longest, int made, int target) {
  return static_cast<int>(min((static_cast<int64_t>(longest) * made + target - 1) / target, static_cast<int64_t>(0x3fffffff)));
}

// Part `group` of the launch's, false behind the last.  Every workgroup counts for itself: the tiles' steps, and from those the parts.
//
// Up to kKvCutTiles tiles every wavefront does so, a lane for `held` tiles in a row.  Parts of one tile are equal, but those of different tiles are
// not, some half of the others, so the long ones come first where there are more than the chip holds at once (64 requests of 3300 to 16384
// tokens: 134 -> 130 us; where there are not, it would cost 0.4).
// Many rows have no more parts than the chip holds at once, two on a compute unit: there the second half of the launch goes the other
// way, and a long one's neighbour is short (parts of 19 to 46 steps, 480 of them, D = 64, fp16: 103 -> 87 us with both;
// 532 parts before, whose last twenty began when the others ended).
struct KvPick {
  int tile, all_cut;  // (the number of all parts of cut tiles)
};
template <bool MANY, int HELD>
__device__ __forceinline__ bool kv_pick(const KvCut &cut, int tiles, int held, const int (&steps)[HELD], int group, KvPart &part, KvPick &pick) {
  constexpr int CLASSES = 8;
  int total = 0;
#pragma unroll
  for (int h = 0; h < HELD; ++h) total += steps[h];
  total = kv_from_lane(kv_sums(total), 63);
  int longest = max((total + cut.target - 1) / cut.target, cut.least), enough = total, rounds = 2;
  if constexpr (MANY) {
    // No more parts than `target`, and rounding every tile's up makes half a part more of each.  Four times total / target is enough
    // whatever the tiles, as they are fewer than three quarters of the parts.
    const int share = (total + cut.target - 1) / cut.target;
    longest = max(static_cast<int>(static_cast<float>(total) / (static_cast<float>(cut.target) - 0.5f * static_cast<float>(tiles))) + 1, cut.least);
    enough = max(static_cast<int>(min(4 * static_cast<int64_t>(share), static_cast<int64_t>(0x3fffffff))), longest);
    rounds = 6;
  }
  int count[HELD], all, in_lane, in_cut;
  for (int round = 0;; ++round) {
    const float by = 1.0f / static_cast<float>(longest);
    in_lane = in_cut = 0;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      count[h] = 0;
      if (h < held) {
        int n = static_cast<int>(static_cast<float>(steps[h]) * by);  // (below 2^12, so one off at most)
        n += n * longest < steps[h] ? 1 : 0;
        n += n * longest < steps[h] ? 1 : 0;
        n -= n > 0 && (n - 1) * longest >= steps[h] ? 1 : 0;
        count[h] = n;
        in_lane += n;
        in_cut += n > 1 ? n : 0;
      }
    }
    all = kv_from_lane(kv_sums(in_lane), 63);
    if (all <= cut.target || longest >= enough || (!MANY && round == rounds)) break;
    longest = MANY && round >= rounds ? enough : min(kv_longer(longest, all, cut.target), enough);
  }
  const int cut_sum = kv_sums(in_cut);
  pick.all_cut = kv_from_lane(cut_sum, 63);
  if (group >= all) return false;
  int at, found = 0, found_kind = CLASSES, kind[HELD] = {};
  if (!MANY && !cut.sorted) {
    const int sums = kv_sums(in_lane);
    found = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sums > group));
    at = group - kv_from_lane(sums - in_lane, found);
    found_kind = 0;
  } else {
    // Parts by length, in classes of longest / 16, all below half of it in the last; two classes' sums in one number (each below 2^16).
    int classes[CLASSES / 2] = {};
    const float by = 2.0f * CLASSES / static_cast<float>(longest);
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      kind[h] = CLASSES;
      if (h < held) {
        const float length = static_cast<float>(steps[h]) * __builtin_amdgcn_rcpf(static_cast<float>(max(count[h], 1)));
        kind[h] = max(min(static_cast<int>(2.0f * CLASSES - length * by), CLASSES - 1), 0);
#pragma unroll
        for (int c = 0; c < CLASSES / 2; ++c) classes[c] += kind[h] >> 1 == c ? count[h] << (16 * (kind[h] & 1)) : 0;
      }
    }
    const int half = (cut.target + 1) >> 1;
    at = !MANY || group < half ? group : all - 1 - (group - half);
#pragma unroll
    for (int c = 0; c < CLASSES; c += 2) {
      const int sums = kv_sums(classes[c >> 1]), sum = kv_from_lane(sums, 63);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int up_to = sums >> (16 * e) & 0xffff, its = sum >> (16 * e) & 0xffff;
        if (found_kind == CLASSES) {
          if (at < its) {
            found = __builtin_ctzll(__builtin_amdgcn_ballot_w64(up_to > at));
            at -= kv_from_lane(up_to - (classes[c >> 1] >> (16 * e) & 0xffff), found);
            found_kind = c + e;
          } else {
            at -= its;
          }
        }
      }
    }
  }
  part.place = kv_from_lane(cut_sum - in_cut, found);
  pick.tile = -1;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    if (h < held && pick.tile < 0) {
      const int n = kv_from_lane(count[h], found), of_kind = kv_from_lane(kind[h], found);
      if (of_kind == found_kind && at < n) {
        pick.tile = found * held + h;
        part.count = n;
      } else {
        at -= of_kind == found_kind ? n : 0;
        part.place += n > 1 ? n : 0;
      }
    }
  }
  part.tile = pick.tile;
  part.index = at;
  part.place += at;
  return true;
}
__device__ __forceinline__ KvRows kv_uniform(const KvRows &r) {
  return {kv_uniform(r.request), kv_uniform(r.start), kv_uniform(r.fresh), kv_uniform(r.length), kv_uniform(r.first), kv_uniform(r.rows), kv_uniform(r.last_key)};
}
__device__ __forceinline__ int2 *kv_map_of(const KvCut &cut, int kv_head) { return cut.map + static_cast<int64_t>(kv_head) * (cut.places + 1); }
__device__ __forceinline__ int2 kv_map_entry(const KvPart &part) { return part.index == 0 ? make_int2(part.tile, part.count) : make_int2(-1, 0); }

template <int THREADS>
__device__ __forceinline__ bool kv_few_part(const KvAttendArgs &a, int tiles, const KvCut &cut, int kv_head, int group, KvPart &part) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  KvRows r = {};
  const auto steps_of = [&](int i) { return kv_few_tile(a, i, r) ? kv_counted_steps(kv_span_of(a, r, r.first, r.rows)) : 0; };
  int2 *const map = kv_map_of(cut, kv_head);
  if (tiles <= 64 && !cut.sorted) {  // a tile a lane, and the order is theirs: a short launch notices every instruction
    const int steps = lane < tiles ? steps_of(lane) : 0;
    const int total = kv_from_lane(kv_sums(steps), 63);
    int longest = max((total + cut.target - 1) / cut.target, cut.least);
    int count = (steps + longest - 1) / longest, sum = kv_sums(count);
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // (rounding every tile's parts up makes more of them than meant)
      const int made = kv_from_lane(sum, 63);
      if (made > cut.target && longest < total) {
        longest = kv_longer(longest, made, cut.target);
        count = (steps + longest - 1) / longest;
        sum = kv_sums(count);
      }
    }
    const int in_cut = count > 1 ? count : 0, cut_sum = kv_sums(in_cut);
    if (group == 0 && tid == 0) map[cut.places] = make_int2(kv_from_lane(cut_sum, 63), 0);
    if (group >= kv_from_lane(sum, 63)) return false;
    const int found = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > group));
    part.tile = found;
    part.count = kv_from_lane(count, found);
    part.index = group - kv_from_lane(sum - count, found);
    part.place = kv_from_lane(cut_sum - in_cut, found) + part.index;
    part.rows = {kv_from_lane(r.request, found), kv_from_lane(r.start, found), kv_from_lane(r.fresh, found), kv_from_lane(r.length, found),
                 kv_from_lane(r.first, found), kv_from_lane(r.rows, found), kv_from_lane(r.last_key, found)};
  } else if (tiles <= kKvCutTiles) {  // no wavefront needs another: the first keys are a barrier nearer
    bool there;
    KvPick pick;
    const int held = (tiles + 63) >> 6;
    int steps[kKvCutTiles / 64];
#pragma unroll
    for (int h = 0; h < kKvCutTiles / 64; ++h) steps[h] = h < held && lane * held + h < tiles ? steps_of(lane * held + h) : 0;
    there = kv_pick<false>(cut, tiles, held, steps, group, part, pick);
    if (there) {
      kv_few_tile(a, part.tile, r);
      part.rows = kv_uniform(r);
    }
    if (group == 0 && tid == 0) map[cut.places] = make_int2(pick.all_cut, 0);
    if (!there) return false;
  } else {
    __shared__ int64_t wave_sums[THREADS / 64];
    __shared__ int2 wave_counts[THREADS / 64];
    __shared__ int found[4];
    __shared__ KvRows found_rows;
    const int chunk = (tiles + THREADS - 1) / THREADS, from = tid * chunk, to = min(from + chunk, tiles);
    int64_t own = 0;
    for (int i = from; i < to; ++i) own += steps_of(i);
    const int only = static_cast<int>(own);  // (of a thread with one tile)
#pragma unroll
    for (int d = 1; d < 64; d *= 2) own += __shfl_xor(static_cast<long long>(own), d, 64);
    if (lane == 0) wave_sums[wave] = own;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) total += wave_sums[w];
    int longest = static_cast<int>(max((total + cut.target - 1) / cut.target, static_cast<int64_t>(cut.least)));
    int count, ahead, cut_ahead, all, all_cut;
    for (int round = 0;; ++round) {
      count = 0;
      int in_cut = 0;
      for (int i = from; i < to; ++i) {
        const int n = ((chunk == 1 ? only : steps_of(i)) + longest - 1) / longest;
        count += n;
        in_cut += n > 1 ? n : 0;
      }
      const int sum = kv_sums(count), cut_sum = kv_sums(in_cut);
      __syncthreads();
      if (lane == 63) wave_counts[wave] = make_int2(sum, cut_sum);
      __syncthreads();
      ahead = sum - count; cut_ahead = cut_sum - in_cut; all = 0; all_cut = 0;
#pragma unroll
      for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) {
          ahead += wave_counts[w].x;
          cut_ahead += wave_counts[w].y;
        }
        all += wave_counts[w].x;
        all_cut += wave_counts[w].y;
      }
      if (chunk > 1 || round == 2 || all <= cut.target || longest >= total) break;  // (many tiles even out by themselves)
      longest = kv_longer(longest, all, cut.target);
    }
    if (group == 0 && tid == 0) map[cut.places] = make_int2(all_cut, 0);
    if (group >= all) return false;
    if (group >= ahead && group < ahead + count) {
      int i = from, n = (steps_of(i) + longest - 1) / longest;
      while (group >= ahead + n) {
        ahead += n;
        cut_ahead += n > 1 ? n : 0;
        n = (steps_of(++i) + longest - 1) / longest;
      }
      found[0] = i;
      found[1] = n;
      found[2] = group - ahead;
      found[3] = cut_ahead + group - ahead;
      found_rows = r;
    }
    __syncthreads();
    part.tile = kv_uniform(found[0]);
    part.count = kv_uniform(found[1]);
    part.index = kv_uniform(found[2]);
    part.place = kv_uniform(found[3]);
    part.rows = kv_uniform(found_rows);
  }
  if (part.count > 1 && tid == 0) map[part.place] = kv_map_entry(part);
  return true;
}

// For many rows requests and tiles are looked up once a workgroup.
struct KvCounted {
  int starts[kKvCutTiles + 2], lengths[kKvCutTiles + 2];  // of the requests
  int steps[kKvCutTiles], requests[kKvCutTiles];          // of the tiles
};
template <int THREADS>
__device__ __forceinline__ bool kv_many_part(const KvAttendArgs &a, int kv_head, int group, KvCounted &counted, KvPart &part) {
  constexpr int HELD = kKvCutTiles / 64;
  const int tid = threadIdx.x, lane = tid & 63, tiles = a.many_tiles;
  for (int i = tid; i <= a.requests + 1; i += THREADS) {
    counted.starts[i] = kv_start_of(a, i);
    counted.lengths[i] = kv_length_of(a, i);
  }
  __syncthreads();
  const auto rows_of = [&](int request, int i, KvRows &r) {
    r.request = request;
    r.start = counted.starts[request];
    r.fresh = max(counted.starts[request + 1] - r.start, 0);
    kv_keys_of(a, r, counted.lengths[request]);
    return kv_rows_of(a, i, r);
  };
  KvRows r;
  for (int i = tid; i < tiles; i += THREADS) {
    const int request = kv_request_of(a, i, [&](int request) { return counted.starts[request]; });
    counted.steps[i] = rows_of(request, i, r) ? kv_counted_steps(kv_span_of(a, r, r.first, r.rows)) : 0;
    counted.requests[i] = request;
  }
  __syncthreads();
  const int held = (tiles + 63) >> 6;
  int steps[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h) steps[h] = h < held && lane * held + h < tiles ? counted.steps[lane * held + h] : 0;
  KvPick pick;
  const bool there = kv_pick<true>(a.many, tiles, held, steps, group, part, pick);
  int2 *const map = kv_map_of(a.many, kv_head);
  if (group == 0 && tid == 0) map[a.many.places] = make_int2(pick.all_cut, 0);
  if (!there) return false;
  rows_of(counted.requests[part.tile], part.tile, r);
  part.rows = kv_uniform(r);
  __syncthreads();  // (the memory is somebody else's from here on)
  if (part.count > 1 && tid == 0) map[part.place] = kv_map_entry(part);
  return true;
}

// The table's entry for a key, as it stands there: it is looked at when the page is asked for, a step later, so that nothing waits for
// it here (loads come back in order: such a wait is one for everything requested before).  Columns behind the table are clamped;
// their keys are behind the last one.
__device__ __forceinline__ int kv_page_at(const KvAttendArgs &a, const int32_t *table, int key) {
  return table[min(key >> a.cache.page_shift, a.table_width - 1)];
}
__device__ __forceinline__ bool kv_page_there(const KvAttendArgs &a, int page) { return static_cast<uint32_t>(page) < static_cast<uint32_t>(a.cache.pages); }
__device__ __forceinline__ int64_t kv_block_of(const KvAttendArgs &a, int page, int kv_head) {  // any that exists, where the page does not
  return static_cast<int64_t>(kv_page_there(a, page) ? page : 0) * a.cache.heads + kv_head;
}

// Where pages hold whole steps (64 tokens and more) a step's page is the same for all lanes: its entry is read and its address made by scalar
// instructions, and lanes add what is theirs.  (Forty vector instructions of a step otherwise, of some three hundred.)
__device__ __forceinline__ int kv_scalar_page_at(const KvAttendArgs &a, const int32_t *table, int key) {
  const int column = __builtin_amdgcn_readfirstlane(min(key >> a.cache.page_shift, a.table_width - 1));
  return *(const __attribute__((address_space(4))) int32_t *)(table + column);
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
  k.low = kv_low_of(a, position);
  return k;
}

// A row's quarter of a query as it comes, and the signs of its dimensions: requested before the keys, so that it is there before them.
template <int D, int SPLIT>
struct KvQuery {
  static constexpr int WORDS = D / 4 * (SPLIT == 2 ? 4 : 2) / 4;
  uint32_t raw[WORDS], signs[D / 16];

  __device__ __forceinline__ void request(const KvAttendArgs &a, const KvRow &row, int g) {
#pragma unroll
    for (int i = 0; i < D / 16; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4 *>(a.cache.signs + g * (D / 4) + 4 * i);
      signs[i] = v.x; signs[i + 1] = v.y; signs[i + 2] = v.z; signs[i + 3] = v.w;
    }
    // (a lane without a row reads one that exists, and makes zeros of it)
    const int64_t at = max(row.token, 0) * a.q_token_stride + row.head * a.q_head_stride + g * (D / 4);
    if (a.q_wide) {
      const uint4 *from = reinterpret_cast<const uint4 *>(static_cast<const char *>(a.q) + at * (SPLIT == 2 ? 4 : 2));
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const uint4 v = from[i / 4];
        raw[i] = v.x; raw[i + 1] = v.y; raw[i + 2] = v.z; raw[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        if constexpr (SPLIT == 2) raw[i] = static_cast<const uint32_t *>(a.q)[at + i];
        else raw[i] = static_cast<const uint16_t *>(a.q)[at + 2 * i] | static_cast<uint32_t>(static_cast<const uint16_t *>(a.q)[at + 2 * i + 1]) << 16;
      }
    }
  }

  // Rotated; gives the largest magnitude of the row.
  //
  // Values of sixteen bits go through the matrix units as they come: H's entries are signs, so every product is exact and the sums are
  // fp32's as in the butterflies.  The k-th chunk's B operand is the lane's dimensions g * D / 4 + 8 c .., row m of tile t is dimension
  // (m >> 2) * D / 4 + 4 t + (m & 3), so that the results lie as the butterflies leave them.  The sign of an entry is the parity of
  // the two dimensions' common bits: those of m >> 2 and g, of m & 3 and the element, the third of t and the element, and a
  // whole operand's sign of t >> 1 and c.  (D = 128: 32 matrix instructions for some 450 vector ones; one request of 1003 tokens 10.5 -> 9.7 us.)
  __device__ __forceinline__ float rotate(bool there, float (&y)[D / 4]) const {
    if constexpr (SPLIT < 2) {
      const int lane = threadIdx.x & 63, m = lane & 15;
      const uint32_t one = SPLIT == 0 ? 0x3f803f80u : 0x3c003c00u, minus = 0x80008000u;
      const uint32_t all = __builtin_popcount((m >> 2) & (lane >> 4)) & 1 ? minus : 0u, odd = m & 1 ? 0x80000000u : 0u, second = m & 2 ? minus : 0u;
      const uint32_t first = one ^ all ^ odd, next = first ^ second;
      const kv_u32x4 entries[2][2] = {{{first, next, first, next}, {first ^ minus, next ^ minus, first ^ minus, next ^ minus}},
                                      {{first, next, first ^ minus, next ^ minus}, {first ^ minus, next ^ minus, first, next}}};
      kv_u32x4 x[D / 32];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const uint32_t low = ((signs[i] << 8) & 0x8000u) | ((signs[i] << 16) & 0x80000000u), high = ((signs[i] >> 8) & 0x8000u) | (signs[i] & 0x80000000u);
        x[i / 2][2 * (i & 1)] = there ? raw[2 * i] ^ low : 0u;
        x[i / 2][2 * (i & 1) + 1] = there ? raw[2 * i + 1] ^ high : 0u;
      }
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        kv_f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const kv_u32x4 h = entries[t & 1][__builtin_popcount((t >> 1) & c) & 1];
          if constexpr (SPLIT == 0) sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(kv_bf16x8, h), __builtin_bit_cast(kv_bf16x8, x[c]), sum, 0, 0, 0);
          else sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(kv_f16x8, h), __builtin_bit_cast(kv_f16x8, x[c]), sum, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) y[4 * t + r] = sum[r];
      }
    } else {
#pragma unroll
      for (int i = 0; i < D / 4; ++i) {
        const float sign = static_cast<float>(static_cast<int8_t>(signs[i / 4] >> (8 * (i & 3))));
        y[i] = there ? __uint_as_float(raw[i]) * sign : 0.0f;
      }
      kv_rotate_lane<D>(y);
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) top = fmaxf(top, fabsf(y[i]));
    return kv_over_groups(top, kv_max_of);
  }
};

// The power of two 2^-exponent puts `top` into [2^10, 2^11).
__device__ __forceinline__ int kv_query_exponent(float top) {
  return top > 0.0f && top < INFINITY ? min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 10, -110), 117) : 0;
}
// How far apart the exponents of rows may be that share one: an entry's last place is then 2^-25 / 2^(10 - spread) of its row's top, and
// the root of D entries' worth of that stays below a part's own rounding (2^-12, of two parts 2^-22).
template <int SPLIT>
constexpr int kv_query_spread() { return SPLIT == 0 ? 16 : 8; }
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

// (fmaxf of values that come from a branch is two instructions: the compiler first makes sure that a NaN is quiet.)
__device__ __forceinline__ float kv_max3(float a, float b, float c) {
  float m;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(a), "v"(b), "v"(c));
  return m;
}

__device__ __forceinline__ float kv_exponent_of(int scale) { return static_cast<float>(max((scale >> 23) - 126, -80)); }  // the scale (its bits) is below 2^this
__device__ __forceinline__ int kv_largest_scale(const float (&vs)[16]) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(vs[i]));
  return static_cast<int>(top);
}

// Scales that are further apart than 2^8 are not of about one size.  (A first token's value is often some 2^4 smaller than the others; the weights
// keep eleven digits down to 2^-16 of the largest where R is 2^8 too high.)
constexpr int kKvMixed = 8;

// (These two by instructions of their own: what they give is otherwise found in front of the branch that asks for it, whether it is taken or not.)
__device__ __forceinline__ int kv_smallest_scale(const float (&vs)[16]) {
  int low = __float_as_int(vs[15]);
#pragma unroll
  for (int i = 1; i < 15; i += 2) asm volatile("v_min3_i32 %0, %0, %1, %2" : "+v"(low) : "v"(vs[i]), "v"(vs[i + 1]));
  return min(low, __float_as_int(vs[0]));
}
__device__ __forceinline__ float kv_exponent_alone(float scale) {
  int bits;
  asm volatile("v_mov_b32 %0, %1" : "=v"(bits) : "v"(scale));
  return kv_exponent_of(bits < 0x7f800000 ? bits : 0);  // (a NaN has no part in where R goes)
}

// x: scores minus R.  Raises R where a weight could pass 2^15, O along with it.  The exponent of the largest of the sixteen scales belongs to a key
// that the row may not see or hardly weigh: it tells cheaply that no weight is near 2^15, and where the scales are of about one size, where R goes.
// Where they are not (mixed()), each key is taken with its own exponent, so that a large value raises R for the rows that it has weight in, and the
// others keep their weights' digits.  (Always with its own: a prompt of 2048, D = 64, 46.0 -> 50 us; so 46.6.)
template <int D, typename Mixed>
__device__ __forceinline__ void kv_keep_in_range(float (&x)[16], const float (&vs)[16], float top_exponent, const Mixed &mixed, KvState &st, kv_f32x4 (&o)[D / 16]) {
  float best = kv_max3(x[0], x[1], x[2]), other = kv_max3(x[3], x[4], x[5]);
  best = kv_max3(best, x[6], x[7]);
  other = kv_max3(other, x[8], x[9]);
  best = kv_max3(best, x[10], x[11]);
  other = kv_max3(other, x[12], x[13]);
  best = kv_max3(best, x[14], x[15]);
  best = kv_max3(best, other, other) + top_exponent;
  if (__builtin_amdgcn_ballot_w64(best > st.limit) != 0) {
    best = kv_over_groups(best, kv_max_of);
    bool raise = best > st.limit;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(mixed()) != 0, false)) {
      best = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) best = fmaxf(best, x[i] + kv_exponent_alone(vs[i]));
      best = kv_over_groups(best, kv_max_of);
      raise = raise && best > fminf(st.limit, 10.0f);  // (wherever it is above 10, so that the next steps need not look)
    }
    // (Down only where nothing is summed up yet.  Scores beyond 2^26 are whole powers of two apart: what is meant may be rounded to an R too low.)
    float up = best - 10.0f;
    up = raise ? (best - up > 15.0f ? best : up) : 0.0f;
    const float half = kv_half_power(fminf(-up, 0.0f)), by = half * half;
    st.ref += up;
    st.sum = st.sum * half * half;
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

// Keys that a row does not see, or that are not there.  A weight of 0 does not undo a scale that is NaN, so none is multiplied by one.
__device__ __forceinline__ bool kv_seen(int key, bool there, const KvRow &row) { return there && key <= row.high && key >= row.low; }

// Where several rows share the scales: in the place of what lies behind the last key, which may be anything, stands the lane's first scale (of the
// others' size), and of a broken value zero.  Those steps are noted, and the rows that see such a value become NaN in the end, not through
// their weights, whose sum is a result too and has no value in it.
struct KvBroken {
  int from, to;  // steps
  __device__ __forceinline__ void begin() { from = 0x7fffffff; to = -1; }
  __device__ __forceinline__ void look(float (&vs)[16], int step) {
    uint32_t top = __float_as_uint(vs[0]);
    const float last = vs[15];
#pragma unroll
    for (int i = 1; i < 15; i += 2) asm volatile("v_max3_u32 %0, %0, %1, %2" : "+v"(top) : "v"(vs[i]), "v"(vs[i + 1]));  // (as above)
#pragma unroll
    for (int i = 0; i < 16; ++i) vs[i] = vs[i] != vs[i] ? 0.0f : vs[i];
    const bool any = __builtin_amdgcn_ballot_w64(max(top, __float_as_uint(last)) > 0x7f800000u) != 0;  // (a branch here costs the steps without a mask, too)
    from = any ? min(from, step) : from;
    to = any ? step : to;
  }
  // NaN for a row that sees one of them, otherwise 0.
  __device__ __forceinline__ float of(const KvAttendArgs &a, const int32_t *table, int last_key, const KvRow &row, int kv_head, int g) const {
    float found = 0.0f;
    const int last = min(min(row.high, last_key), 64 * to + 63), in_page = (1 << a.cache.page_shift) - 1;
    for (int key = max(row.low, 64 * from) + g; key <= last; key += 4) {
      const int page = table[key >> a.cache.page_shift];
      if (!kv_page_there(a, page)) continue;
      const float scale = bf16_bits_to_f32(a.cache.v_scales[(kv_block_of(a, page, kv_head) << a.cache.page_shift) + (key & in_page)]);
      found = scale != scale ? NAN : found;
    }
    return kv_over_groups(found, kv_sum_of);
  }
};

// Sixteen token bytes of two dimensions -> the A operands of the even and the odd one, tiles 2 * half and 2 * half + 1 side by side.
__device__ __forceinline__ void kv_decode_values(uint32_t x, uint32_t y, kv_f16x8 &even, kv_f16x8 &odd) {
  even = kv_decode8((x & 0x0f0f0f0fu) | ((y & 0x0f0f0f0fu) << 4));
  odd = kv_decode8(((x >> 4) & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u));
}

// Eight dimensions of a row's result, rotated back but for the signs, from `at` on: of the output's row `index`, or in the parts.
template <int D, int SPLIT>
__device__ __forceinline__ void kv_store8(const KvAttendArgs &a, int64_t index, int at, const uint32_t *signs, float *part_out, const float *y) {
  const uint2 sign = *reinterpret_cast<const uint2 *>(signs + at / 4);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(__float_as_uint(y[e]) ^ (((e < 4 ? sign.x : sign.y) << (24 - 8 * (e & 3))) & 0x80000000u));
  if (SPLIT == 2 || part_out != nullptr) {
    float *to = part_out != nullptr ? part_out + at : static_cast<float *>(a.out) + index * D + at;
    reinterpret_cast<float4 *>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = SPLIT == 1 ? f32_to_f16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_f16_bits(v[2 * e + 1])) << 16
                        : f32_to_bf16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16;
    }
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + index * D + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ float kv_share(float l, bool part) { return part ? 1.0f : l != 0.0f ? 1.0f / l : 0.0f; }  // (no key: zeros)
__device__ __forceinline__ float kv_lse(float ref, float l) { return l != 0.0f ? (ref + __builtin_amdgcn_logf(l)) * 0.693147180559945f : -INFINITY; }

// A row's result: rotated back, and stored as the output, or at its place in the parts.
template <int D, int SPLIT>
__device__ __forceinline__ void kv_finish(const KvAttendArgs &a, const KvRow &row, int g, const uint32_t *signs, float *part_out, float2 *part_stats,
                                          const KvState &st, const kv_f32x4 (&o)[D / 16]) {
  const float l = kv_over_groups(st.sum, kv_sum_of);
  const float by = kv_share(l, part_out != nullptr) * (1.0f / D);
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
#pragma unroll
  for (int j = 0; j < D / 32; ++j) kv_store8<D, SPLIT>(a, index, 32 * j + 8 * g, signs, part_out, y + 8 * j);
  if (g != 0) return;
  if (part_out != nullptr) *part_stats = make_float2(st.reference(), l);
  else if (a.lse != nullptr) a.lse[index] = kv_lse(st.ref, l);
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
template <bool WIDE>
__device__ __forceinline__ KvPages kv_pages_of(const KvAttendArgs &a, const int32_t *table, int n, int g, int step) {
  if constexpr (WIDE) {
    const int page = kv_scalar_page_at(a, table, step * 64);
    return {page, page};
  }
  return {kv_page_at(a, table, step * 64 + 16 * (n >> 2)), kv_page_at(a, table, step * 64 + 16 * g)};
}
// Where a step's keys begin, in tokens of the whole cache (all heads): of a lane's group of sixteen, or of the step.
template <bool WIDE>
__device__ __forceinline__ int64_t kv_tokens_at(const KvAttendArgs &a, int kv_head, int page, int step, int group) {
  const int shift = a.cache.page_shift;
  return (kv_block_of(a, page, kv_head) << shift) + ((step * 64 + (WIDE ? 0 : 16 * group)) & ((1 << shift) - 1));
}
template <int D, bool WIDE>
__device__ __forceinline__ void kv_request_keys(const KvAttendArgs &a, int kv_head, int n, int g, int s, const KvPages &page, KvRaw<D> &to) {
  constexpr int W = D / 32;
  const int64_t keys = kv_tokens_at<WIDE>(a, kv_head, page.k, s, n >> 2), scales = kv_tokens_at<WIDE>(a, kv_head, page.v, s, g);
  const uint32_t in_keys = ((WIDE ? 16 * (n >> 2) : 0) + (n & 3)) * (D / 8) + g * W;  // dwords
  const uint32_t *from = reinterpret_cast<const uint32_t *>(a.cache.k_codes) + keys * (D / 8);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (W == 2) {
      const uint2 v = *reinterpret_cast<const uint2 *>(from + in_keys + 4 * t * (D / 8));
      to.k[t][0] = v.x; to.k[t][1] = v.y;
    } else {
#pragma unroll
      for (int w = 0; w < W; w += 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(from + in_keys + 4 * t * (D / 8) + w);
        to.k[t][w] = v.x; to.k[t][w + 1] = v.y; to.k[t][w + 2] = v.z; to.k[t][w + 3] = v.w;
      }
    }
  }
  const uint32_t in_scales = WIDE ? 2 * g : 0;  // of eight
  const uint4 *k_from = reinterpret_cast<const uint4 *>(a.cache.k_scales + scales), *v_from = reinterpret_cast<const uint4 *>(a.cache.v_scales + scales);
  to.k_scale[0] = k_from[in_scales]; to.k_scale[1] = k_from[in_scales + 1];
  to.v_scale[0] = v_from[in_scales]; to.v_scale[1] = v_from[in_scales + 1];
  to.here = kv_page_there(a, page.v);
}
template <int D, bool WIDE>
__device__ __forceinline__ void kv_request_values(const KvAttendArgs &a, int kv_head, int n, int g, int s, const KvPages &page, KvRaw<D> &to) {
  const int shift = a.cache.page_shift;
  const int64_t block = kv_block_of(a, page.v, kv_head);
  const uint8_t *from = a.cache.v_codes + ((block * (D / 2)) << shift) + ((s * 64 + (WIDE ? 0 : 16 * g)) & ((1 << shift) - 1));
  const uint32_t in_values = (static_cast<uint32_t>(n) << shift) + (WIDE ? 16 * g : 0);
#pragma unroll
  for (int j = 0; j < D / 32; ++j) to.v[j] = *reinterpret_cast<const uint4 *>(from + (static_cast<uint32_t>(16 * j) << shift) + in_values);
}
template <int D, bool WIDE>
__device__ __forceinline__ void kv_request(const KvAttendArgs &a, int kv_head, int n, int g, int s, const KvPages &page, KvRaw<D> &to) {
  kv_request_keys<D, WIDE>(a, kv_head, n, g, s, page, to);
  kv_request_values<D, WIDE>(a, kv_head, n, g, s, page, to);
}

// ---- few rows ------------------------------------------------------------------------------------------------------
// Sixteen rows a workgroup; its four wavefronts take every fourth step of the part's keys and are joined through LDS (or one
// wavefront takes them all, where requests are short and many).  A step's
// keys, scales and values (8.4 KB at D = 128) are requested a step of the wavefront's ahead, into the registers of the ones just used.
// Long ones are bound by memory: 131101 tokens, 8 heads of 128, 138 MB in 26.9 us; 64 requests, 668 MB in 127 (least 122), 5.3 TB/s of the 6.3 that a
// read of nothing else reaches (vector instructions issue in half of the cycles, the matrix units are busy in 15 %).  Short ones by
// latency: 1003 tokens 8.9 us, three dependent loads (length, page, keys) and four steps a wavefront.  Eight wavefronts a workgroup: 9.3.
template <int D, int SPLIT, bool WIDE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, 2) void kv_attend_few_kernel(KvAttendArgs a) {
  constexpr int W = D / 32;  // dwords of codes that a lane has of a key, and matrix instructions along the dimensions
  constexpr int PITCH = D + 4;
  __shared__ __attribute__((aligned(16))) float join[WAVES][16][PITCH];
  __shared__ float refs[WAVES][16], sums[WAVES][16];
  __shared__ uint32_t signs[D / 4];
  if (threadIdx.x < D / 4) signs[threadIdx.x] = reinterpret_cast<const uint32_t *>(a.cache.signs)[threadIdx.x];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kv_head = blockIdx.x % a.cache.heads, group = blockIdx.x / a.cache.heads;

  KvPart part;
  if (WAVES == 1 || a.few.target == 0) {  // (one wavefront: of launches of few steps, which are not cut)
    part = {{}, group, 0, 1, 0};
    if (!kv_few_tile(a, group, part.rows)) return;
  } else if constexpr (WAVES > 1) {
    if (!kv_few_part<64 * WAVES>(a, a.few_requests * a.few_tiles, a.few, kv_head, group, part)) return;
  }
  const KvRows r = part.rows;
  const KvSpan span = kv_span_of(a, r, r.first, r.rows);
  const int steps = span.highest >= span.lowest ? kv_steps_of(span) : 0;
  int step = (span.lowest >> 6) + part.from(steps, part.index) + wave;
  const int end = (span.lowest >> 6) + part.from(steps, part.index + 1);

  const int32_t *table = a.table + r.request * a.table_stride;
  KvRaw<D> raw;
  KvPages next = {0, 0};
  const KvRow row = kv_row_of(a, r, kv_head, r.first + n, n < r.rows);
  kv_f16x8 q[W], q_rest[SPLIT > 0 ? W : 1];
  float factor;
  {
    // the first step is on its way while the queries are rotated (in heads of 256 there are no registers for both)
    KvQuery<D, SPLIT> query;
    query.request(a, row, g);
    const auto request = [&] {
      if (step < end) {
        kv_request<D, WIDE>(a, kv_head, n, g, step, kv_pages_of<WIDE>(a, table, n, g, step), raw);
        next = kv_pages_of<WIDE>(a, table, n, g, step + WAVES);
      }
    };
    if constexpr (D < 256) request();
    float y[D / 4];
    const int exponent = kv_query_exponent(query.rotate(row.token >= 0, y));
    factor = a.scale * (1.44269504088896f / D) * kv_power_of_two(exponent);
    kv_query_parts<D, SPLIT>(y, kv_power_of_two(-exponent), q, q_rest);
    if constexpr (D == 256) request();
  }

  KvState st;
  st.begin();
  kv_f32x4 o[D / 16];
#pragma unroll
  for (int j = 0; j < D / 16; ++j) o[j] = kv_f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // The last step is one of its own: a request that depends on whether there is a next step is one that the compiler cannot count, and it
  // then waits for all of them.
  const auto take_step = [&](auto more) {
    KvPages later = next;
    if constexpr (more) later = kv_pages_of<WIDE>(a, table, n, g, step + 2 * WAVES);  // (before what is requested next: loads come back in order)
    float x[16], vs[16];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      kv_f32x4 score = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const kv_f16x8 codes = kv_decode8(raw.k[k][c]);
        if constexpr (SPLIT > 0) score = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q_rest[c], score, 0, 0, 0);
        score = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, q[c], score, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * k + i] = score[i];
    }
    {
      const uint32_t kw[8] = {raw.k_scale[0].x, raw.k_scale[0].y, raw.k_scale[0].z, raw.k_scale[0].w, raw.k_scale[1].x, raw.k_scale[1].y, raw.k_scale[1].z, raw.k_scale[1].w};
      const uint32_t vw[8] = {raw.v_scale[0].x, raw.v_scale[0].y, raw.v_scale[0].z, raw.v_scale[0].w, raw.v_scale[1].x, raw.v_scale[1].y, raw.v_scale[1].z, raw.v_scale[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[2 * i] = fmaf(x[2 * i], __uint_as_float(kw[i] << 16) * factor, -st.ref);
        x[2 * i + 1] = fmaf(x[2 * i + 1], __uint_as_float(kw[i] & 0xffff0000u) * factor, -st.ref);
        vs[2 * i] = __uint_as_float(vw[i] << 16);
        vs[2 * i + 1] = __uint_as_float(vw[i] & 0xffff0000u);
      }
    }
    const bool here = raw.here;
    // The scales' registers are free now; left to itself the compiler takes others and moves them at the end of the step, which
    // is a wait for all that was just requested.
#pragma unroll
    for (int i = 0; i < 16; ++i) asm volatile("" : "+v"(x[i]), "+v"(vs[i])::"memory");
    if constexpr (more) kv_request_keys<D, WIDE>(a, kv_head, n, g, step + WAVES, next, raw);
    const int first = step * 64;
    if (first + 63 > span.all_high || first < span.all_low || __builtin_amdgcn_ballot_w64(!here) != 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = first + 16 * g + i;
        const bool seen = kv_seen(key, here && key <= r.last_key, row);
        x[i] = seen ? x[i] : -INFINITY;
        vs[i] = seen ? vs[i] : 0.0f;
      }
    }
    const int top = kv_largest_scale(vs);
    kv_keep_in_range<D>(x, vs, kv_exponent_of(top), [&] { return top - kv_smallest_scale(vs) >= kKvMixed << 23; }, st, o);
    kv_f16x8 p[2], p_rest[SPLIT > 1 ? 2 : 1];
    kv_weights<SPLIT>(x, vs, st.sum, p, p_rest);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint32_t w[4] = {raw.v[j].x, raw.v[j].y, raw.v[j].z, raw.v[j].w};
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
    if constexpr (more) kv_request_values<D, WIDE>(a, kv_head, n, g, step + WAVES, next, raw);
    next = later;
  };
  for (; step + WAVES < end; step += WAVES) take_step(std::true_type{});
  if (step < end) take_step(std::false_type{});
  st.ref = st.reference();

  // The wavefronts, in their order.  A lane has eight dimensions of a row now, as it has where vectors are written to the cache,
  // so that a row's sums and its rotation are many lanes' work: with four rows one wavefront's, eight values a lane instead of 32.
  const float own_sum = kv_over_groups(st.sum, kv_sum_of);
  if (n < r.rows) {
    if (g == 0) {
      refs[wave][n] = st.ref;
      sums[wave][n] = own_sum;
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {  // dimension 32 j + 8 g + 2 r + parity is in o[2 j + parity][r]
      float4 *to = reinterpret_cast<float4 *>(&join[wave][n][32 * j + 8 * g]);
      to[0] = make_float4(o[2 * j][0], o[2 * j + 1][0], o[2 * j][1], o[2 * j + 1][1]);
      to[1] = make_float4(o[2 * j][2], o[2 * j + 1][2], o[2 * j][3], o[2 * j + 1][3]);
    }
  }
  __syncthreads();
  const bool is_part = part.count > 1;
  const int dims = 8 * kv_part_of<D>(lane);
  for (int from = wave * (512 / D); from < r.rows; from += WAVES * (512 / D)) {
    const int at = from + kv_vector_of<D>(lane);
    const bool there = at < r.rows;
    float half[WAVES], both = kKvNothing, l = 0.0f, y[8];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      half[w] = there ? refs[w][at] : kKvNothing;
      both = fmaxf(both, half[w]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.0f;
    if (there) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        half[w] = kv_half_power(half[w] - both);
        const float of = half[w] * half[w];
        l = fmaf(sums[w][at] * half[w], half[w], l);
        const float4 u = *reinterpret_cast<const float4 *>(&join[w][at][dims]), v = *reinterpret_cast<const float4 *>(&join[w][at][dims + 4]);
        const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], of, y[e]);
      }
    }
    const float by = kv_share(l, is_part) * (1.0f / D);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= by;
    kv_butterflies<D>(y, lane);
    if (!there) continue;
    const KvRow of_row = kv_row_of(a, r, kv_head, r.first + at, true);
    const int64_t index = static_cast<int64_t>(of_row.token) * a.heads + of_row.head;
    const int64_t place = (static_cast<int64_t>(kv_head) * a.few.places + part.place) * 16 + at;
    kv_store8<D, SPLIT>(a, index, dims, signs, is_part ? a.few.out + place * D : nullptr, y);
    if (dims != 0) continue;
    if (is_part) a.few.stats[place] = make_float2(both, l);
    else if (a.lse != nullptr) a.lse[index] = kv_lse(both, l);
  }
}

// ---- many rows -----------------------------------------------------------------------------------------------------
// 128 rows a workgroup, 16 * RT a wavefront, all on the same keys.  Decoding a step costs as many vector instructions as the softmax
// of 32 rows: each wavefront decodes a part of it into LDS, in the order of the operands (conflict-free on both sides), for the next step while
// this one's products run; one barrier a step.
// Bound by instruction issue: 8192 tokens, 32 heads of 128 in bf16, 565 us, 0.97 PFLOP/s (a large product of the library: 1.21); vector
// instructions, eight a score and lane, take 56 % of the cycles, the matrix instructions 41 %, and on one SIMD these two do not overlap.
// Matrix instructions of 32 x 32 overlap in part but leave too few registers: 576 to 587 us.
template <int D>
constexpr int kv_many_waves() { return D == 256 ? 8 : 4; }
template <int D>
constexpr size_t kv_many_lds() { return 2 * (4 * (D / 32) * 64 * 16 + (D / 32) * 4 * 64 * 16 + 512); }

template <int D, int SPLIT, bool WIDE>
__global__ __launch_bounds__(64 * kv_many_waves<D>(), 2) void kv_attend_many_kernel(KvAttendArgs a) {
  constexpr int WAVES = kv_many_waves<D>(), RT = kKvManyRows / 16 / WAVES;
  constexpr int C = D / 32;
  constexpr int KD = D * 2 / (16 * WAVES), VD = KD;  // dwords of a step's keys and values that a lane decodes
  struct Step {
    kv_f16x8 k[4][C][64];         // [tile][dimensions][lane]
    kv_f16x8 v[D / 32][2][2][64]; // [dimensions][half of the keys][even, odd][lane]
    float ks[64], vs[64];         // times the scale of the scores; as it is
  };
  static_assert(2 * sizeof(Step) == kv_many_lds<D>(), "what the launch reserves");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ uint32_t signs[D / 4];
  __shared__ float own_factors[kKvManyRows];  // (of rows that do not share one; in registers they would be spilled)
  if (threadIdx.x < D / 4) signs[threadIdx.x] = reinterpret_cast<const uint32_t *>(a.cache.signs)[threadIdx.x];
  Step *steps = reinterpret_cast<Step *>(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int kv_head = blockIdx.x % a.cache.heads, group = blockIdx.x / a.cache.heads;

  KvPart part;
  if (a.many.target == 0) {
    part = {{}, a.many_tiles - 1 - group, 0, 1, 0};
    if (!kv_many_tile(a, part.tile, part.rows)) return;
  } else if (!kv_many_part<64 * WAVES>(a, kv_head, group, *reinterpret_cast<KvCounted *>(lds), part)) {
    return;
  }
  const KvRows r = part.rows;
  const KvSpan span = kv_span_of(a, r, r.first, r.rows);
  const int all_steps = span.highest >= span.lowest ? kv_steps_of(span) : 0;
  int step = (span.lowest >> 6) + part.from(all_steps, part.index);
  const int end = (span.lowest >> 6) + part.from(all_steps, part.index + 1);

  // what this wavefront decodes: keys of one tile, all or half of their dimensions; values of one j, both halves of the keys or one
  const int shift = a.cache.page_shift;
  const int32_t *table = a.table + r.request * a.table_stride;
  const int k_tile = WAVES == 8 ? wave >> 1 : wave, k_from = WAVES == 8 ? (wave & 1) * KD : 0;
  const int v_j = VD == 2 ? wave >> 1 : wave, v_from = VD == 2 ? wave & 1 : 0;
  const uint32_t in_keys = ((WIDE ? 16 * (n >> 2) : 0) + 4 * k_tile + (n & 3)) * (D / 8) + g * (D / 32) + k_from;  // dwords
  const uint32_t in_values = (static_cast<uint32_t>(16 * v_j + n) << shift) + (WIDE ? 16 * g : 0) + 8 * v_from, in_scales = WIDE ? lane : n;
  uint32_t k_raw[KD], v_raw[VD], scale_raw = 0;
  const auto load = [&](int s, const KvPages &page) {
    const int64_t keys = kv_tokens_at<WIDE>(a, kv_head, page.k, s, n >> 2), scales = kv_tokens_at<WIDE>(a, kv_head, page.v, s, g);
    const uint32_t *k_at = reinterpret_cast<const uint32_t *>(a.cache.k_codes) + keys * (D / 8);
    const uint8_t *v_at = a.cache.v_codes + ((kv_block_of(a, page.v, kv_head) * (D / 2)) << shift) + ((s * 64 + (WIDE ? 0 : 16 * g)) & ((1 << shift) - 1));
    if constexpr (KD == 2) {
      const uint2 k = *reinterpret_cast<const uint2 *>(k_at + in_keys), v = *reinterpret_cast<const uint2 *>(v_at + in_values);
      k_raw[0] = k.x; k_raw[1] = k.y; v_raw[0] = v.x; v_raw[1] = v.y;
    } else {
      const uint4 k = *reinterpret_cast<const uint4 *>(k_at + in_keys), v = *reinterpret_cast<const uint4 *>(v_at + in_values);
      k_raw[0] = k.x; k_raw[1] = k.y; k_raw[2] = k.z; k_raw[3] = k.w; v_raw[0] = v.x; v_raw[1] = v.y; v_raw[2] = v.z; v_raw[3] = v.w;
    }
    if (wave < 2) scale_raw = ((wave == 0 ? a.cache.k_scales : a.cache.v_scales) + scales)[in_scales];
  };
  KvRow row[RT];
  KvQuery<D, SPLIT> query[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int at = (wave * RT + t) * 16 + n;
    row[t] = kv_row_of(a, r, kv_head, r.first + at, at < r.rows);
    query[t].request(a, row[t], g);
  }
  KvPages page = {0, 0}, next = page, later = page;  // of the step that is computed (whether its keys are there), of the one requested, and of the one after it
  if (step < end) {
    page = kv_pages_of<WIDE>(a, table, n, g, step);
    next = kv_pages_of<WIDE>(a, table, n, g, step + 1);
    load(step, page);
  }

  // One power of two for the workgroup's rows, whose factor goes into the keys' scales once a step; where rows are further apart than the format
  // holds, each has its own, which multiplies its scores: a product more of each, so that is a loop of its own.  (The other one keeps its time: a
  // prompt of 8192 566 us with and without; with one loop gone through again for each class of sizes 608.)
  kv_f16x8 q[RT][C], q_rest[RT][SPLIT > 0 ? C : 1];
  float factor;
  bool apart;
  {
    constexpr short NONE = -1000;
    float y[RT][D / 4];
    int own[RT];
    kv_i16x2 reach = {NONE, NONE};  // the largest exponent, and what the smallest lacks to 0
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float own_top = query[t].rotate(row[t].token >= 0, y[t]);
      own[t] = kv_query_exponent(own_top);
      const short e = static_cast<short>(own[t]);
      if (own_top > 0.0f && own_top < INFINITY) reach = __builtin_elementwise_max(reach, kv_i16x2{e, static_cast<short>(-e)});  // (a broken row is its own affair, zeros have any exponent)
    }
    reach = kv_row_max(reach);
    kv_i16x2 *reaches = reinterpret_cast<kv_i16x2 *>(steps[1].ks);  // (the first step decodes into steps[0])
    if (lane == 0) reaches[wave] = reach;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) reach = __builtin_elementwise_max(reach, reaches[w]);
    const int exponent = kv_uniform(reach[0] != NONE ? reach[0] : 0);
    apart = kv_uniform(reach[0] + reach[1]) > kv_query_spread<SPLIT>();
    factor = a.scale * (1.44269504088896f / D) * (apart ? 1.0f : kv_power_of_two(exponent));
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int of_row = apart ? own[t] : exponent;
      if (apart && g == 0) own_factors[(wave * RT + t) * 16 + n] = kv_power_of_two(of_row);  // (read behind the loop's first barrier)
      kv_query_parts<D, SPLIT>(y[t], kv_power_of_two(-of_row), q[t], q_rest[t]);
    }
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
    if (step + 1 < end) load(step + 1, next);
    later = kv_pages_of<WIDE>(a, table, n, g, step + 2);
  }
  KvBroken broken;
  broken.begin();
  const auto walk = [&](auto each) __attribute__((always_inline)) {
    for (int now = 0; step < end; ++step, now ^= 1) {
      __syncthreads();  // this step is decoded, and nobody reads the one before it any more
      const Step &from = steps[now];
      const bool here = kv_page_there(a, page.v);
      if (step + 1 < end) {
        decode(steps[now ^ 1]);
        if (step + 2 < end) load(step + 2, later);
      }
      page = next;
      next = later;
      later = kv_pages_of<WIDE>(a, table, n, g, step + 3);
      const int first = step * 64;
      if (wave_rows <= 0 || first > own.highest || first + 63 < own.lowest) continue;

      float own_factor[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) own_factor[t] = each ? own_factors[(wave * RT + t) * 16 + n] : 1.0f;
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
          for (int t = 0; t < RT; ++t) x[t][4 * k + i] = fmaf(s[t][i], each ? ks[i] * own_factor[t] : ks[i], -st[t].ref);
        }
      }
      if (first + 63 > own.all_high || first < own.all_low || __builtin_amdgcn_ballot_w64(!here) != 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = first + 16 * g + i;
          const bool there = here && key <= r.last_key;
#pragma unroll
          for (int t = 0; t < RT; ++t) x[t][i] = kv_seen(key, there, row[t]) ? x[t][i] : -INFINITY;
          vs[i] = there ? vs[i] : i > 0 ? vs[0] : 0.0f;
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (all masks at once are more than there are scalar registers)
        }
        broken.look(vs, step);
      }
      const float top_exponent = kv_exponent_of(kv_largest_scale(vs));
      const auto mixed = [&] {  // (a lane for each key, against the first, which is the smaller one if one is)
        int key = lane;
        asm volatile("" : "+v"(key));
        const int scale = __float_as_int(from.vs[key]);
        return static_cast<uint32_t>(scale - kv_uniform(scale) + (2 << 23)) >= static_cast<uint32_t>(kKvMixed) << 23;
      };
      kv_f16x8 p[RT][2], p_rest[RT][SPLIT > 1 ? 2 : 1];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        kv_keep_in_range<D>(x[t], vs, top_exponent, mixed, st[t], o[t]);
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
  };
  if (apart) walk(std::true_type{});
  else walk(std::false_type{});
  if (broken.to >= 0) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const float nan = broken.of(a, table, r.last_key, row[t], kv_head, g);
#pragma unroll
      for (int j = 0; j < D / 16; ++j) o[t][j] += nan;
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int64_t place = (static_cast<int64_t>(kv_head) * a.many.places + part.place) * kKvManyRows + (wave * RT + t) * 16 + n;
    kv_finish<D, SPLIT>(a, row[t], g, signs, part.count > 1 ? a.many.out + place * D : nullptr, a.many.stats + place, st[t], o[t]);
  }
}

template <int D, int SPLIT, bool WIDE>
bool kv_attend_launch(const KvAttendArgs &a, hipStream_t stream) {
  const unsigned heads = static_cast<unsigned>(a.cache.heads);
  if (a.many_tiles > 0) {
    const auto kernel = kv_attend_many_kernel<D, SPLIT, WIDE>;
    if (!reserve_dynamic_lds(reinterpret_cast<const void *>(kernel), kv_many_lds<D>())) return false;
    launch_kernel(kernel, dim3(heads * (a.many.target != 0 ? a.many.target : a.many_tiles)), dim3(64 * kv_many_waves<D>()), kv_many_lds<D>(), stream, a);
  }
  if (a.few_requests > 0) {
    const dim3 grid(heads * (a.few.target + a.few_requests * a.few_tiles));
    if (a.few_alone) launch_kernel(kv_attend_few_kernel<D, SPLIT, WIDE, 1>, grid, dim3(64), 0, stream, a);
    else launch_kernel(kv_attend_few_kernel<D, SPLIT, WIDE, 4>, grid, dim3(256), 0, stream, a);
  }
  return true;
}

template <int D>
bool kv_attend_of(const KvAttendArgs &a, int split, hipStream_t stream) {
  if (a.cache.page_shift >= 6)
    return split == 0 ? kv_attend_launch<D, 0, true>(a, stream) : split == 1 ? kv_attend_launch<D, 1, true>(a, stream) : kv_attend_launch<D, 2, true>(a, stream);
  return split == 0 ? kv_attend_launch<D, 0, false>(a, stream) : split == 1 ? kv_attend_launch<D, 1, false>(a, stream) : kv_attend_launch<D, 2, false>(a, stream);
}

}  // namespace oq
