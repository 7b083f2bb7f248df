// Around the 4-bit key/value cache: pages and slots for new tokens, keys and values into it, and back out of it.
// (No counterpart in the reference, which has no cache.)
#include "kv_cache.h"
#include "kv_rows.h"

namespace oq {
namespace {

// ---- pages and slots ---------------------------------------------------------------------------------------------
// Request r holds before[r] tokens in have = ceil(before / page) pages and gets new[r] more: fresh = ceil((before + new) /
// page) - have pages, taken from the free list in request order.  Everything follows from two running sums over the
// requests (new tokens, fresh pages), which every workgroup makes for itself in LDS: a few thousand requests are some KB, and one launch
// without a grid-wide wait is what a call of some microseconds can afford.  A thread sums a run of requests, the threads' sums are
// summed by lane shifts and one barrier; a token finds its request by bisection, four tokens of a thread side by side.
// Nothing that one workgroup writes is read by another: the page of a new token is in the old part of the table or in the free list.
// Bound by latency: one request 2.2 us (the launch), 509 requests with 71 thousand new tokens 7.1 us, three memory round trips.
constexpr int kAssignThreads = 256, kAssignTokens = 4;  // tokens a thread

__device__ __forceinline__ int last_not_above(const int *sums, int count, int value) {  // largest r with sums[r] <= value
  int low = 0, high = count;  // sums[0] = 0 <= value
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (sums[mid] <= value) low = mid; else high = mid;
  }
  return low;
}

__device__ __forceinline__ int pages_of(int tokens, int page_shift) { return static_cast<int>((static_cast<uint32_t>(tokens) + (1u << page_shift) - 1) >> page_shift); }

__global__ __launch_bounds__(kAssignThreads) void kv_assign_kernel(KvAssignArgs a) {
  extern __shared__ int lds[];
  __shared__ int2 wave_sum[kAssignThreads / 64];
  int *starts = lds, *upto = lds + a.requests + 1, *before = lds + 2 * (a.requests + 1);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int page = 1 << a.page_shift;
  const int taken = max(*a.taken, 0);
  const int run = (a.requests + kAssignThreads - 1) / kAssignThreads, from = min(tid * run, a.requests), to = min(from + run, a.requests);
  int2 own = make_int2(0, 0);  // new tokens, fresh pages
  for (int r = from; r < to; ++r) {
    const int was = max(a.lengths[r], 0), more = max(a.new_lengths[r], 0);
    before[r] = was;
    starts[r] = more;  // (the thread's own until it writes the sum there)
    own.x += more;
    own.y += pages_of(was + more, a.page_shift) - pages_of(was, a.page_shift);
  }
  const int2 sum = make_int2(kv_sums(own.x), kv_sums(own.y));
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();
  int2 ahead = make_int2(sum.x - own.x, sum.y - own.y), carry = make_int2(0, 0);
#pragma unroll
  for (int w = 0; w < kAssignThreads / 64; ++w) {
    if (w < wave) {
      ahead.x += wave_sum[w].x;
      ahead.y += wave_sum[w].y;
    }
    carry.x += wave_sum[w].x;
    carry.y += wave_sum[w].y;
  }
  for (int r = from; r < to; ++r) {
    const int was = before[r], more = starts[r];
    starts[r] = ahead.x;
    upto[r] = ahead.y;
    if (blockIdx.x == 0) {
      a.starts[r] = ahead.x;
      a.lengths_after[r] = was + more;
    }
    ahead.x += more;
    ahead.y += pages_of(was + more, a.page_shift) - pages_of(was, a.page_shift);
  }
  const int total = carry.x, total_fresh = carry.y;
  if (tid == 0) {
    starts[a.requests] = total;
    upto[a.requests] = total_fresh;
    if (blockIdx.x == 0) {
      a.starts[a.requests] = total;
      *a.taken_after = static_cast<int>(min(static_cast<int64_t>(taken) + total_fresh, static_cast<int64_t>(a.free_count)));
    }
  }
  __syncthreads();
  const auto free_page = [&](int64_t index) { return index < a.free_count ? a.free_pages[index] : -1; };
  const int64_t own_fresh = static_cast<int64_t>(blockIdx.x) * kAssignThreads + tid;
  const int own_page = own_fresh < total_fresh ? free_page(taken + own_fresh) : 0;  // (on its way while the tokens are looked up)
  int low[kAssignTokens] = {};
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kAssignTokens * kAssignThreads + tid;
  for (int span = a.requests; span > 1; span = (span + 1) >> 1) {  // the last request that does not begin behind the token, among span from low on
    const int half = (span + 1) >> 1;
#pragma unroll
    for (int i = 0; i < kAssignTokens; ++i) {
      const int mid = low[i] + half;
      if (mid < a.requests && starts[mid] <= first + i * kAssignThreads) low[i] = mid;
    }
  }
#pragma unroll
  for (int i = 0; i < kAssignTokens; ++i) {
    const int64_t t = first + i * kAssignThreads;
    if (t >= a.tokens) break;
    int64_t slot = -1;
    int position = -1;
    if (t < total) {
      const int r = low[i];
      position = before[r] + static_cast<int>(t) - starts[r];
      const int column = position >> a.page_shift, have = (before[r] + page - 1) >> a.page_shift;
      int at = -1;
      if (column < a.table_width) at = column < have ? a.table[r * a.table_stride + column] : free_page(static_cast<int64_t>(taken) + upto[r] + column - have);
      if (at >= 0) slot = (static_cast<int64_t>(at) << a.page_shift) + (position & (page - 1));
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
  for (int64_t f = own_fresh; f < total_fresh; f += static_cast<int64_t>(gridDim.x) * kAssignThreads) {
    const int r = last_not_above(upto, a.requests, static_cast<int>(f));
    const int column = ((before[r] + page - 1) >> a.page_shift) + static_cast<int>(f) - upto[r];
    if (column < a.table_width) a.table[r * a.table_stride + column] = f == own_fresh ? own_page : free_page(taken + f);
  }
}

// ---- into the cache and back -----------------------------------------------------------------------------------------
// A workgroup takes one head of sixteen tokens, keys and values all requested at once.  A token's key is D / 2 bytes in a row, but its
// value is spread over the page, one byte in each of D / 2 rows: the bytes of the sixteen tokens change places in LDS, and four tokens
// whose slots follow each other in a page (a prompt's, nearly always) are one dword of a row.  MI355X, 8192 tokens of 8 heads of 128 in
// bf16 (42 MB): write 16 us, read 16 (with 64 tokens a workgroup 37 together, with one byte a store and lanes exchanged through LDS 52).
// Bound by vector instructions, 23 and 25 a value, which issue in 78 and 92 % of the cycles: ten and eleven of them the seven stages of the
// transform; the bytes alone take 9.  On the way in the order of the sums decides codes.  On the way out it does not: a scale times a code is a
// multiple of half the scale's last bit, and so is every partial sum, which stays below 2^20 of it and is exact in fp32 in any order.

// On the way out, where the slots are waited for, as they are.
__device__ __forceinline__ void group_slots(int64_t (&slots)[kKvGroup], const int64_t *from, int64_t first, int64_t tokens, int64_t most) {
  if (threadIdx.x < kKvGroup) {
    int64_t slot = -1;
    if (first + threadIdx.x < tokens) slot = from[first + threadIdx.x];
    slots[threadIdx.x] = slot < most ? slot : -1;
  }
}

// Values of a lane: sixteen on the way in, where a vector's scale is found once for twice as many of them and one stage fewer lies between lanes
// (write 18.1 -> 16.2 us), eight on the way out (sixteen 16.3 -> 16.8).
constexpr int kKvWriteEach = 16;

template <int D, int DT>
__global__ __launch_bounds__(kv_write_threads(D)) void kv_write_kernel(KvWriteArgs a) {
  constexpr int E = kKvWriteEach, THREADS = kv_write_threads(D);
  constexpr int AT_ONCE = THREADS * E / D;         // vectors that the workgroup's lanes hold
  constexpr int PASSES = 2 * kKvGroup / AT_ONCE;   // keys, then values
  __shared__ KvPlace places[kKvGroup];
  __shared__ uint32_t bytes[kKvGroup][D / 8 + 1];  // of the values
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = kv_part_of<D, E>(lane);
  const int head = blockIdx.x % a.cache.heads;
  const int64_t first = static_cast<int64_t>(blockIdx.x / a.cache.heads) * kKvGroup;
  const int shift = a.cache.page_shift;
  float y[PASSES][E];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int vector = p * AT_ONCE + wave * (64 * E / D) + kv_vector_of<D, E>(lane);
    const int64_t token = min(first + (vector & (kKvGroup - 1)), a.tokens - 1);
#pragma unroll
    for (int i = 0; i < E; i += 8) {
      if (vector >= kKvGroup) load8<DT>(a.v, token * a.v_token_stride + head * a.v_head_stride + E * part + i, a.v_wide, y[p] + i);
      else load8<DT>(a.k, token * a.k_token_stride + head * a.k_head_stride + E * part + i, a.k_wide, y[p] + i);
    }
  }
  const uint4 signs = reinterpret_cast<const uint4 *>(a.cache.signs)[part];
  const uint32_t words[4] = {signs.x, signs.y, signs.z, signs.w};
  group_places<D>(places, a.cache, a.slots, first, a.tokens, head);
  __syncthreads();
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int vector = p * AT_ONCE + wave * (64 * E / D) + kv_vector_of<D, E>(lane), token = vector & (kKvGroup - 1);
    times_signs(y[p], words);
    kv_butterflies<D>(y[p], lane);
    uint16_t scale;
    uint32_t codes[E / 8];
    kv_encode<D>(y[p], scale, codes);
    const bool there = places[token].slot >= 0;
    const int64_t at = places[token].key;
    if (vector >= kKvGroup) {
#pragma unroll
      for (int w = 0; w < E / 8; ++w) bytes[token][E / 8 * part + w] = codes[w];
      if (there && part == 0) a.cache.v_scales[at] = scale;
    } else if (there) {
      reinterpret_cast<uint2 *>(a.cache.k_codes)[at * (D / E) + part] = make_uint2(codes[0], codes[1]);
      if (part == 0) a.cache.k_scales[at] = scale;
    }
  }
  __syncthreads();
  store_values<D, THREADS>(a.cache, places, bytes);
}

template <int D, int DT>
__global__ __launch_bounds__(kv_read_threads(D)) void kv_read_kernel(KvReadArgs a) {
  constexpr int AT_ONCE = 2048 / D, PASSES = 2 * kKvGroup / AT_ONCE;
  constexpr int ROWS = (D / 2) * (kKvGroup / 4);   // dwords of the values, turned by LDS
  __shared__ int64_t slots[kKvGroup];
  __shared__ uint32_t bytes[kKvGroup][D / 8 + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = kv_part_of<D>(lane);
  const int head = blockIdx.x % a.cache.heads;
  const int64_t first = static_cast<int64_t>(blockIdx.x / a.cache.heads) * kKvGroup;
  const int shift = a.cache.page_shift;
  const uint2 signs = reinterpret_cast<const uint2 *>(a.cache.signs)[part];
  const uint32_t words[2] = {signs.x, signs.y};
  group_slots(slots, a.slots, first, a.tokens, a.cache.pages << shift);
  __syncthreads();
  uint32_t keys[PASSES];
  float scales[PASSES];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int vector = p * AT_ONCE + wave * (AT_ONCE / 4) + kv_vector_of<D>(lane);
    const int64_t slot = slots[vector & (kKvGroup - 1)];
    const int64_t at = ((((slot >> shift) * a.cache.heads + head) << shift) + (slot & ((1 << shift) - 1)));
    keys[p] = 0;
    scales[p] = 0.0f;
    if (slot >= 0) {
      if (vector < kKvGroup) keys[p] = reinterpret_cast<const uint32_t *>(a.cache.k_codes)[at * (D / 8) + part];
      scales[p] = bf16_bits_to_f32((vector < kKvGroup ? a.cache.k_scales : a.cache.v_scales)[at]);
    }
  }
  for (int i = threadIdx.x; i < ROWS; i += 256) {
    const int row = i / (kKvGroup / 4), t = i % (kKvGroup / 4) * 4;
    const auto place = [&](int64_t slot) { return a.cache.v_codes + ((((slot >> shift) * a.cache.heads + head) * (D / 2) + row) << shift) + (slot & ((1 << shift) - 1)); };
    uint32_t word = 0;
    if (in_a_row(slots + t, shift)) {
      __builtin_memcpy(&word, place(slots[t]), 4);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (slots[t + k] >= 0) word |= static_cast<uint32_t>(*place(slots[t + k])) << (8 * k);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) reinterpret_cast<uint8_t *>(bytes[t + k])[row] = static_cast<uint8_t>(word >> (8 * k));
  }
  __syncthreads();
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int vector = p * AT_ONCE + wave * (AT_ONCE / 4) + kv_vector_of<D>(lane), token = vector & (kKvGroup - 1);
    const kv_f16x8 c = kv_decode8(vector < kKvGroup ? keys[p] : bytes[token][part]);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = static_cast<float>(c[i]) * scales[p];
    kv_butterflies<D>(y, lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= 1.0f / D;
    times_signs(y, words);
    if (first + token < a.tokens) store8<DT>(vector < kKvGroup ? a.k : a.v, ((first + token) * a.cache.heads + head) * D + 8 * part, y);
  }
}

template <template <int, int> class Run, typename Args>
int by_type(const Args &a, int dim, int dtype, hipStream_t stream) {
  const auto with = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (dtype == OQ_F32) Run<D, OQ_F32>::go(a, stream);
    else if (dtype == OQ_F16) Run<D, OQ_F16>::go(a, stream);
    else Run<D, OQ_BF16>::go(a, stream);
  };
  if (dim == 64) with(std::integral_constant<int, 64>{});
  else if (dim == 128) with(std::integral_constant<int, 128>{});
  else with(std::integral_constant<int, 256>{});
  return OQ_OK;
}

inline dim3 group_grid(int64_t tokens, int heads) { return dim3(static_cast<unsigned>((tokens + kKvGroup - 1) / kKvGroup * heads)); }
template <int D, int DT>
struct RunWrite {
  static void go(const KvWriteArgs &a, hipStream_t s) { launch_kernel(kv_write_kernel<D, DT>, group_grid(a.tokens, a.cache.heads), dim3(kv_write_threads(D)), 0, s, a); }
};
template <int D, int DT>
struct RunRead {
  static void go(const KvReadArgs &a, hipStream_t s) { launch_kernel(kv_read_kernel<D, DT>, group_grid(a.tokens, a.cache.heads), dim3(kv_read_threads(D)), 0, s, a); }
};

}  // namespace

int kv_assign_dispatch(const KvAssignArgs &a, hipStream_t stream) {
  const size_t lds = sizeof(int) * (3 * static_cast<size_t>(a.requests) + 2);
  if (!reserve_dynamic_lds(reinterpret_cast<const void *>(kv_assign_kernel), lds))
    return fail(OQ_ERR_LAUNCH, "kv_assign: no LDS for %d requests", a.requests);
  constexpr int64_t per_block = kAssignThreads * kAssignTokens;
  const int64_t blocks = (a.tokens + per_block - 1) / per_block;
  launch_kernel(kv_assign_kernel, dim3(static_cast<unsigned>(blocks > 1 ? blocks : 1)), dim3(kAssignThreads), lds, stream, a);
  return check_launch("kv_assign");
}

int kv_write_dispatch(const KvWriteArgs &a, int dim, int dtype, hipStream_t stream) {
  by_type<RunWrite>(a, dim, dtype, stream);
  return check_launch("kv_write");
}

int kv_read_dispatch(const KvReadArgs &a, int dim, int dtype, hipStream_t stream) {
  by_type<RunRead>(a, dim, dtype, stream);
  return check_launch("kv_read");
}

}  // namespace oq
