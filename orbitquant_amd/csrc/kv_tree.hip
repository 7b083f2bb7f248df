// Trees of drafted tokens over the 4-bit cache: positions and masks before the step, the accepted path after it.
// (No counterpart in the reference, which has no cache.)
#include "kv_tree.h"

namespace oq {
namespace {

__device__ __forceinline__ int start_of(const int32_t *starts, int64_t tokens, int r) { return static_cast<int>(min(static_cast<int64_t>(max(starts[r], 0)), tokens)); }

// ---- positions and masks ----------------------------------------------------------------------------------------------
// Token i of a request's new ones hangs on parents[i] < i, or on what the request has cached already.  mask_i = bit i | mask_parent: every
// token takes in what its ancestor has gathered and moves on to that one's ancestor, so that a path of 2^n tokens is whole after n
// rounds.  Its depth is the number of its bits.  A workgroup a request, a thread a token; the last one has the tokens of no request.
// Bound by latency: three loads one behind the other, and log2(nodes) rounds in LDS: one tree of 26 nodes 1.7 us, which is a launch, 64 of up to 250 3.7.
template <int WORDS>
__global__ __launch_bounds__(64 * WORDS) void kv_tree_kernel(KvTreeArgs a) {
  __shared__ uint64_t masks[2][64 * WORDS][WORDS];  // (a round writes one and reads it, the next the other: one barrier a round)
  __shared__ int up[2][64 * WORDS];
  const int r = blockIdx.x, i = threadIdx.x;
  const int first = start_of(a.starts, a.tokens, r);
  if (r == a.requests) {
    for (int64_t t = first + i; t < a.tokens; t += 64 * WORDS) {
      a.positions[t] = -1;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) a.masks[t * WORDS + w] = 0;
    }
    return;
  }
  const int count = max(start_of(a.starts, a.tokens, r + 1) - first, 0);
  const int before = max(a.lengths[r], 0) - count;
  if (count > 64 * WORDS) {  // more than there are bits: a prompt, one token behind the other
    for (int t = i; t < count; t += 64 * WORDS) {
      a.positions[first + t] = before + t;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) a.masks[(static_cast<int64_t>(first) + t) * WORDS + w] = 0;
    }
    return;
  }
  uint64_t mask[WORDS];
#pragma unroll
  for (int w = 0; w < WORDS; ++w) mask[w] = i >> 6 == w ? 1ull << (i & 63) : 0;
  int ancestor = i < count ? a.parents[first + i] : -1;
  if (ancestor >= i) ancestor = -1;
  for (int reach = 1, now = 0; reach < count; reach *= 2, now ^= 1) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) masks[now][i][w] = mask[w];
    up[now][i] = ancestor;
    __syncthreads();
    if (ancestor >= 0) {
#pragma unroll
      for (int w = 0; w < WORDS; ++w) mask[w] |= masks[now][ancestor][w];
      ancestor = up[now][ancestor];
    }
  }
  if (i >= count) return;
  int depth = 0;
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    depth += __popcll(mask[w]);
    a.masks[(static_cast<int64_t>(first) + i) * WORDS + w] = mask[w];
  }
  a.positions[first + i] = before + depth - 1;
}

// ---- the accepted path -----------------------------------------------------------------------------------------------
// kept[r] names tokens of request r's new ones in rising order; the i-th becomes its i-th new token, and the others are forgotten.
// A list that begins with OQ_KV_KEEP_ALL is a request that stays as the step left it.  Another ends at its first entry that does not rise, is none of the request's tokens, has no slot, or would go where there is none.
//
// One launch for all layers.  A wavefront takes one head of one request in one cache.  A lane has the same bytes of all
// entries: a dword of the keys, a row of the values (two of heads of 256), a scale.  So whatever an entry moves onto, its lane has read before:
// the places rise with the list and are never behind their sources, and of a batch all are read before the first is written.
// The bytes are few (132 an entry at D = 128): bound by the latency of four loads one behind the other (starts, list, slots, entries), 5.2 us for one request and two
// layers, and by the lines that values lie on.  A page's rows of one byte a token are 16, 64 or 128 bytes apart, so an entry's 64 bytes of values are on 8, 32 or 64 lines of 128, read and
// written: 64 requests, eight layers of eight heads, three entries that move, 7.5, 12.2 and 18.8 us, and with the same lists of entries that stay where they are 4.1, 3.7 and 3.7 (empty
// lists 3.6, 3.2, 3.2): the chain that every wavefront walks for itself is four of these microseconds, the rest the lines, 0.2 for each.
// The counts are one workgroup's, a thread for a run of requests, four or more lists one behind the other from a thousand on: 256 requests 5.2 us, 1024 14.7, 8192 137.
constexpr int kKeepThreads = 256, kKeepBatch = 8;

struct Path {
  int first, fresh;
};
__device__ __forceinline__ Path path_of(const KvKeepArgs &a, int r) {
  const int first = start_of(a.starts, a.tokens, r);
  return {first, max(start_of(a.starts, a.tokens, r + 1) - first, 0)};
}
__device__ __forceinline__ int64_t slot_at(const KvKeepArgs &a, int64_t token) {
  const int64_t slot = a.slots[token];
  return slot < a.pages << a.page_shift ? slot : -1;
}

// A request of which everything stays (a prompt beside trees, say, longer than any list).
__device__ __forceinline__ bool all_stay(const KvKeepArgs &a, int r) { return a.most > 0 && a.kept[static_cast<int64_t>(r) * a.most] == OQ_KV_KEEP_ALL; }

// How many entries of a request's list count.  Eight at a time, whose loads do not wait for each other.
__device__ __forceinline__ int kept_of(const KvKeepArgs &a, int r, const Path &path) {
  int last = -1;
  for (int base = 0; base < a.most; base += kKeepBatch) {
    int k[kKeepBatch];
    int64_t slot[kKeepBatch], place[kKeepBatch];
#pragma unroll
    for (int b = 0; b < kKeepBatch; ++b) k[b] = base + b < a.most ? a.kept[static_cast<int64_t>(r) * a.most + base + b] : -1;
#pragma unroll
    for (int b = 0; b < kKeepBatch; ++b) slot[b] = k[b] >= 0 && k[b] < path.fresh ? slot_at(a, static_cast<int64_t>(path.first) + k[b]) : -1;
#pragma unroll
    for (int b = 0; b < kKeepBatch; ++b) place[b] = k[b] > base + b && k[b] < path.fresh ? slot_at(a, static_cast<int64_t>(path.first) + base + b) : 0;  // (of what moves)
#pragma unroll
    for (int b = 0; b < kKeepBatch; ++b) {
      if (k[b] <= last || slot[b] < 0 || place[b] < 0) return base + b;
      last = k[b];
    }
  }
  return a.most;
}

// The pages that kv_assign has drawn for a request's new tokens: for columns [have, need), also where these lie behind the table, which go back from `dropped` on.
struct Fresh {
  int have, need, dropped;
};
__device__ __forceinline__ Fresh fresh_of(const KvKeepArgs &a, int length, int fresh, bool all) {
  const auto pages_of = [&](int tokens) { return static_cast<int>((static_cast<uint32_t>(tokens) + (1u << a.page_shift) - 1) >> a.page_shift); };
  const int have = pages_of(max(length - fresh, 0)), need = pages_of(length);
  return {have, need, all ? need : max(have, a.table_width)};
}
__device__ __forceinline__ Fresh fresh_of(const KvKeepArgs &a, int r) { return fresh_of(a, max(a.lengths[r], 0), path_of(a, r).fresh, all_stay(a, r)); }

// Before every thread of the workgroup's `own`, the sum of the threads before; upto[kKeepThreads]: of all.  Behind a barrier, and one behind it.
__device__ void upto_of(int own, int (&upto)[kKeepThreads + 1]) {
  __shared__ int wave_sums[kKeepThreads / 64];
  const int tid = threadIdx.x, wave = tid >> 6, sum = kv_sums(own);
  if ((tid & 63) == 63) wave_sums[wave] = sum;
  __syncthreads();
  int ahead = sum - own;
#pragma unroll
  for (int w = 0; w < kKeepThreads / 64; ++w) ahead += w < wave ? wave_sums[w] : 0;
  upto[tid] = ahead;
  if (tid == kKeepThreads - 1) upto[kKeepThreads] = ahead + own;
  __syncthreads();
}

// Pages for columns that the table does not have: kv_assign has drawn them too, and no row names them.  But the step's pages are the last of the list before `taken`, in
// request order, so that they are found there: moved up to the end of what is taken, their number is the result.  Where the step's first page is:
//   - a column that got one (the first such) names it, and its place in the list tells;
//   - where no column has got one, `taken` less the step's pages, unless the list may have run out (then some were not drawn, and which is not known).
// Neither is believed where the call has but a part of kv_assign's requests, whose pages are not the list's last: the pages are lost then, never listed twice.
// A rare path, at the end of a request's row: latency of a few loads and barriers, 64 requests that are all there 3.8 us, where none is 3.4; elsewhere one comparison a request.
__device__ int keep_dropped(const KvKeepArgs &a, int taken) {
  __shared__ int fresh_upto[kKeepThreads + 1], dropped_upto[kKeepThreads + 1];
  __shared__ int anchor, anchor_page, found, others, elsewhere;  // (each written between two barriers alone)
  constexpr int kNone = 0x7fffffff;
  const int tid = threadIdx.x, run = (a.requests + kKeepThreads - 1) / kKeepThreads;
  const auto first_of = [&](int thread) { return min(thread * run, a.requests); };
  const int from = first_of(tid), to = first_of(tid + 1);
  if (tid == 0) {
    anchor = kNone;
    found = -1;
    others = 0;
    elsewhere = 0;
  }
  int own = 0;
  for (int r = from; r < to; ++r) {
    const Fresh f = fresh_of(a, r);
    own += f.need - f.have;
  }
  upto_of(own, fresh_upto);
  const int total = fresh_upto[kKeepThreads];
  int named = kNone, page = -1, index = fresh_upto[tid];
  for (int r = from; r < to && named == kNone; ++r) {
    const Fresh f = fresh_of(a, r);
    for (int column = f.have; column < min(f.need, a.table_width) && named == kNone; ++column) {
      page = a.table[r * a.table_stride + column];
      if (page >= 0) named = index + column - f.have;
    }
    index += f.need - f.have;
  }
  if (named != kNone) atomicMin(&anchor, named);
  __syncthreads();
  if (named != kNone && named == anchor) anchor_page = page;
  __syncthreads();
  const int last = start_of(a.starts, a.tokens, a.requests);
  if (anchor != kNone) {
    for (int i = max(taken - total, 0) + tid; i < taken; i += kKeepThreads) {
      if (a.free_pages[i] == anchor_page) atomicMax(&found, i);
    }
  } else {
    for (int64_t t = static_cast<int64_t>(last) + tid; t < a.tokens; t += kKeepThreads) {
      if (slot_at(a, t) >= 0) others = 1;
    }
  }
  __syncthreads();
  const int first = anchor != kNone ? found - anchor : taken - total;  // of the step's pages
  const int64_t behind = static_cast<int64_t>(first) + total;
  const bool known = anchor != kNone ? found >= 0 && (behind == taken || (behind > taken && taken == a.free_count))
                                     : taken < a.free_count && others == 0 && a.starts[0] <= 0 && a.starts[a.requests] <= a.tokens;
  if (first < 0 || !known) return 0;  // (the same for all)
  // Every page that a column got has to stand where it would: a list that was given its pages back already, or in parts, is another one.
  index = fresh_upto[tid];
  for (int r = from; r < to; ++r) {
    const Fresh f = fresh_of(a, r);
    for (int column = f.have; column < min(f.need, a.table_width); ++column) {
      const int at = first + index + column - f.have, got = a.table[r * a.table_stride + column];
      if (at >= 0 && at < taken ? a.free_pages[at] != got : got >= 0) elsewhere = 1;
    }
    index += f.need - f.have;
  }
  __syncthreads();
  if (elsewhere != 0) return 0;
  const auto dropped_of = [&](const Fresh &f, int index) {  // of a request whose first page is the step's `index`-th; a list that has run out has not given all
    return max(min(taken - first - (index + f.dropped - f.have), f.need - f.dropped), 0);
  };
  own = 0;
  index = fresh_upto[tid];
  for (int r = from; r < to; ++r) {
    const Fresh f = fresh_of(a, r);
    own += dropped_of(f, index);
    index += f.need - f.have;
  }
  upto_of(own, dropped_upto);
  const int dropped = dropped_upto[kKeepThreads];
  if (dropped < 0 || dropped > taken - first) return 0;  // (starts that are nobody's, whose sums pass 32 bits)
  // From the last one on: none moves down, so that what is read has not been written.
  for (int top = dropped; top > 0; top -= kKeepThreads) {
    int rest = top - 1 - tid;
    const int to_place = taken - dropped + rest;
    page = -1;
    if (rest >= 0) {
      int low = 0;
      for (int high = kKeepThreads; high - low > 1;) {
        const int mid = (low + high) >> 1;
        if (dropped_upto[mid] <= rest) low = mid; else high = mid;
      }
      rest -= dropped_upto[low];
      index = fresh_upto[low];
      for (int r = first_of(low); r < first_of(low + 1); ++r) {
        const Fresh f = fresh_of(a, r);
        const int count = dropped_of(f, index);
        if (rest < count) {
          const int at = first + index + f.dropped - f.have + rest;
          if (at >= first && at < taken) page = a.free_pages[at];  // (the same)
          break;
        }
        rest -= count;
        index += f.need - f.have;
      }
    }
    __syncthreads();
    if (top - 1 - tid >= 0) a.free_pages[to_place] = page;
    __syncthreads();
  }
  return dropped;
}

// Lengths, and the pages behind them onto the free list again, in front of those that it gives out next, in request order (those that no row names behind the others).
__device__ void keep_counts(const KvKeepArgs &a) {
  __shared__ int wave_sums[kKeepThreads / 64];
  __shared__ bool wave_dropped[kKeepThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int run = (a.requests + kKeepThreads - 1) / kKeepThreads, from = min(tid * run, a.requests), to = min(from + run, a.requests);
  const int taken = a.taken != nullptr ? min(max(*a.taken, 0), a.free_count) : 0;
  const auto pages_of = [&](int tokens) { return static_cast<int>(min((static_cast<int64_t>(max(tokens, 0)) + (1 << a.page_shift) - 1) >> a.page_shift, static_cast<int64_t>(a.table_width))); };
  // each(page) for a request's pages from `column` on, four of them requested at once
  const auto over_pages = [&](int r, int column, int end, const auto &each) {
    const int32_t *const row = a.table + r * a.table_stride;
    for (; column < end; column += 4) {
      int page[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) page[c] = column + c < end ? row[column + c] : -1;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (page[c] >= 0) each(page[c]);
      }
    }
  };
  int own = 0;
  bool dropped = false;
  for (int r = from; r < to; ++r) {
    const int length = max(a.lengths[r], 0);
    const Path path = path_of(a, r);
    const bool all = all_stay(a, r);
    const int kept = all ? length : max(length - path.fresh, 0) + kept_of(a, r, path);
    a.lengths_after[r] = kept;
    if (a.taken == nullptr) continue;
    over_pages(r, pages_of(kept), pages_of(length), [&](int) { ++own; });
    const Fresh f = fresh_of(a, length, path.fresh, all);
    dropped |= f.dropped < f.need;
  }
  if (a.taken == nullptr) return;
  const int sum = kv_sums(own);
  const bool some_dropped = __builtin_amdgcn_ballot_w64(dropped) != 0;
  if (lane == 63) {
    wave_sums[wave] = sum;
    wave_dropped[wave] = some_dropped;
  }
  __syncthreads();
  int ahead = sum - own, all = 0;
  bool any_dropped = false;
#pragma unroll
  for (int w = 0; w < kKeepThreads / 64; ++w) {
    ahead += w < wave ? wave_sums[w] : 0;
    all += wave_sums[w];
    any_dropped |= wave_dropped[w];
  }
  const int begin = taken - all - (any_dropped ? keep_dropped(a, taken) : 0);
  if (tid == 0) *a.taken_after = max(begin, 0);
  if (own == 0) return;
  int at = begin + ahead;
  for (int r = from; r < to; ++r) {
    over_pages(r, pages_of(a.lengths_after[r]) /* this thread's own */, pages_of(a.lengths[r]), [&](int page) {
      if (at >= 0) a.free_pages[at] = page;
      ++at;
    });
  }
}

template <int D>
__global__ __launch_bounds__(kKeepThreads) void kv_keep_kernel(KvKeepArgs a) {
  const int counting = a.counts ? 1 : 0;
  if (static_cast<int>(blockIdx.x) < counting) {
    keep_counts(a);
    return;
  }
  const int lane = threadIdx.x & 63;
  // (a launch has fewer than 2^26 of these: 2^32 threads)
  const uint32_t unit = (blockIdx.x - counting) * (kKeepThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t rest = unit / static_cast<uint32_t>(a.heads), layer = rest / static_cast<uint32_t>(a.requests);
  if (layer >= static_cast<uint32_t>(a.caches)) return;
  const int head = static_cast<int>(unit - rest * a.heads), r = static_cast<int>(rest - layer * a.requests);
  const auto &cache = a.cache[layer];
  const Path path = path_of(a, r);
  const int shift = a.page_shift, in_page = (1 << shift) - 1;
  int before = -1;  // the last entry of the lanes' batch before
  for (int base = 0; base < a.most; base += 64) {
    const int i = base + lane;
    const int k = i < a.most ? a.kept[static_cast<int64_t>(r) * a.most + i] : -1;
    const int ahead = __shfl_up(k, 1, 64), last = lane == 0 ? before : ahead;
    int64_t source = -1, target = -1;
    if (k > last && k < path.fresh) {
      source = slot_at(a, static_cast<int64_t>(path.first) + k);
      target = slot_at(a, static_cast<int64_t>(path.first) + i);  // (i <= k: a token of the request)
      if (target < 0) source = -1;
    }
    const uint64_t bad = __builtin_amdgcn_ballot_w64(source < 0);
    const int good = bad == 0 ? 64 : __builtin_ctzll(bad);
    before = __builtin_amdgcn_readlane(k, 63);
    // vectors of the cache, of codes and scales
    const auto vector_of = [&](int64_t slot) { return ((((slot >> shift) * a.heads + head) << shift) + (slot & in_page)); };
    const auto column_of = [&](int64_t slot) { return ((((slot >> shift) * a.heads + head) * (D / 2)) << shift) + (slot & in_page); };
    const auto of_lane = [&](int64_t x, int from) {
      return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x), from))) |
                                  static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(x >> 32), from))) << 32);
    };
    uint64_t moves = __builtin_amdgcn_ballot_w64(lane < good && source != target);
    while (moves != 0) {
      constexpr int ROWS = (D / 2 + 63) / 64;
      int64_t to[kKeepBatch];
      uint32_t key[kKeepBatch];
      uint16_t scale[kKeepBatch];
      uint8_t value[kKeepBatch][ROWS];
      int count = 0;
#pragma unroll
      for (int b = 0; b < kKeepBatch; ++b) {
        if (moves == 0) continue;
        const int from_lane = __builtin_ctzll(moves);
        moves &= moves - 1;
        const int64_t from = of_lane(source, from_lane);
        to[b] = of_lane(target, from_lane);
        count = b + 1;
        if (lane < D / 8) key[b] = reinterpret_cast<const uint32_t *>(cache.k_codes)[vector_of(from) * (D / 8) + lane];
        if (lane < 2) scale[b] = (lane == 0 ? cache.k_scales : cache.v_scales)[vector_of(from)];
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          if (64 * j + lane < D / 2) value[b][j] = cache.v_codes[column_of(from) + (static_cast<int64_t>(64 * j + lane) << shift)];
        }
      }
#pragma unroll
      for (int b = 0; b < kKeepBatch; ++b) {
        if (b >= count) continue;
        if (lane < D / 8) reinterpret_cast<uint32_t *>(cache.k_codes)[vector_of(to[b]) * (D / 8) + lane] = key[b];
        if (lane < 2) (lane == 0 ? cache.k_scales : cache.v_scales)[vector_of(to[b])] = scale[b];
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          if (64 * j + lane < D / 2) cache.v_codes[column_of(to[b]) + (static_cast<int64_t>(64 * j + lane) << shift)] = value[b][j];
        }
      }
    }
    if (good < 64) break;
  }
}

}  // namespace

int kv_tree_dispatch(const KvTreeArgs &a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.requests + 1));
  if (a.words == 1) launch_kernel(kv_tree_kernel<1>, grid, dim3(64), 0, stream, a);
  else if (a.words == 2) launch_kernel(kv_tree_kernel<2>, grid, dim3(128), 0, stream, a);
  else if (a.words == 3) launch_kernel(kv_tree_kernel<3>, grid, dim3(192), 0, stream, a);
  else launch_kernel(kv_tree_kernel<4>, grid, dim3(256), 0, stream, a);
  return check_launch("kv_tree");
}

int64_t kv_keep_blocks(const KvKeepArgs &a) {
  const int64_t units = static_cast<int64_t>(a.requests) * a.heads * a.caches, each = kKeepThreads / 64;
  return (units + each - 1) / each + (a.counts ? 1 : 0);
}

int kv_keep_dispatch(const KvKeepArgs &a, int dim, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(kv_keep_blocks(a)));
  if (dim == 64) launch_kernel(kv_keep_kernel<64>, grid, dim3(kKeepThreads), 0, stream, a);
  else if (dim == 128) launch_kernel(kv_keep_kernel<128>, grid, dim3(kKeepThreads), 0, stream, a);
  else launch_kernel(kv_keep_kernel<256>, grid, dim3(kKeepThreads), 0, stream, a);
  return check_launch("kv_keep");
}

}  // namespace oq
