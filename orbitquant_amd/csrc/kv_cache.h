// What the entry points hand to the kernels of the 4-bit key/value cache.
#pragma once

#include "kv_format.h"

namespace oq {

struct KvAssignArgs {
  const int32_t *lengths, *new_lengths, *free_pages, *taken;
  int32_t *table;
  int64_t table_stride;
  int table_width, requests, free_count, page_shift;
  int64_t tokens;
  int64_t *slots;
  int32_t *positions, *starts, *lengths_after, *taken_after;
};

struct KvWriteArgs {
  KvCache cache;
  const void *k, *v;
  const int64_t *slots;
  int64_t tokens, k_token_stride, k_head_stride, v_token_stride, v_head_stride;  // strides in elements
  bool k_wide, v_wide;  // every vector begins on 16 bytes
};

struct KvReadArgs {
  KvCache cache;
  const int64_t *slots;
  void *k, *v;  // [tokens, heads, D], 16-byte aligned
  int64_t tokens;
};

// How a launch shares its work: for each key head, a tile's steps are cut into equal parts no longer than `longest` = max(least, all
// tiles' steps / target), a workgroup for each, so that there are about `target` of them however many tiles there are and whatever their lengths
// (of many rows, where a launch is cut only if it has fewer tiles than that, no more than `target`).
struct KvCut {
  int target, least;  // target 0: nothing is cut
  bool sorted;        // few rows: the longest parts first (for more parts than the chip holds at once)
  int places;         // for the parts of tiles that are cut: of few rows 2 * target (a tile of n > 1 parts has more than (n - 1) * longest steps), of many target
  float *out;         // [key heads, places, rows of a tile, D]
  float2 *stats;      // [key heads, places, rows of a tile]: R and l
  int2 *map;          // [key heads, places + 1]: of a tile's first part, the tile and the number of its parts, (-1, 0) of the others; and their number
};

struct KvAttendArgs {
  KvCache cache;
  const void *q;
  int q_dtype;
  int64_t tokens, q_token_stride, q_head_stride;
  bool q_wide;
  int heads, group, requests;         // query heads, query heads of a key head
  const int32_t *table, *lengths, *starts;  // starts: NULL for one query a request
  int64_t table_stride;
  int table_width, window;            // window: 0 for none
  bool causal;
  float scale;
  int few_tiles, few_requests, few_rows, few_in_tile;  // kernel for few rows: tiles of a request, requests (0: not launched), the rows of a request up to which it has it, rows of a tile at most
  bool few_alone;                     // in the first: one wavefront a workgroup
  int many_tiles;                     // kernel for many rows (0: not launched)
  KvCut few, many;
  void *out;
  float *lse;                         // NULL or [tokens, heads]
};

constexpr int64_t kKvMostThreads = 0xffffffffLL;  // of a launch
// Write and read: a workgroup has one head of sixteen tokens.
constexpr int kKvGroup = 16;
constexpr int kv_write_threads(int64_t dim) { return dim == 64 ? 128 : 256; }
constexpr int kv_read_threads(int64_t) { return 256; }

int kv_assign_dispatch(const KvAssignArgs &a, hipStream_t stream);
int kv_write_dispatch(const KvWriteArgs &a, int dim, int dtype, hipStream_t stream);
int kv_read_dispatch(const KvReadArgs &a, int dim, int dtype, hipStream_t stream);
// Cuts the work, whose parts go into `workspace`; the bytes that they need.
uint64_t kv_attend_plan(KvAttendArgs &a, int dim, int64_t max_length, int64_t max_new, void *workspace);
bool kv_attend_fits(const KvAttendArgs &a, int dim);  // a planned one's launches
int kv_attend_dispatch(const KvAttendArgs &a, int dim, hipStream_t stream);

}  // namespace oq
