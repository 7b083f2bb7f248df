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
  // How the work is cut: tiles of the kernel for many rows (0: not launched); requests (0 likewise) and tiles of each for the one for
  // few; the rows of a request up to which the latter has it; parts of the keys, and steps of 64 keys in one.
  int many_tiles, few_requests, few_tiles, few_rows, parts, part_steps;
  void *out;
  float *lse;                         // NULL or [tokens, heads]
  float *part_out;                    // where parts > 1: [parts, tokens, heads, D], and of each row R and l
  float2 *part_stats;
};

int kv_assign_dispatch(const KvAssignArgs &a, hipStream_t stream);
int kv_write_dispatch(const KvWriteArgs &a, int dim, int dtype, hipStream_t stream);
int kv_read_dispatch(const KvReadArgs &a, int dim, int dtype, hipStream_t stream);
// Cuts the work; the bytes of part_out and part_stats (0: none).
uint64_t kv_attend_plan(KvAttendArgs &a, int dim, int64_t max_length, int64_t max_new);
int kv_attend_dispatch(const KvAttendArgs &a, int dim, hipStream_t stream);

}  // namespace oq
