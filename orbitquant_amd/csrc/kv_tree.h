// What the entry points hand to the kernels around trees of drafted tokens.
#pragma once

#include "kv_format.h"

namespace oq {

constexpr int kKvMaskWords = 4;    // of a mask, at most: 256 new tokens of a request
constexpr int kKvMostKept = 256;   // of a request's tokens
constexpr int kKvKeepCaches = 64;  // of one launch

struct KvTreeArgs {
  const int32_t *parents, *starts, *lengths;
  int requests, words;
  int64_t tokens;
  int32_t *positions;
  uint64_t *masks;
};

struct KvKeepArgs {
  const int32_t *kept, *lengths, *starts;
  const int64_t *slots;
  int64_t tokens, pages, table_stride;
  int requests, most, heads, page_shift, table_width, free_count;
  const int32_t *table, *taken;    // taken NULL: no page is given back
  int32_t *free_pages, *lengths_after, *taken_after;
  bool counts;                     // the launch whose first workgroup makes lengths and free pages
  int caches;
  struct {
    uint8_t *k_codes, *v_codes;
    uint16_t *k_scales, *v_scales;
  } cache[kKvKeepCaches];
};

int kv_tree_dispatch(const KvTreeArgs &a, hipStream_t stream);
int64_t kv_keep_blocks(const KvKeepArgs &a);
int kv_keep_dispatch(const KvKeepArgs &a, int dim, hipStream_t stream);

}  // namespace oq
