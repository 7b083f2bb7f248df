// What the entry points hand to the kernels of norms and rotary positions.
#pragma once

#include "qk_rotary.h"

namespace oq {

constexpr int kQkMostDim = 512;
constexpr int kQkThreads = 256;

struct QkArgs {
  QkNormRotary how;
  QkSide side[2];          // queries, keys
  int64_t tokens;
  int dim;
  uint32_t q_blocks, k_blocks;
};

struct KvAppendArgs {
  KvWriteArgs write;       // (its k as it comes)
  QkNormRotary how;
  QkSide q;
  uint32_t kv_blocks, q_blocks;
};

// Lanes of a head: eight pairs each.
constexpr int qk_lanes(int dim) {
  int lanes = 1;
  while (16 * lanes < dim) lanes *= 2;
  return lanes;
}
inline int64_t qk_blocks(int64_t tokens, int groups, int dim, int threads) {
  const int64_t units = threads / qk_lanes(dim);
  return (tokens * groups + units - 1) / units;
}

int qk_norm_rotary_dispatch(const QkArgs &a, int dtype, hipStream_t stream);
int kv_append_dispatch(const KvAppendArgs &a, int dim, int dtype, hipStream_t stream);

}  // namespace oq
