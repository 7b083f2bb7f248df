// Attention over the 4-bit key/value cache, heads of 256.
#include "kv_attend_kernel.h"

namespace oq {

bool kv_attend_256(const KvAttendArgs &a, int split, hipStream_t stream) {
  if (split == 0) return kv_attend_launch<256, 0>(a, stream);
  return split == 1 ? kv_attend_launch<256, 1>(a, stream) : kv_attend_launch<256, 2>(a, stream);
}

}  // namespace oq
