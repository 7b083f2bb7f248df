// Attention over the 4-bit key/value cache, heads of 128.
#include "kv_attend_kernel.h"

namespace oq {

bool kv_attend_128(const KvAttendArgs &a, int split, hipStream_t stream) {
  if (split == 0) return kv_attend_launch<128, 0>(a, stream);
  return split == 1 ? kv_attend_launch<128, 1>(a, stream) : kv_attend_launch<128, 2>(a, stream);
}

}  // namespace oq
