// Attention over the 4-bit key/value cache, heads of 256.
#include "kv_attend_kernel.h"

namespace oq {

void kv_attend_256(const KvAttendArgs &a, int rt, int split, hipStream_t stream) {
  (void)rt;  // (always one)
  if (split == 0) kv_attend_launch<256, 1, 0>(a, stream);
  else if (split == 1) kv_attend_launch<256, 1, 1>(a, stream);
  else kv_attend_launch<256, 1, 2>(a, stream);
}

}  // namespace oq
