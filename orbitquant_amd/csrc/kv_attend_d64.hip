// Attention over the 4-bit key/value cache, heads of 64.
#include "kv_attend_kernel.h"

namespace oq {

void kv_attend_64(const KvAttendArgs &a, int rt, int split, hipStream_t stream) {
  if (rt == 2) {
    if (split == 0) kv_attend_launch<64, 2, 0>(a, stream);
    else if (split == 1) kv_attend_launch<64, 2, 1>(a, stream);
    else kv_attend_launch<64, 2, 2>(a, stream);
    return;
  }
  if (split == 0) kv_attend_launch<64, 1, 0>(a, stream);
  else if (split == 1) kv_attend_launch<64, 1, 1>(a, stream);
  else kv_attend_launch<64, 1, 2>(a, stream);
}

}  // namespace oq
