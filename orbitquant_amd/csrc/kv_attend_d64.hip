// Attention over the 4-bit key/value cache, heads of 64.
#include "kv_attend_kernel.h"

namespace oq {

bool kv_attend_64(const KvAttendArgs &a, int split, hipStream_t stream) { return kv_attend_of<64, false>(a, split, stream); }

}  // namespace oq
