// Attention over the 4-bit key/value cache, heads of 256.
#include "kv_attend_kernel.h"

namespace oq {

bool kv_attend_256(const KvAttendArgs &a, int split, hipStream_t stream) { return kv_attend_of<256, false>(a, split, stream); }

}  // namespace oq
