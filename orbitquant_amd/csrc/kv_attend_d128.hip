// Attention over the 4-bit key/value cache, heads of 128.
#include "kv_attend_kernel.h"

namespace oq {

bool kv_attend_128(const KvAttendArgs &a, int split, hipStream_t stream) { return kv_attend_of<128>(a, split, stream); }

}  // namespace oq
