// Attention of drafted tokens over the 4-bit key/value cache, heads of 256.
#include "kv_attend_kernel.h"

namespace oq {

bool kv_attend_tree_256(const KvAttendArgs &a, int split, hipStream_t stream) { return kv_attend_of<256, true>(a, split, stream); }

}  // namespace oq
