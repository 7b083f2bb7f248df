// Norms of queries and keys for each head and their rotary positions, in one pass.  (No counterpart in the reference, whose models do
// this in torch operations.)
#include "qk_rotary.h"
#include "qk_rotary_calls.h"

namespace oq {
namespace {

// The first workgroups have the queries, the others the keys.
template <int DT, int L, int PIECE, bool INTERLEAVED, bool FULL>
__global__ __launch_bounds__(kQkThreads) void qk_norm_rotary_kernel(QkArgs a) {
  const bool keys = blockIdx.x >= a.q_blocks;
  qk_block<DT, L, qk_form(INTERLEAVED, L, PIECE), PIECE, FULL, kQkThreads>(a.how, a.side[keys], keys, a.tokens, a.dim, blockIdx.x - (keys ? a.q_blocks : 0));
}

template <int DT, int L, int PIECE, bool FULL>
void launch(const QkArgs &a, hipStream_t stream) {
  const dim3 grid(a.q_blocks + a.k_blocks);
  if (a.how.interleaved) launch_kernel(qk_norm_rotary_kernel<DT, L, PIECE, true, FULL>, grid, dim3(kQkThreads), 0, stream, a);
  else launch_kernel(qk_norm_rotary_kernel<DT, L, PIECE, false, FULL>, grid, dim3(kQkThreads), 0, stream, a);
}
template <int DT, int L>
void launch(const QkArgs &a, hipStream_t stream) {
  if (a.how.piece == 8 && a.dim == 16 * L) launch<DT, L, 8, true>(a, stream);
  else if (a.how.piece == 8) launch<DT, L, 8, false>(a, stream);
  else if (a.how.piece == 4) launch<DT, L, 4, false>(a, stream);
  else launch<DT, L, 1, false>(a, stream);
}
template <int L>
void launch(const QkArgs &a, int dtype, hipStream_t stream) {
  if (dtype == OQ_F32) launch<OQ_F32, L>(a, stream);
  else if (dtype == OQ_F16) launch<OQ_F16, L>(a, stream);
  else launch<OQ_BF16, L>(a, stream);
}

}  // namespace

int qk_norm_rotary_dispatch(const QkArgs &a, int dtype, hipStream_t stream) {
  switch (qk_lanes(a.dim)) {
    case 1: launch<1>(a, dtype, stream); break;
    case 2: launch<2>(a, dtype, stream); break;
    case 4: launch<4>(a, dtype, stream); break;
    case 8: launch<8>(a, dtype, stream); break;
    case 16: launch<16>(a, dtype, stream); break;
    default: launch<32>(a, dtype, stream); break;
  }
  return check_launch("qk_norm_rotary");
}

}  // namespace oq
