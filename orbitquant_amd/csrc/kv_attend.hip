// Attention over the 4-bit key/value cache: how the work is cut, and the launch that joins the parts of the keys.
// (No counterpart in the reference.)
#include "kv_attend_kernel.h"

namespace oq {

// One file each: they compile side by side.
void kv_attend_64(const KvAttendArgs &a, int rt, int split, hipStream_t stream);
void kv_attend_128(const KvAttendArgs &a, int rt, int split, hipStream_t stream);
void kv_attend_256(const KvAttendArgs &a, int rt, int split, hipStream_t stream);

namespace {

constexpr int kMaxParts = 128;

// out = sum_p e^(lse_p) out_p / sum_p e^(lse_p), over the parts in order; a wavefront a row.
template <int D>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttendArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t rows = a.tokens * a.heads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float best = -INFINITY;
  bool broken = false;
  for (int p = lane; p < a.parts; p += 64) {
    const float s = a.part_lse[p * rows + row];
    broken |= s != s;
    best = fmaxf(best, s);
  }
#pragma unroll
  for (int x = 1; x < 64; x *= 2) best = fmaxf(best, __shfl_xor(best, x, 64));
  float sum = 0.0f, y[E] = {};
  if (best > -INFINITY || __builtin_amdgcn_ballot_w64(broken) != 0) {
    for (int p = 0; p < a.parts; ++p) {
      const float s = a.part_lse[p * rows + row];
      const float w = kv_exp2((s - best) * 1.44269504088896f);
      if (w == 0.0f) continue;
      sum += w;
      const float *from = a.part_out + (p * rows + row) * D + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) y[e] += w * from[e];
    }
  }
  const float by = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float v = y[e] * by;
    const int64_t at = row * D + lane * E + e;
    if (a.q_dtype == OQ_F32) store_from_f32<OQ_F32>(a.out, at, v);
    else if (a.q_dtype == OQ_F16) store_from_f32<OQ_F16>(a.out, at, v);
    else store_from_f32<OQ_BF16>(a.out, at, v);
  }
  if (a.lse != nullptr && lane == 0) a.lse[row] = sum != 0.0f ? best + __builtin_amdgcn_logf(sum) * 0.693147180559945f : -INFINITY;
}

// Row tiles a wavefront holds: two where a prompt's rows fill them, one for single tokens and for heads of 256, whose outputs take
// the registers of two.
int row_tiles(const KvAttendArgs &a, int dim, int64_t max_new) {
  return a.starts != nullptr && dim < 256 && max_new * a.group > 16 ? 2 : 1;
}

}  // namespace

uint64_t kv_attend_plan(KvAttendArgs &a, int dim, int64_t max_length, int64_t max_new) {
  const int rt = row_tiles(a, dim, max_new);
  const int tile_rows = 64 * rt;
  int64_t busy;  // workgroups with work
  if (a.starts == nullptr) {
    a.tiles = static_cast<int>(a.tokens * ((a.group + tile_rows - 1) / tile_rows));
    busy = a.tiles;
  } else {
    a.tiles = static_cast<int>(kv_tile_base(a.tokens * a.group, a.requests, tile_rows)) + 1;
    busy = (a.tokens * a.group + tile_rows - 1) / tile_rows;
  }
  busy *= a.cache.heads;
  int64_t keys = static_cast<int64_t>(a.table_width) << a.cache.page_shift;
  if (max_length >= 0 && max_length < keys) keys = max_length;
  if (a.window != 0 && keys > a.window + max_new) keys = a.window + max_new + 63;
  const int64_t steps = (keys + 63) / 64;
  int64_t parts = busy > 0 ? (1024 + busy - 1) / busy : 1;
  if (parts > steps / 4) parts = steps / 4;
  if (parts > kMaxParts) parts = kMaxParts;
  if (parts < 1) parts = 1;
  a.part_steps = static_cast<int>(steps > 0 ? (steps + parts - 1) / parts : 1);
  a.parts = static_cast<int>(steps > 0 ? (steps + a.part_steps - 1) / a.part_steps : 1);
  return a.parts > 1 ? static_cast<uint64_t>(a.parts) * a.tokens * a.heads * (dim + 1) * sizeof(float) : 0;
}

int kv_attend_dispatch(KvAttendArgs &a, int dim, int64_t max_new, hipStream_t stream) {
  const int rt = row_tiles(a, dim, max_new), split = a.q_dtype == OQ_F32 ? 2 : a.q_dtype == OQ_F16 ? 1 : 0;
  if (dim == 64) kv_attend_64(a, rt, split, stream);
  else if (dim == 128) kv_attend_128(a, rt, split, stream);
  else kv_attend_256(a, rt, split, stream);
  const int status = check_launch("kv_attend");
  if (status != OQ_OK || a.parts == 1) return status;
  const dim3 grid(static_cast<unsigned>((a.tokens * a.heads + 3) / 4));
  if (dim == 64) launch_kernel(kv_join_kernel<64>, grid, dim3(256), 0, stream, a);
  else if (dim == 128) launch_kernel(kv_join_kernel<128>, grid, dim3(256), 0, stream, a);
  else launch_kernel(kv_join_kernel<256>, grid, dim3(256), 0, stream, a);
  return check_launch("kv_attend");
}

}  // namespace oq
