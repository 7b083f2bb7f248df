// Attention over the 4-bit key/value cache: how the work is cut, and the launch that joins the parts of the keys.
// (No counterpart in the reference.)
#include "kv_attend_kernel.h"

namespace oq {

// One file each: they compile side by side.
bool kv_attend_64(const KvAttendArgs &a, int split, hipStream_t stream);
bool kv_attend_128(const KvAttendArgs &a, int split, hipStream_t stream);
bool kv_attend_256(const KvAttendArgs &a, int split, hipStream_t stream);

namespace {

constexpr int kMaxParts = 128;

// out = sum_p 2^(R_p) o_p / sum_p 2^(R_p) l_p.  TPR threads a row: D / 4 of them have the four dimensions each, and as many sets of those
// as there are take every so many-th part, so that a row of a hundred parts is not a chain of a hundred loads.
template <int D, int TPR>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttendArgs a) {
  constexpr int SETS = TPR / (D / 4), ROWS = 256 / TPR;
  __shared__ float2 stats[ROWS][kMaxParts];
  __shared__ float4 sums[ROWS][SETS][D / 4];
  const int in_block = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int64_t rows = a.tokens * a.heads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + in_block;
  if (row < rows) {
    for (int p = t; p < a.parts; p += TPR) stats[in_block][p] = a.part_stats[p * rows + row];
  }
  __syncthreads();
  const int set = t / (D / 4), d = t % (D / 4);
  float best = kKvNothing, l = 0.0f;
  float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (row < rows) {
    for (int p = 0; p < a.parts; ++p) best = fmaxf(best, stats[in_block][p].x);
    for (int p = 0; p < a.parts; ++p) l += kv_exp2(stats[in_block][p].x - best) * stats[in_block][p].y;
#pragma unroll 4
    for (int p = set; p < a.parts; p += SETS) {
      const float w = kv_exp2(stats[in_block][p].x - best);
      const float4 o = reinterpret_cast<const float4 *>(a.part_out + (p * rows + row) * D)[d];
      y.x += w * o.x; y.y += w * o.y; y.z += w * o.z; y.w += w * o.w;
    }
  }
  sums[in_block][set][d] = y;
  __syncthreads();
  if (set != 0 || row >= rows) return;
#pragma unroll
  for (int s = 1; s < SETS; ++s) {
    const float4 o = sums[in_block][s][d];
    y.x += o.x; y.y += o.y; y.z += o.z; y.w += o.w;
  }
  const float by = l != 0.0f ? 1.0f / l : 0.0f;
  const float v[4] = {y.x * by, y.y * by, y.z * by, y.w * by};
  const int64_t at = row * D + 4 * d;
  if (a.q_dtype == OQ_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    uint32_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      w[e] = a.q_dtype == OQ_F16 ? f32_to_f16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_f16_bits(v[2 * e + 1])) << 16
                                 : f32_to_bf16_bits(v[2 * e]) | static_cast<uint32_t>(f32_to_bf16_bits(v[2 * e + 1])) << 16;
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at) = make_uint2(w[0], w[1]);
  }
  if (a.lse != nullptr && d == 0) a.lse[row] = l != 0.0f ? (best + __builtin_amdgcn_logf(l)) * 0.693147180559945f : -INFINITY;
}

template <int D>
void join(const KvAttendArgs &a, hipStream_t stream) {
  const int64_t rows = a.tokens * a.heads;
  if (a.parts > 8) launch_kernel(kv_join_kernel<D, 256>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, a);
  else launch_kernel(kv_join_kernel<D, 64>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, stream, a);
}

}  // namespace

uint64_t kv_attend_plan(KvAttendArgs &a, int dim, int64_t max_length, int64_t max_new) {
  const int64_t rows = a.tokens * a.group;
  int64_t busy;  // workgroups with work
  a.many_tiles = 0;
  a.few_rows = 0;
  if (a.starts == nullptr) {
    a.few_requests = a.requests;
    a.few_tiles = (a.group + 15) / 16;
    busy = static_cast<int64_t>(a.few_requests) * a.few_tiles;
  } else {
    // A lone request's rows are known to be many, or few; of several, each may be either.
    const bool many = rows > kKvFewRows, few = !many || a.requests > 1;
    if (many) a.many_tiles = static_cast<int>(kv_tile_base(rows, a.requests)) + 1;
    a.few_requests = few ? a.requests + 1 : 0;
    a.few_tiles = static_cast<int>(((rows < kKvFewRows ? rows : kKvFewRows) + 15) / 16);
    a.few_rows = few ? kKvFewRows : 0;
    busy = many ? (rows + kKvManyRows - 1) / kKvManyRows : a.few_tiles;
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
  return a.parts > 1 ? static_cast<uint64_t>(a.parts) * a.tokens * a.heads * (dim + 2) * sizeof(float) : 0;
}

int kv_attend_dispatch(const KvAttendArgs &a, int dim, hipStream_t stream) {
  const int split = a.q_dtype == OQ_F32 ? 2 : a.q_dtype == OQ_F16 ? 1 : 0;
  const bool fits = dim == 64 ? kv_attend_64(a, split, stream) : dim == 128 ? kv_attend_128(a, split, stream) : kv_attend_256(a, split, stream);
  if (!fits) return fail(OQ_ERR_LAUNCH, "kv_attend: no LDS for heads of %d", dim);
  const int status = check_launch("kv_attend");
  if (status != OQ_OK || a.parts == 1) return status;
  if (dim == 64) join<64>(a, stream);
  else if (dim == 128) join<128>(a, stream);
  else join<256>(a, stream);
  return check_launch("kv_attend");
}

}  // namespace oq
