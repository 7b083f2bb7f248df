// Attention over the 4-bit key/value cache: how the work is cut, and the launch that joins the parts of the keys.
// (No counterpart in the reference.)
#include "kv_attend_kernel.h"

namespace oq {

// One file each: they compile side by side.
bool kv_attend_64(const KvAttendArgs &a, int split, hipStream_t stream);
bool kv_attend_128(const KvAttendArgs &a, int split, hipStream_t stream);
bool kv_attend_256(const KvAttendArgs &a, int split, hipStream_t stream);

namespace {

// How launches are cut (MI355X, D = 128; a step is 64 keys).
// Few rows.  One launch and no join up to sixteen steps (1003 tokens, 32 heads: 8.9 us), and up to 64 where there are workgroups enough
// without, four for every step beyond sixteen, of shorter heads fewer, of longer ones more: 64 requests of up to 4096 tokens, 8 key heads, 47 -> 38 us,
// 16 of up to 2000 15.3 -> 12.9, but 4 of them 11.1 -> 12.5, and 16 of up to 4096, with the rest of their step, 24.8 -> 27.1; D = 64, 16 of up to
// 2000, 13.2 -> 10.5; D = 256, 4 key heads, 17.7 -> 19.3.  Longer ones could leave one workgroup at work alone for too long, 0.22 us a step.
// Cut, 512 workgroups or more, two on each compute unit at once: 131101 tokens, 8 heads, 34 us (before the other steps 1024: 39.7, 256: 35.0, 512: 34.6).
// Up to three times as many where a part keeps 60 steps, so that requests of different lengths even out, the longest parts first: 64 of up to
// 16384, 130 us (512 workgroups: 139; four times: 132).  Four steps a part at least, one a wavefront: 1500 of 5000 tokens, D = 256, 15.9 us.
// Short and many: one wavefront a workgroup instead of four that share few steps, where there are enough of them to fill the chip (500 requests of up to 60
// tokens, 8 heads, 31.5 -> 14.5 us, of up to 500 49 -> 43; 128 of up to 256 13.2 -> 10.1, but 64 of them 8.7 -> 9.4).
constexpr int kFewAlone = 8;  // steps
constexpr int kFewWhole = 16, kFewWholeMost = 64, kFewGroups = 512, kFewSteps = 60, kFewLeast = 4;
// Many rows.  A part is 128 rows of fp32 that are written and read again: only above sixteen steps (500 behind 300 tokens, 8 heads, 31 -> 36 us), and
// only where tiles are fewer than the workgroups that the chip holds, two on a compute unit, of heads of 256 one (2048 on their own, 264
// tiles of few steps each: 68 -> 97 us), into eight steps at least (with sixteen: 1500 in fp32, 4 heads, 58 us, now 50; 64 rows behind 2000 tokens, D = 256, 59
// and 43; with six these are as often slower).  512 queries behind 3584 tokens, 8 heads, 128 tiles: 117 -> 66 us.
constexpr int kManyGroups = 512, kManyWhole = 16, kManyLeast = 8;

constexpr int kJoinBlocks = 4;  // workgroups of a tile, at most

// The parts of the tiles that a launch has cut: out = sum_p 2^(R_p) o_p / sum_p 2^(R_p) l_p, in the order of the keys.  TPR threads a row:
// D / 4 of them have four dimensions each, and as many sets of those as there are take every so many-th part, so that a row of
// a hundred parts is not a chain of a hundred loads.
template <int D, int TPR, bool MANY>
__device__ __forceinline__ void join_tile(const KvAttendArgs &a, int block, int blocks) {
  constexpr int SETS = TPR / (D / 4), ROWS = 256 / TPR, TILE = MANY ? kKvManyRows : 16;
  __shared__ float4 sums[ROWS][SETS][D / 4];
  __shared__ float2 totals[ROWS][SETS];  // of a set: its largest R and its l
  const KvCut &cut = MANY ? a.many : a.few;
  const int in_block = threadIdx.x / TPR, t = threadIdx.x % TPR, set = t / (D / 4), d = t % (D / 4);
  const int in_launch = block / blocks;
  const int kv_head = in_launch % a.cache.heads, first = in_launch / a.cache.heads;
  const int2 *maps = cut.map + static_cast<int64_t>(kv_head) * (cut.places + 1);
  if (first >= maps[cut.places].x) return;  // (the same for the block, as is what follows)
  const int2 map = maps[first];
  if (map.x < 0) return;
  KvRows r;
  if (!kv_tile<MANY>(a, map.x, r)) return;
  for (int from = block % blocks * ROWS; from < r.rows; from += blocks * ROWS) {
    const int in_tile = from + in_block;
    const bool there = in_tile < r.rows;
    float best = kKvNothing, l = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const auto add = [&](const float2 &stats, const float4 &o) {
      const float both = fmaxf(best, stats.x), my_half = kv_half_power(best - both), their_half = kv_half_power(stats.x - both);
      const float mine = my_half * my_half, theirs = their_half * their_half;
      best = both;
      l = fmaf(l * my_half, my_half, stats.y * their_half * their_half);
      y.x = fmaf(y.x, mine, o.x * theirs); y.y = fmaf(y.y, mine, o.y * theirs);
      y.z = fmaf(y.z, mine, o.z * theirs); y.w = fmaf(y.w, mine, o.w * theirs);
    };
    if (there) {
      const int64_t place = (static_cast<int64_t>(kv_head) * cut.places + first) * TILE + in_tile;
#pragma unroll 4
      for (int p = set; p < map.y; p += SETS)
        add(cut.stats[place + static_cast<int64_t>(p) * TILE], reinterpret_cast<const float4 *>(cut.out + (place + static_cast<int64_t>(p) * TILE) * D)[d]);
    }
    if constexpr (SETS > 1) {
      sums[in_block][set][d] = y;
      if (d == 0) totals[in_block][set] = make_float2(best, l);
      __syncthreads();
      if (set == 0) {
#pragma unroll
        for (int s = 1; s < SETS; ++s) add(totals[in_block][s], sums[in_block][s][d]);
      }
      __syncthreads();
    }
    if (set != 0 || !there) continue;
    const KvRow at_row = kv_row_of(a, r, kv_head, r.first + in_tile, true);
    const int64_t row = static_cast<int64_t>(at_row.token) * a.heads + at_row.head;
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
}

// The first `many_blocks` workgroups have the prompts' tiles, the others those of few rows: FEW threads for one of these, `few_blocks` workgroups for a tile.
template <int D, int FEW>
__global__ __launch_bounds__(256) void kv_join_kernel(KvAttendArgs a, int many_blocks, int few_blocks) {
  const int block = blockIdx.x;
  if (block < many_blocks) join_tile<D, D / 4, true>(a, block, kJoinBlocks);
  else join_tile<D, FEW, false>(a, block - many_blocks, few_blocks);
}

template <int D>
void join(const KvAttendArgs &a, hipStream_t stream) {
  const int many = a.cache.heads * a.many.places * kJoinBlocks;
  // Few tiles have many parts each, and a row of them is a workgroup's; many have few.
  const bool long_rows = static_cast<int64_t>(a.few_requests) * a.few_tiles * a.cache.heads < 256;
  const int in_tile = long_rows ? a.few_in_tile : (a.few_in_tile + 3) / 4, few_blocks = in_tile < kJoinBlocks ? in_tile : kJoinBlocks;
  const dim3 grid(static_cast<unsigned>(many + a.cache.heads * a.few.places * few_blocks));
  if (long_rows) launch_kernel(kv_join_kernel<D, 256>, grid, dim3(256), 0, stream, a, many, few_blocks);
  else launch_kernel(kv_join_kernel<D, 64>, grid, dim3(256), 0, stream, a, many, few_blocks);
}

uint64_t kv_places(KvCut &cut, int places_a_head, int heads, int rows, int dim, char *workspace, uint64_t from) {
  cut.places = cut.target == 0 ? 0 : places_a_head;
  if (cut.target == 0) return from;
  const uint64_t places = static_cast<uint64_t>(places_a_head) * heads * rows;
  cut.out = reinterpret_cast<float *>(workspace + from);
  cut.stats = reinterpret_cast<float2 *>(workspace + from + places * dim * sizeof(float));
  cut.map = reinterpret_cast<int2 *>(workspace + from + places * (dim + 2) * sizeof(float));
  return from + places * (dim + 2) * sizeof(float) + (((places_a_head + 1ull) * heads * sizeof(int2) + 15) & ~15ull);
}

}  // namespace

uint64_t kv_attend_plan(KvAttendArgs &a, int dim, int64_t max_length, int64_t max_new, void *workspace) {
  const int64_t rows = a.tokens * a.group;
  const int heads = a.cache.heads;
  a.many_tiles = 0;
  a.few_rows = 0;
  if (a.starts == nullptr) {
    a.few_requests = a.requests;
    a.few_tiles = (a.group + 15) / 16;
    a.few_in_tile = a.group < 16 ? a.group : 16;
  } else {
    // A lone request's rows are known to be many, or few; of several, each may be either.
    const bool many = rows > kKvFewRows, few = !many || a.requests > 1;
    if (many) a.many_tiles = static_cast<int>(kv_tile_base(rows, a.requests)) + 1;
    a.few_requests = few ? a.requests + 1 : 0;
    a.few_tiles = static_cast<int>(((rows < kKvFewRows ? rows : kKvFewRows) + 15) / 16);
    a.few_in_tile = rows < 16 ? static_cast<int>(rows) : 16;
    a.few_rows = few ? kKvFewRows : 0;
  }
  int64_t keys = static_cast<int64_t>(a.table_width) << a.cache.page_shift;
  if (max_length >= 0 && max_length < keys) keys = max_length;
  if (a.window != 0 && keys > a.window + max_new) keys = a.window + max_new + 63;
  const int64_t steps = (keys + 63) / 64;
  a.few.target = a.many.target = 0;
  a.few.sorted = false;
  a.few.least = kFewLeast;
  a.many.least = kManyLeast;
  const int64_t whole = static_cast<int64_t>(a.few_requests) * a.few_tiles * heads;
  if (a.few_requests > 0 && steps > kFewWhole && (steps > kFewWholeMost || whole * 32 < (steps - kFewWhole) * dim)) {
    const int64_t parts = static_cast<int64_t>(a.requests) * steps * heads / kFewSteps;
    const int64_t groups = parts < kFewGroups ? kFewGroups : parts > 3 * kFewGroups ? 3 * kFewGroups : parts;
    a.few.sorted = groups > kFewGroups;
    a.few.target = groups > heads ? static_cast<int>(groups / heads) : 1;
  }
  a.few_alone = a.few_requests > 0 && a.few.target == 0 && steps <= kFewAlone && (steps <= 1 || whole > 128 * steps);
  const int many_groups = dim == 256 ? kManyGroups / 2 : kManyGroups;
  if (a.many_tiles > 0 && steps > kManyWhole && static_cast<int64_t>(a.many_tiles) * heads < many_groups * 3 / 4) a.many.target = heads < many_groups ? many_groups / heads : 1;
  const uint64_t bytes = kv_places(a.few, 2 * a.few.target, heads, 16, dim, static_cast<char *>(workspace), 0);
  return kv_places(a.many, a.many.target, heads, kKvManyRows, dim, static_cast<char *>(workspace), bytes);
}

bool kv_attend_fits(const KvAttendArgs &a, int dim) {
  const int64_t heads = a.cache.heads;
  const int64_t few = a.few_requests > 0 ? heads * (a.few.target + static_cast<int64_t>(a.few_requests) * a.few_tiles) : 0;
  const int64_t many = a.many_tiles > 0 ? heads * (a.many.target != 0 ? a.many.target : a.many_tiles) : 0;
  return few <= kKvMostThreads / (a.few_alone ? 64 : 256) && many <= kKvMostThreads / (64 * (dim == 256 ? kv_many_waves<256>() : kv_many_waves<64>()));
}

int kv_attend_dispatch(const KvAttendArgs &a, int dim, hipStream_t stream) {
  const int split = a.q_dtype == OQ_F32 ? 2 : a.q_dtype == OQ_F16 ? 1 : 0;
  const bool fits = dim == 64 ? kv_attend_64(a, split, stream) : dim == 128 ? kv_attend_128(a, split, stream) : kv_attend_256(a, split, stream);
  if (!fits) return fail(OQ_ERR_LAUNCH, "kv_attend: no LDS for heads of %d", dim);
  const int status = check_launch("kv_attend");
  if (status != OQ_OK || (a.few.target == 0 && a.many.target == 0)) return status;
  if (dim == 64) join<64>(a, stream);
  else if (dim == 128) join<128>(a, stream);
  else join<256>(a, stream);
  return check_launch("kv_attend");
}

}  // namespace oq
