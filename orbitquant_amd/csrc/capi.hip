// extern "C" entry points: argument validation and kernel selection.
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <map>
#include <memory>
#include <mutex>
#include <new>
#include <utility>

#include "dense_gemm.h"
#include "gemm_epilogue.h"
#include "kv_cache.h"
#include "kv_tree.h"
#include "qk_rotary_calls.h"
#include "rotate_plan.h"

namespace oq {

static thread_local char g_error[512] = "";

void set_error(const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
}

int fail(oq_status code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return static_cast<int>(code);
}

int check_launch(const char *what) {
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return fail(OQ_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(err));
  return OQ_OK;
}

bool reserve_dynamic_lds(const void *kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return true;
  static std::mutex lock;
  static std::map<std::pair<const void *, int>, size_t> granted;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  std::lock_guard<std::mutex> guard(lock);
  size_t &have = granted[std::make_pair(kernel, dev)];
  if (bytes <= have) return true;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)) != hipSuccess) return false;
  have = bytes;
  return true;
}

namespace {
const char *const kEnvNames[ENV_COUNT] = {"OQ_GEMM_TILE", "OQ_NO_TOKEN_LINEAR", "OQ_RQ_ONE_GROUP", "OQ_GEMV_CFG", "OQ_RQ_WAVES",
                                          "OQ_RQ_FAST_MIN_M", "OQ_NO_GEMV_GROUP", "OQ_GEMV_GROUP_R", "OQ_GEMV_NO_ASTAGE",
                                          "OQ_GEMV_MAX_M", "OQ_GEMM_WG_SPLIT", "OQ_FLOAT_GEMM_MIN_M", "OQ_GEMM_STAMPS", "OQ_DENSE_GEMM"};
const char *env_values[ENV_COUNT];
bool overrides_allowed = false;  // ORBITQUANT_DEBUG=1 in the environment the process started with
void env_load() {
  static std::once_flag once;
  std::call_once(once, [] {
    for (int i = 0; i < ENV_COUNT; ++i) env_values[i] = getenv(kEnvNames[i]);
    const char *debug = getenv("ORBITQUANT_DEBUG");
    overrides_allowed = debug != nullptr && strcmp(debug, "1") == 0;
  });
}
}  // namespace

// The experiment switches: read from the environment once per process, then only changed through
// oq_debug_override.
const char *debug_env(int which) {
  env_load();
  return env_values[which];
}

int debug_env_set(const char *name, const char *value) {
  env_load();
  if (!overrides_allowed)  // a switch changes which kernel runs and so the bits of a result: not for a serving process
    return fail(OQ_ERR_INVALID, "debug_override: switches are fixed in this process (start it with ORBITQUANT_DEBUG=1 to change them at run time)");
  for (int i = 0; i < ENV_COUNT; ++i) {
    if (strcmp(name, kEnvNames[i]) == 0) {
      env_values[i] = value != nullptr ? strdup(value) : nullptr;  // a few bytes per call, never freed: readers may hold the old one
      return OQ_OK;
    }
  }
  return fail(OQ_ERR_INVALID, "debug_override: unknown switch %s", name);
}

// kernels (defined in the other translation units)
int rotate_quantize_dispatch(const void *x, int x_dtype, int64_t M, int64_t K, const int32_t *perm,
                             const int8_t *signs, const float *boundaries, const float *centroids,
                             int levels, int64_t block, float eps, float inv_sqrt_block,
                             void *codes_out, int code_format, void *values_out, int values_mode,
                             float *norms_out, const uint16_t *input_map, const void *plan, hipStream_t stream);
int quantize_weight_fast(const void *w, int w_dtype, int64_t N, int64_t K, const void *plan, const float *boundaries,
                         int levels, int64_t block, float eps, float inv_sqrt_block, int bits, uint8_t *packed_out,
                         uint16_t *row_norms_out, hipStream_t stream);
int gemm_tiled_dispatch(bool f16, const void *x, const float *token_scale, const uint8_t *w, int bits, const uint16_t *row_norms,
                        const float *w_cents, const void *bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void *out,
                        int out_dtype, void *workspace, uint64_t workspace_bytes, hipStream_t stream);
uint64_t gemm_tiled_workspace_bytes(int64_t M, int64_t N, int64_t K, int bits, bool f16);
uint64_t gemm_workspace_bytes(int64_t M, int64_t N, int64_t K, int bits, bool byte_codes, bool decoded);
int gemm_staged_dispatch(const void *x, const float *token_scale, const uint8_t *w, int bits, const uint16_t *row_norms,
                         const float *w_cents, const void *bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void *out,
                         int out_dtype, hipStream_t stream);
int adaln_int4_dispatch(const uint16_t *x, const uint8_t *packed, const uint16_t *scales, const uint16_t *bias, int64_t M,
                        int64_t N, int64_t K, int64_t group, uint16_t *out, hipStream_t stream);
int adaln_quantize_dispatch(const void *w, int w_dtype, int64_t N, int64_t K, int64_t group, uint8_t *packed, float *scales,
                            hipStream_t stream);
int pack_lowbit_dispatch(const uint8_t *values, int bits, int64_t count, uint8_t *packed, hipStream_t stream);
int dequantize_dispatch(const uint8_t *packed, int bits, const uint16_t *row_norms, const float *centroids, int64_t N, int64_t K,
                        void *out, int out_dtype, hipStream_t stream);
bool token_linear_supported(int x_dtype, int64_t M, int64_t N, int64_t K, int levels, int bits, const void *x,
                            const int32_t *perm, const int8_t *signs);
int token_linear_dispatch(const void *x, int x_dtype, const uint16_t *input_map, int64_t K, const int32_t *perm,
                          const int8_t *signs, const float *boundaries, const float *act_cents, int levels,
                          int64_t block, float eps, float inv_sqrt_block, const void *plan, const uint8_t *packed_w, int bits,
                          const uint16_t *row_norms, const float *w_cents, const void *bias, int bias_dtype,
                          int64_t N, void *out, int out_dtype, const uint16_t *out_map, hipStream_t stream, bool *launched);
int generic_matmul_float(const void *x, int x_dtype, const float *token_scale, const uint8_t *packed_w,
                         int bits, const uint16_t *row_norms, const float *w_cents, const void *bias,
                         int bias_dtype, int64_t M, int64_t N, int64_t K, void *out, int out_dtype,
                         hipStream_t stream);
int generic_linear_codes(const void *codes, int code_format, const float *token_norms,
                         const float *act_cents, int a_levels, const uint8_t *packed_w, int bits,
                         const uint16_t *row_norms, const float *w_cents, const void *bias,
                         int bias_dtype, int64_t M, int64_t N, int64_t K, void *out, int out_dtype,
                         hipStream_t stream);
int unpack_dispatch(const uint8_t *packed, int bits, int64_t count, uint8_t *out, hipStream_t stream);
bool gemm_supported(int64_t K, int bits);
double gemm_call_price(int64_t M, int64_t N, int64_t K, int bits, bool without_small = false);
int gemm_dispatch(int a_mode, const void *a, const float *row_scale, const float *act_cents, int a_levels,
                  const uint8_t *w, int bits, const uint16_t *row_norms, const float *w_cents,
                  const void *bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void *out,
                  int out_dtype, const uint16_t *out_map, void *workspace, uint64_t workspace_bytes, hipStream_t stream);
int apply_value_map(void *out, int64_t count, const uint16_t *table, hipStream_t stream);
int gemm_choose_tile(int64_t M, int64_t N, int64_t K, int bits);
bool gemm_av_supported(int64_t K, int bits);
int gemm_av_dispatch(bool f16, const void *a, const float *row_scale, const uint8_t *w, int bits,
                     const uint16_t *row_norms, const float *w_cents, const void *bias, int bias_dtype,
                     int64_t M, int64_t N, int64_t K, void *out, int out_dtype, int tile, hipStream_t stream);
bool gemv_supported(int64_t M, int64_t K, int bits, int code_format, int a_levels);
int gemv_dispatch(const void *codes, int code_format, const float *row_scale, const float *act_cents, int a_levels,
                  const uint8_t *w, int bits, const uint16_t *row_norms, const float *w_cents,
                  const void *bias, int bias_dtype, int64_t M, int64_t N, int64_t K, void *out,
                  int out_dtype, const uint16_t *out_map, hipStream_t stream);
int gemv_group_dispatch(const void *codes, int code_format, const float *row_scale, const float *act_cents, int a_levels,
                        int count, const uint8_t *const *w, const int *bits, const uint16_t *const *row_norms,
                        const float *const *w_cents, const void *const *bias, int bias_dtype, int64_t M,
                        const int64_t *N, int64_t K, void *const *out, int out_dtype, hipStream_t stream, bool *launched);
// Scratch of oq_quantized_linear_static: the activation codes and token norms that pass from the
// quantizer launch to the matmul launch.  One copy per GPU, at its own address there; host code
// only ever uses the address hipGetSymbolAddress returns for the current device.
constexpr size_t kStaticScratchBytes = OQ_STATIC_SCRATCH_BYTES;
static __device__ __attribute__((used)) __align__(256) unsigned char scratch[kStaticScratchBytes];

constexpr int kMaxDevices = 64;
static int static_scratch_address(unsigned char **out) {
  static std::mutex lock;
  static unsigned char *address[kMaxDevices];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return fail(OQ_ERR_LAUNCH, "no HIP device is current");
  if (dev < 0 || dev >= kMaxDevices) return fail(OQ_ERR_UNSUPPORTED, "device index %d is beyond %d", dev, kMaxDevices - 1);
  std::lock_guard<std::mutex> guard(lock);
  if (address[dev] == nullptr) {
    void *ptr = nullptr;
    const hipError_t err = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
    if (err != hipSuccess || ptr == nullptr)
      return fail(OQ_ERR_LAUNCH, "cannot resolve the static scratch on device %d: %s", dev, hipGetErrorString(err));
    address[dev] = static_cast<unsigned char *>(ptr);
  }
  *out = address[dev];
  return OQ_OK;
}

static bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static bool valid_dtype(int dt) { return dt == OQ_F32 || dt == OQ_F16 || dt == OQ_BF16; }

static int check_matmul_common(const char *who, const uint8_t *packed_w, int bits, const uint16_t *row_norms,
                               const float *w_cents, const void *bias, int bias_dtype, int64_t M, int64_t N,
                               int64_t K, const void *out, int out_dtype) {
  if (M < 0 || N <= 0 || K <= 0) return fail(OQ_ERR_INVALID, "%s: M=%lld N=%lld K=%lld", who, (long long)M, (long long)N, (long long)K);
  if (bits < 1 || bits > 8) return fail(OQ_ERR_INVALID, "%s: bits=%d not in [1, 8]", who, bits);
  if (packed_w == nullptr || row_norms == nullptr || w_cents == nullptr || (out == nullptr && M > 0))
    return fail(OQ_ERR_INVALID, "%s: null pointer", who);
  if (!valid_dtype(out_dtype)) return fail(OQ_ERR_INVALID, "%s: out_dtype=%d", who, out_dtype);
  if (bias != nullptr && !valid_dtype(bias_dtype)) return fail(OQ_ERR_INVALID, "%s: bias_dtype=%d", who, bias_dtype);
  return OQ_OK;
}

}  // namespace oq

using namespace oq;

extern "C" {

const char *oq_last_error(void) { return g_error; }

const char *oq_version(void) { return "orbitquant-hip 0.1 (gfx950)"; }

int oq_device_ok(void) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return fail(OQ_ERR_LAUNCH, "no HIP device is current");
  hipDeviceProp_t prop;
  if (hipGetDeviceProperties(&prop, dev) != hipSuccess) return fail(OQ_ERR_LAUNCH, "cannot query device %d", dev);
  if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    return fail(OQ_ERR_UNSUPPORTED, "device %d is %s; this library holds gfx950 code only", dev, prop.gcnArchName);
  unsigned char *unused = nullptr;
  return static_scratch_address(&unused);  // resolved here so that later calls (e.g. under graph capture) only look it up
}

int oq_rotate_quantize(const void *x, int x_dtype, int64_t M, int64_t K, const int32_t *perm,
                       const int8_t *signs, const float *boundaries, const float *centroids, int levels,
                       int64_t block, float eps, float inv_sqrt_block, const void *rotate_plan, void *codes_out,
                       int code_format, void *values_out, int values_mode, float *norms_out, void *stream) {
  return rotate_quantize_dispatch(x, x_dtype, M, K, perm, signs, boundaries, centroids, levels, block, eps,
                                  inv_sqrt_block, codes_out, code_format, values_out, values_mode, norms_out,
                                  nullptr, rotate_plan, as_stream(stream));
}

uint64_t oq_rotate_plan_bytes(int64_t K) { return K > 0 ? plan::plan_bytes(K) : 0u; }

int oq_rotate_plan_build(const int32_t *perm, const int8_t *signs, const float *boundaries, int levels, int64_t K,
                         int64_t block, float inv_sqrt_block, void *plan_out, void *stream) {
  return rotate_plan_build(perm, signs, boundaries, levels, K, block, inv_sqrt_block, plan_out, nullptr, nullptr, as_stream(stream));
}

int oq_rotate_plan_build_copy(const int32_t *perm, const int8_t *signs, const float *boundaries, int levels, int64_t K, int64_t block,
                              float inv_sqrt_block, void *plan_out, int32_t *perm_copy, int8_t *signs_copy, void *stream) {
  if (perm_copy == nullptr || signs_copy == nullptr) return fail(OQ_ERR_INVALID, "rotate_plan_build_copy: null copy");
  return rotate_plan_build(perm, signs, boundaries, levels, K, block, inv_sqrt_block, plan_out, perm_copy, signs_copy, as_stream(stream));
}

int oq_rotate_quantize_mapped(const void *x, int x_dtype, const uint16_t *input_map, int64_t M, int64_t K,
                              const int32_t *perm, const int8_t *signs, const float *boundaries,
                              const float *centroids, int levels, int64_t block, float eps, float inv_sqrt_block,
                              const void *rotate_plan, void *codes_out, int code_format, void *values_out,
                              int values_mode, float *norms_out, void *stream) {
  if (input_map == nullptr) return fail(OQ_ERR_INVALID, "rotate_quantize_mapped: input_map is null");
  return rotate_quantize_dispatch(x, x_dtype, M, K, perm, signs, boundaries, centroids, levels, block, eps,
                                  inv_sqrt_block, codes_out, code_format, values_out, values_mode, norms_out,
                                  input_map, rotate_plan, as_stream(stream));
}

int oq_quantize_weight(const void *w, int w_dtype, int64_t N, int64_t K, const void *rotate_plan,
                       const float *boundaries, int levels, int64_t block, float eps, float inv_sqrt_block, int bits,
                       uint8_t *packed_out, uint16_t *row_norms_out, void *stream) {
  const int rc = quantize_weight_fast(w, w_dtype, N, K, rotate_plan, boundaries, levels, block, eps, inv_sqrt_block, bits,
                                      packed_out, row_norms_out, as_stream(stream));
  return rc < 0 ? fail(OQ_ERR_UNSUPPORTED, "quantize_weight: no kernel for block %lld", (long long)block) : rc;
}

// oq_packed_linear with an optional output map (applied where the tile and the streaming kernels store, by a
// small elementwise launch after the other kernels).
static int packed_linear_impl(const void *codes, int code_format, const float *token_norms,
                              const float *act_centroids, int a_bits, const uint8_t *packed_w, int w_bits,
                              const uint16_t *row_norms, const float *w_centroids, const void *bias, int bias_dtype,
                              int64_t M, int64_t N, int64_t K, void *out, int out_dtype, const uint16_t *out_map,
                              void *workspace, uint64_t workspace_bytes, void *stream) {
  if (int rc = check_matmul_common("packed_linear", packed_w, w_bits, row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype)) return rc;
  if (M == 0) return OQ_OK;
  if (codes == nullptr || act_centroids == nullptr) return fail(OQ_ERR_INVALID, "packed_linear: null codes/centroids");
  if (a_bits < 1 || a_bits > 8) return fail(OQ_ERR_INVALID, "packed_linear: a_bits=%d", a_bits);
  if (code_format != OQ_CODES_U8 && code_format != OQ_CODES_NIBBLE) return fail(OQ_ERR_INVALID, "packed_linear: code_format=%d", code_format);
  if (code_format == OQ_CODES_NIBBLE && (a_bits > 4 || (K & 1))) return fail(OQ_ERR_INVALID, "packed_linear: nibble codes need a_bits <= 4 and even K");
  if (out_map != nullptr) {
    if (out_dtype == OQ_F32) return fail(OQ_ERR_INVALID, "packed_linear: an output map needs a 16-bit output dtype");
    if (!aligned16(out_map)) return fail(OQ_ERR_INVALID, "packed_linear: the output map must be 16-byte aligned");
  }
  const int a_levels = 1 << a_bits;
  hipStream_t s = as_stream(stream);
  const bool fast_ptrs = aligned16(codes) && aligned16(packed_w);
  const bool tiled_out = gemm_output_ok(N, out);  // the tiled kernels store 16-byte row segments
  int rc;
  if (fast_ptrs && gemv_supported(M, K, w_bits, code_format, a_levels)) {
    return gemv_dispatch(codes, code_format, token_norms, act_centroids, a_levels, packed_w, w_bits, row_norms, w_centroids,
                         bias, bias_dtype, M, N, K, out, out_dtype, out_map, s);
  } else if (fast_ptrs && tiled_out && gemm_supported(K, w_bits) && (code_format == OQ_CODES_NIBBLE || M > 16)) {
    return gemm_dispatch(code_format == OQ_CODES_NIBBLE ? 0 : 1, codes, token_norms, act_centroids, a_levels, packed_w, w_bits, row_norms, w_centroids,
                         bias, bias_dtype, M, N, K, out, out_dtype, out_map, workspace, workspace_bytes, s);
  } else {
    rc = generic_linear_codes(codes, code_format, token_norms, act_centroids, a_levels, packed_w, w_bits, row_norms,
                              w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, s);
  }
  if (rc != OQ_OK || out_map == nullptr) return rc;
  return apply_value_map(out, M * N, out_map, s);
}

int oq_debug_override(const char *name, const char *value) {
  if (name == nullptr) return fail(OQ_ERR_INVALID, "debug_override: null name");
  return debug_env_set(name, value);
}

static uint64_t linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int code_format, int a_bits, bool decoded) {
  if (M <= 0 || N <= 0 || K <= 0 || a_bits < 1 || a_bits > 8) return 0;
  if (gemv_supported(M, K, w_bits, code_format, 1 << a_bits)) return 0;  // the streaming kernel
  if (N % 8 != 0 || !gemm_supported(K, w_bits) || !(code_format == OQ_CODES_NIBBLE || M > 16)) return 0;
  return gemm_workspace_bytes(M, N, K, w_bits, code_format == OQ_CODES_U8, decoded);
}

uint64_t oq_packed_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int code_format, int a_bits) {
  return linear_workspace_bytes(M, N, K, w_bits, code_format, a_bits, true);
}

uint64_t oq_packed_linear_least_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int code_format, int a_bits) {
  return linear_workspace_bytes(M, N, K, w_bits, code_format, a_bits, false);
}

uint64_t oq_matmul_packed_weight_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int x_dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || (x_dtype != OQ_BF16 && (x_dtype != OQ_F16 || M <= 8)) || N % 8 != 0 || !gemm_supported(K, w_bits)) return 0;
  return gemm_tiled_workspace_bytes(M, N, K, w_bits, x_dtype == OQ_F16);
}

int oq_packed_linear(const void *codes, int code_format, const float *token_norms, const float *act_centroids,
                     int a_bits, const uint8_t *packed_w, int w_bits, const uint16_t *row_norms,
                     const float *w_centroids, const void *bias, int bias_dtype, int64_t M, int64_t N,
                     int64_t K, void *out, int out_dtype, void *workspace, uint64_t workspace_bytes, void *stream) {
  return packed_linear_impl(codes, code_format, token_norms, act_centroids, a_bits, packed_w, w_bits, row_norms,
                            w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, nullptr, workspace, workspace_bytes, stream);
}

// Tile of the int8 launch, -1 where it does not run or oq_packed_linear, with the workspace that it asks for, is as
// fast.  That one multiplies the same integers in bf16, at half the rate, without the two passes.  Measured against it:
// 4608 x 36864 x 4096 1122 -> 616 us, 1024 x 14336 x 4096 100 -> 74 us, 2048 x 4096 x 4096 67 -> 52 us,
// 2048 x 4608 x 1152 34 -> 46 us; where it shares K between workgroups 74 x 784 x 8000 18 -> 45 us, 300 x 2048 x 7488
// 25 -> 50 us.  Asked for 10 %, the prices (dense_choose_tile, gemm_call_price) send 261 of 650 measured shapes here,
// 5 of them to more than 3 % more time, all with rows of some hundred values.
static int int8_choose_tile(int64_t M, int64_t N, int64_t K) {
  if (M <= 64 || N <= 0 || K <= 0 || K > 131071) return -1;  // (sums of K products of two int8 values stay below 2^31)
  double cost = 0.0;
  const int tile = dense_choose_tile(M, N, K, dense_rows_at_a_time(M, K, MF_I8), MF_I8, 1.5 * static_cast<double>(K) * static_cast<double>(M + N), &cost);
  if (tile < 0 || debug_env(ENV_DENSE_GEMM) != nullptr) return tile;
  // (its sums are whole numbers: the 64x64 tiles, which sum in fp32, take no problem from it that the larger ones leave)
  return cost < 0.9 * fmax(gemm_call_price(M, N, K, 4), gemm_call_price(M, N, K, 4, true)) ? tile : -1;
}

uint64_t oq_packed_linear_int8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (int8_choose_tile(M, N, K) < 0) return 0;
  return dense_workspace_bytes(M, N, K, MF_I8);
}

int oq_packed_linear_int8(const void *codes, const float *token_norms, float scale, const int8_t *act_table, const uint8_t *packed_w,
                          const uint16_t *row_norms, const int8_t *w_table, const void *bias, int bias_dtype, int64_t M, int64_t N,
                          int64_t K, void *out, int out_dtype, void *workspace, uint64_t workspace_bytes, void *stream) {
  if (int rc = check_matmul_common("packed_linear_int8", packed_w, 4, row_norms, reinterpret_cast<const float *>(w_table), bias, bias_dtype, M, N, K, out, out_dtype)) return rc;
  if (M == 0) return OQ_OK;
  if (codes == nullptr || act_table == nullptr) return fail(OQ_ERR_INVALID, "packed_linear_int8: null codes/table");
  const int tile = int8_choose_tile(M, N, K);
  const uint64_t need = tile < 0 ? 0 : dense_workspace_bytes(M, N, K, MF_I8);
  if (need == 0 || !aligned16(codes) || !aligned16(packed_w) || !gemm_output_ok(N, out))
    return fail(OQ_ERR_UNSUPPORTED, "packed_linear_int8: M=%lld N=%lld K=%lld or an alignment (oq_packed_linear takes it)", (long long)M, (long long)N, (long long)K);
  if (workspace == nullptr || workspace_bytes < need || !aligned16(workspace)) return fail(OQ_ERR_INVALID, "packed_linear_int8: %llu bytes of workspace needed", (unsigned long long)need);
  hipStream_t s = as_stream(stream);
  const int64_t rows = dense_rows_at_a_time(M, K, MF_I8);
  unsigned char *a_values = static_cast<unsigned char *>(workspace), *w_values = a_values + operand_order_bytes(rows, K, 1);
  for (int64_t m = 0; m < M; m += rows) {
    const int64_t count = M - m < rows ? M - m : rows;
    if (int rc = decode_operands_int8(static_cast<const uint8_t *>(codes) + m * (K / 2), act_table, count, K, a_values, s)) return rc;
    if (m == 0)
      if (int rc = decode_operands_int8(packed_w, w_table, N, K, w_values, s)) return rc;
    if (int rc = dense_gemm(MF_I8, a_values, w_values, token_norms != nullptr ? token_norms + m : nullptr, scale, row_norms, bias, bias_dtype, count, N, K,
                            static_cast<unsigned char *>(out) + m * N * dtype_size(out_dtype), out_dtype, nullptr, tile, s))
      return rc;
  }
  return OQ_OK;
}

int oq_packed_linear_group(const void *codes, int code_format, const float *token_norms, const float *act_centroids,
                           int a_bits, int count, const uint8_t *const *packed_w, const int *w_bits,
                           const uint16_t *const *row_norms, const float *const *w_centroids, const void *const *bias,
                           int bias_dtype, int64_t M, const int64_t *N, int64_t K, void *const *out, int out_dtype,
                           void *workspace, uint64_t workspace_bytes, void *stream) {
  if (count < 1 || count > 64) return fail(OQ_ERR_INVALID, "packed_linear_group: count=%d (1..64)", count);
  if (packed_w == nullptr || w_bits == nullptr || row_norms == nullptr || w_centroids == nullptr || N == nullptr || out == nullptr)
    return fail(OQ_ERR_INVALID, "packed_linear_group: null argument array");
  for (int i = 0; i < count; ++i)
    if (int rc = check_matmul_common("packed_linear_group", packed_w[i], w_bits[i], row_norms[i], w_centroids[i],
                                     bias != nullptr ? bias[i] : nullptr, bias_dtype, M, N[i], K, out[i], out_dtype))
      return rc;
  if (M == 0) return OQ_OK;
  if (codes == nullptr || act_centroids == nullptr) return fail(OQ_ERR_INVALID, "packed_linear_group: null codes/centroids");
  if (a_bits < 1 || a_bits > 8) return fail(OQ_ERR_INVALID, "packed_linear_group: a_bits=%d", a_bits);
  if (code_format != OQ_CODES_U8 && code_format != OQ_CODES_NIBBLE) return fail(OQ_ERR_INVALID, "packed_linear_group: code_format=%d", code_format);
  bool launched = false;
  if (int rc = gemv_group_dispatch(codes, code_format, token_norms, act_centroids, 1 << a_bits, count, packed_w, w_bits,
                                   row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, as_stream(stream),
                                   &launched))
    return rc;
  if (launched) return OQ_OK;
  for (int i = 0; i < count; ++i)
    if (int rc = packed_linear_impl(codes, code_format, token_norms, act_centroids, a_bits, packed_w[i], w_bits[i],
                                    row_norms[i], w_centroids[i], bias != nullptr ? bias[i] : nullptr, bias_dtype, M,
                                    N[i], K, out[i], out_dtype, nullptr, workspace, workspace_bytes, stream))
      return rc;
  return OQ_OK;
}

int oq_packed_linear_mapped(const void *codes, int code_format, const float *token_norms,
                            const float *act_centroids, int a_bits, const uint8_t *packed_w, int w_bits,
                            const uint16_t *row_norms, const float *w_centroids, const void *bias, int bias_dtype,
                            int64_t M, int64_t N, int64_t K, void *out, int out_dtype, const uint16_t *output_map,
                            void *workspace, uint64_t workspace_bytes, void *stream) {
  if (output_map == nullptr) return fail(OQ_ERR_INVALID, "packed_linear_mapped: output_map is null");
  return packed_linear_impl(codes, code_format, token_norms, act_centroids, a_bits, packed_w, w_bits, row_norms,
                            w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, output_map, workspace, workspace_bytes, stream);
}

int oq_quantized_linear(const void *x, int x_dtype, const uint16_t *input_map, int64_t M, int64_t K,
                        const int32_t *perm, const int8_t *signs, const float *boundaries,
                        const float *act_centroids, int a_bits, int64_t block, float eps, float inv_sqrt_block,
                        const void *rotate_plan, const uint8_t *packed_w, int w_bits, const uint16_t *row_norms, const float *w_centroids,
                        const void *bias, int bias_dtype, int64_t N, void *codes_scratch, float *norms_scratch,
                        void *out, int out_dtype, const uint16_t *output_map, void *workspace, uint64_t workspace_bytes,
                        void *stream) {
  if (int rc = check_matmul_common("quantized_linear", packed_w, w_bits, row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype)) return rc;
  if (M == 0) return OQ_OK;
  if (a_bits < 1 || a_bits > 8) return fail(OQ_ERR_INVALID, "quantized_linear: a_bits=%d", a_bits);
  if (act_centroids == nullptr) return fail(OQ_ERR_INVALID, "quantized_linear: null activation centroids");
  const int levels = 1 << a_bits;
  hipStream_t s = as_stream(stream);
  if (output_map != nullptr && (out_dtype == OQ_F32 || !aligned16(output_map)))
    return fail(OQ_ERR_INVALID, "quantized_linear: an output map needs a 16-bit output dtype and 16-byte alignment");
  if (aligned16(packed_w) && token_linear_supported(x_dtype, M, N, K, levels, w_bits, x, perm, signs)) {
    bool launched = false;
    const int rc = token_linear_dispatch(x, x_dtype, input_map, K, perm, signs, boundaries, act_centroids, levels, block,
                                         eps, inv_sqrt_block, rotate_plan, packed_w, w_bits, row_norms, w_centroids, bias,
                                         bias_dtype, N, out, out_dtype, output_map, s, &launched);
    if (rc != OQ_OK || launched) return rc;
  }
  if (codes_scratch == nullptr || norms_scratch == nullptr)
    return fail(OQ_ERR_INVALID, "quantized_linear: this shape takes two launches and needs the scratch buffers");
  const int fmt = (a_bits <= 4 && (K & 1) == 0) ? OQ_CODES_NIBBLE : OQ_CODES_U8;
  if (int rc = rotate_quantize_dispatch(x, x_dtype, M, K, perm, signs, boundaries, nullptr, levels, block, eps,
                                        inv_sqrt_block, codes_scratch, fmt, nullptr, OQ_VALUES_NONE, norms_scratch,
                                        input_map, rotate_plan, s))
    return rc;
  return packed_linear_impl(codes_scratch, fmt, norms_scratch, act_centroids, a_bits, packed_w, w_bits, row_norms,
                            w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, output_map, workspace, workspace_bytes, stream);
}

int oq_quantized_linear_group(const void *x, int x_dtype, const uint16_t *input_map, int64_t M, int64_t K,
                              const int32_t *perm, const int8_t *signs, const float *boundaries,
                              const float *act_centroids, int a_bits, int64_t block, float eps, float inv_sqrt_block,
                              const void *rotate_plan, int count, const uint8_t *const *packed_w, const int *w_bits,
                              const uint16_t *const *row_norms, const float *const *w_centroids, const void *const *bias,
                              int bias_dtype, const int64_t *N, void *codes_scratch, float *norms_scratch,
                              void *const *out, int out_dtype, void *workspace, uint64_t workspace_bytes, void *stream) {
  if (count < 1 || count > 64) return fail(OQ_ERR_INVALID, "quantized_linear_group: count=%d (1..64)", count);
  if (packed_w == nullptr || w_bits == nullptr || row_norms == nullptr || w_centroids == nullptr || N == nullptr || out == nullptr)
    return fail(OQ_ERR_INVALID, "quantized_linear_group: null argument array");
  for (int i = 0; i < count; ++i)
    if (int rc = check_matmul_common("quantized_linear_group", packed_w[i], w_bits[i], row_norms[i], w_centroids[i],
                                     bias != nullptr ? bias[i] : nullptr, bias_dtype, M, N[i], K, out[i], out_dtype))
      return rc;
  if (M == 0) return OQ_OK;
  if (a_bits < 1 || a_bits > 8) return fail(OQ_ERR_INVALID, "quantized_linear_group: a_bits=%d", a_bits);
  if (act_centroids == nullptr) return fail(OQ_ERR_INVALID, "quantized_linear_group: null activation centroids");
  const int levels = 1 << a_bits;
  hipStream_t s = as_stream(stream);
  if (codes_scratch == nullptr || norms_scratch == nullptr)
    return fail(OQ_ERR_INVALID, "quantized_linear_group: null scratch buffers");
  const int fmt = (a_bits <= 4 && (K & 1) == 0) ? OQ_CODES_NIBBLE : OQ_CODES_U8;
  if (int rc = rotate_quantize_dispatch(x, x_dtype, M, K, perm, signs, boundaries, nullptr, levels, block, eps,
                                        inv_sqrt_block, codes_scratch, fmt, nullptr, OQ_VALUES_NONE, norms_scratch,
                                        input_map, rotate_plan, s))
    return rc;
  return oq_packed_linear_group(codes_scratch, fmt, norms_scratch, act_centroids, a_bits, count, packed_w, w_bits,
                                row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, workspace, workspace_bytes,
                                stream);
}

int oq_quantized_linear_static(const void *x, int x_dtype, const uint16_t *input_map, int64_t M, int64_t K,
                               const int32_t *perm, const int8_t *signs, const float *boundaries,
                               const float *act_centroids, int a_bits, int64_t block, float eps, float inv_sqrt_block,
                               const void *rotate_plan, const uint8_t *packed_w, int w_bits, const uint16_t *row_norms,
                               const float *w_centroids, const void *bias, int bias_dtype, int64_t N, void *out,
                               int out_dtype, const uint16_t *output_map, void *stream) {
  if (M < 0 || K <= 0) return fail(OQ_ERR_INVALID, "quantized_linear_static: M=%lld K=%lld", (long long)M, (long long)K);
  // layout of the scratch: codes (nibble or byte per value) rounded up to 256 bytes, then the norms
  const bool nibble = a_bits <= 4 && (K & 1) == 0;
  const uint64_t codes_bytes = static_cast<uint64_t>(M) * static_cast<uint64_t>(nibble ? K / 2 : K);
  const uint64_t norms_at = (codes_bytes + 255u) & ~static_cast<uint64_t>(255);
  if (static_cast<uint64_t>(K) > (1u << 20) || norms_at + 4u * static_cast<uint64_t>(M) > kStaticScratchBytes)
    return fail(OQ_ERR_UNSUPPORTED,
                "quantized_linear_static: %lld tokens of %lld values need %llu bytes of scratch, the static buffer holds %zu; "
                "use oq_quantized_linear with caller-owned scratch",
                (long long)M, (long long)K, (unsigned long long)(norms_at + 4u * static_cast<uint64_t>(M)), kStaticScratchBytes);
  unsigned char *base = nullptr;
  if (int rc = static_scratch_address(&base)) return rc;
  // (no workspace: the launch shapes that need no buffer beyond the scratch)
  return oq_quantized_linear(x, x_dtype, input_map, M, K, perm, signs, boundaries, act_centroids, a_bits, block, eps,
                             inv_sqrt_block, rotate_plan, packed_w, w_bits, row_norms, w_centroids, bias, bias_dtype, N, base,
                             reinterpret_cast<float *>(base + norms_at), out, out_dtype, output_map, nullptr, 0, stream);
}

int oq_matmul_packed_weight(const void *x, int x_dtype, const float *token_scale, const uint8_t *packed_w,
                            int bits, const uint16_t *row_norms, const float *w_centroids, const void *bias,
                            int bias_dtype, int64_t M, int64_t N, int64_t K, void *out, int out_dtype,
                            void *workspace, uint64_t workspace_bytes, void *stream) {
  if (int rc = check_matmul_common("matmul_packed_weight", packed_w, bits, row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype)) return rc;
  if (M == 0) return OQ_OK;
  if (x == nullptr || !valid_dtype(x_dtype)) return fail(OQ_ERR_INVALID, "matmul_packed_weight: x / x_dtype");
  hipStream_t s = as_stream(stream);
  // bf16 activations take the tile kernel from two tokens on (one token on large matrices): measured against
  // the float-activation kernels below it is 3-4 times faster from 9 to 255 tokens (4096x4096 W4: 104 -> 28 us)
  // and up to 13 times at 2 to 8; only a single token on a small matrix is 2-3 us quicker on the
  // shape-agnostic kernel.  OQ_FLOAT_GEMM_MIN_M overrides, for measurements.
  int64_t tile_kernel_from = N * K >= (int64_t{32} << 20) ? 1 : 2;
  if (const char *v = debug_env(ENV_FLOAT_GEMM_MIN_M)) tile_kernel_from = atoi(v) > 1 ? atoi(v) : 1;
  if (x_dtype == OQ_BF16 && M >= tile_kernel_from && K % 64 == 0 && aligned16(x) && aligned16(packed_w) && gemm_output_ok(N, out) &&
      gemm_supported(K, bits)) {
    // Large M: the tile kernel of the code path on activation values.  Either one pass first puts the activations
    // into the matrix core's operand order (fastest on large problems; needs the caller's workspace), or every
    // wavefront stages its own rows through LDS (no buffer).
    const char *force = debug_env(ENV_GEMM_TILE);
    const bool force_staged = force != nullptr && force[0] != '\0' && force[1] == 's';
    if (!force_staged) {
      const int rc = gemm_tiled_dispatch(false, x, token_scale, packed_w, bits, row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype,
                                         workspace, workspace_bytes, s);
      if (rc >= 0) return rc;
    }
    if (M * K * 2 < (int64_t{1} << 32))
      return gemm_staged_dispatch(x, token_scale, packed_w, bits, row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype, s);
  }
  if (x_dtype != OQ_F32 && M > 8 && aligned16(x) && aligned16(packed_w) && gemm_output_ok(N, out) && gemm_av_supported(K, bits))
  {
    // fp16 with the caller's workspace: the same tile kernel in fp16 (512 x 12288 x 3072, W4: 118 -> 54 us;
    // up to eight tokens the shape-agnostic kernel keeps its fp32 centroids)
    if (x_dtype == OQ_F16) {
      const int rc = gemm_tiled_dispatch(true, x, token_scale, packed_w, bits, row_norms, w_centroids, bias, bias_dtype, M, N, K, out, out_dtype,
                                         workspace, workspace_bytes, s);
      if (rc >= 0) return rc;
    }
    // The float-activation kernel has its own (measured) preference: 256x256 tiles once there are
    // at least half as many of them as CUs, 128x128 tiles below that; OQ_GEMM_TILE still overrides.
    const int64_t big_tiles = ((M + 255) / 256) * ((N + 255) / 256);
    const int tile = debug_env(ENV_GEMM_TILE) != nullptr ? gemm_choose_tile(M, N, K, bits) : (big_tiles >= 128 ? 2 : 0);
    return gemm_av_dispatch(x_dtype == OQ_F16, x, token_scale, packed_w, bits, row_norms, w_centroids, bias, bias_dtype,
                            M, N, K, out, out_dtype, tile, s);
  }
  return generic_matmul_float(x, x_dtype, token_scale, packed_w, bits, row_norms, w_centroids, bias, bias_dtype, M, N,
                              K, out, out_dtype, s);
}

int oq_matmul_packed_adaln_int4(const uint16_t *x, const uint8_t *packed_weight, const uint16_t *scales,
                                const uint16_t *bias, int64_t M, int64_t N, int64_t K, int64_t group_size, uint16_t *out,
                                void *stream) {
  return adaln_int4_dispatch(x, packed_weight, scales, bias, M, N, K, group_size, out, as_stream(stream));
}

int oq_quantize_adaln_weight(const void *w, int w_dtype, int64_t N, int64_t K, int64_t group_size, uint8_t *packed_out,
                             float *scales_out, void *stream) {
  return adaln_quantize_dispatch(w, w_dtype, N, K, group_size, packed_out, scales_out, as_stream(stream));
}

int oq_unpack_lowbit(const uint8_t *packed, int bits, int64_t count, uint8_t *out, void *stream) {
  if (bits < 1 || bits > 8 || count < 0) return fail(OQ_ERR_INVALID, "unpack_lowbit: bits=%d count=%lld", bits, (long long)count);
  if (count > 0 && (packed == nullptr || out == nullptr)) return fail(OQ_ERR_INVALID, "unpack_lowbit: null pointer");
  return unpack_dispatch(packed, bits, count, out, as_stream(stream));
}

int oq_pack_lowbit(const uint8_t *values, int bits, int64_t count, uint8_t *packed_out, void *stream) {
  if (bits < 1 || bits > 8 || count < 0) return fail(OQ_ERR_INVALID, "pack_lowbit: bits=%d count=%lld", bits, (long long)count);
  if (count > 0 && (values == nullptr || packed_out == nullptr)) return fail(OQ_ERR_INVALID, "pack_lowbit: null pointer");
  return pack_lowbit_dispatch(values, bits, count, packed_out, as_stream(stream));
}

int oq_dequantize_packed_weight(const uint8_t *packed_weight, int bits, const uint16_t *row_norms, const float *centroids,
                                int64_t N, int64_t K, void *out, int out_dtype, void *stream) {
  if (bits < 1 || bits > 8 || N < 0 || K < 0) return fail(OQ_ERR_INVALID, "dequantize_packed_weight: bits=%d N=%lld K=%lld", bits, (long long)N, (long long)K);
  if (out_dtype != OQ_F32 && out_dtype != OQ_F16 && out_dtype != OQ_BF16) return fail(OQ_ERR_INVALID, "dequantize_packed_weight: out_dtype=%d", out_dtype);
  if (N > 0 && K > 0 && (packed_weight == nullptr || row_norms == nullptr || centroids == nullptr || out == nullptr))
    return fail(OQ_ERR_INVALID, "dequantize_packed_weight: null pointer");
  return dequantize_dispatch(packed_weight, bits, row_norms, centroids, N, K, out, out_dtype, as_stream(stream));
}

// ---- the 4-bit key/value cache ----

namespace {
int log2_exact(int64_t v) { return v > 0 && (v & (v - 1)) == 0 ? __builtin_ctzll(static_cast<unsigned long long>(v)) : -1; }
bool aligned(const void *p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool known_dtype(int dt) { return dt == OQ_F32 || dt == OQ_F16 || dt == OQ_BF16; }
bool known_head_dim(int64_t d) { return d == 64 || d == 128 || d == 256; }
int page_shift_of(int64_t page_size) { return page_size < oq::kKvMinPage || page_size > oq::kKvMaxPage ? -1 : log2_exact(page_size); }

// The cache as the kernels take it; an error status where it is none.
int kv_cache_of(const char *what, const oq_kv_cache *c, oq::KvCache &out) {
  if (c == nullptr) return fail(OQ_ERR_INVALID, "%s: no cache", what);
  if (!known_head_dim(c->head_dim)) return fail(OQ_ERR_UNSUPPORTED, "%s: head_dim=%lld (64, 128 or 256)", what, (long long)c->head_dim);
  const int shift = page_shift_of(c->page_size);
  if (shift < 0) return fail(OQ_ERR_UNSUPPORTED, "%s: page_size=%lld (a power of two, 16 to 1024)", what, (long long)c->page_size);
  if (c->pages < 1 || c->pages > 0x7fffffffLL || c->kv_heads < 1 || c->kv_heads > 65535)
    return fail(OQ_ERR_INVALID, "%s: pages=%lld kv_heads=%lld", what, (long long)c->pages, (long long)c->kv_heads);
  if (c->k_codes == nullptr || c->k_scales == nullptr || c->v_codes == nullptr || c->v_scales == nullptr || c->signs == nullptr)
    return fail(OQ_ERR_INVALID, "%s: null pointer in the cache", what);
  if (!aligned(c->k_codes, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_codes, 16) || !aligned(c->v_scales, 16) || !aligned(c->signs, 16))
    return fail(OQ_ERR_INVALID, "%s: the cache is not aligned to 16 bytes", what);
  out.k_codes = c->k_codes; out.v_codes = c->v_codes; out.k_scales = c->k_scales; out.v_scales = c->v_scales; out.signs = c->signs;
  out.pages = c->pages; out.heads = static_cast<int>(c->kv_heads); out.page_shift = shift;
  return OQ_OK;
}

bool vectors_wide(const void *p, int64_t token_stride, int64_t head_stride, int dtype) {
  const int64_t per = 16 / oq::dtype_size(dtype);
  return aligned(p, 16) && token_stride % per == 0 && head_stride % per == 0;
}

// Write and read: a launch of `threads` for every head of sixteen tokens.
int kv_vectors_fit(const char *what, int64_t tokens, const oq_kv_cache *c, int threads) {
  if (tokens < 0) return fail(OQ_ERR_INVALID, "%s: tokens=%lld", what, (long long)tokens);
  if (tokens > (1LL << 40) || (tokens + oq::kKvGroup - 1) / oq::kKvGroup * c->kv_heads > oq::kKvMostThreads / threads)
    return fail(OQ_ERR_UNSUPPORTED, "%s: tokens=%lld kv_heads=%lld exceed the grid", what, (long long)tokens, (long long)c->kv_heads);
  return OQ_OK;
}

int kv_attend_shape(oq::KvAttendArgs &a, int64_t tokens, int64_t heads, int64_t table_width, int64_t requests, int64_t window) {
  const int64_t kv_heads = a.cache.heads;
  if (tokens < 0 || heads < 1 || heads % kv_heads != 0 || requests < 0 || table_width < 0 || window < 0)
    return fail(OQ_ERR_INVALID, "kv_attend: tokens=%lld heads=%lld kv_heads=%lld requests=%lld table_width=%lld window=%lld", (long long)tokens,
                (long long)heads, (long long)kv_heads, (long long)requests, (long long)table_width, (long long)window);
  if (tokens > 0x3fffffffLL || requests > 0x3fffffffLL || heads > 65535 || tokens * heads > 0x7fffffffLL ||
      (tokens * heads + (requests + 2) * kv_heads * (heads / kv_heads / 16 + 4)) > 0x7fffffffLL || table_width > (1LL << 30) >> a.cache.page_shift)
    return fail(OQ_ERR_UNSUPPORTED, "kv_attend: tokens=%lld heads=%lld requests=%lld table_width=%lld exceed the grid", (long long)tokens,
                (long long)heads, (long long)requests, (long long)table_width);
  a.tokens = tokens; a.heads = static_cast<int>(heads); a.group = static_cast<int>(heads / kv_heads); a.requests = static_cast<int>(requests);
  a.table_width = static_cast<int>(table_width); a.window = static_cast<int>(window < 0x7fffffffLL ? window : 0x7fffffffLL);
  return OQ_OK;
}

int64_t most_queries(int64_t tokens, bool has_starts, int64_t max_new) { return !has_starts ? 1 : max_new >= 1 && max_new < tokens ? max_new : tokens; }
}  // namespace

int oq_kv_assign(const int32_t *lengths, const int32_t *new_lengths, int64_t requests, int32_t *table, int64_t table_stride,
                 int64_t table_width, const int32_t *free_pages, int64_t free_count, const int32_t *taken, int64_t page_size,
                 int64_t tokens, int64_t *slots, int32_t *positions, int32_t *starts, int32_t *lengths_after, int32_t *taken_after,
                 void *stream) {
  const int shift = page_shift_of(page_size);
  if (shift < 0) return fail(OQ_ERR_UNSUPPORTED, "kv_assign: page_size=%lld (a power of two, 16 to 1024)", (long long)page_size);
  if (requests < 0 || tokens < 0 || table_width < 0 || free_count < 0 || (requests > 1 && table_stride < table_width))
    return fail(OQ_ERR_INVALID, "kv_assign: requests=%lld tokens=%lld table_width=%lld table_stride=%lld free_count=%lld", (long long)requests,
                (long long)tokens, (long long)table_width, (long long)table_stride, (long long)free_count);
  if (requests > oq::kKvMaxRequests || tokens > 0x7fffffffLL || table_width > 0x7fffffffLL || free_count > 0x7fffffffLL)
    return fail(OQ_ERR_UNSUPPORTED, "kv_assign: requests=%lld (at most %d) tokens=%lld", (long long)requests, oq::kKvMaxRequests, (long long)tokens);
  if ((requests > 0 && (lengths == nullptr || new_lengths == nullptr || lengths_after == nullptr)) ||
      (requests > 0 && table_width > 0 && table == nullptr) || (free_count > 0 && free_pages == nullptr) || taken == nullptr ||
      (tokens > 0 && (slots == nullptr || positions == nullptr)) || starts == nullptr || taken_after == nullptr)
    return fail(OQ_ERR_INVALID, "kv_assign: null pointer");
  oq::KvAssignArgs a{};
  a.lengths = lengths; a.new_lengths = new_lengths; a.free_pages = free_pages; a.taken = taken; a.table = table; a.table_stride = table_stride;
  a.table_width = static_cast<int>(table_width); a.requests = static_cast<int>(requests); a.free_count = static_cast<int>(free_count);
  a.page_shift = shift; a.tokens = tokens; a.slots = slots; a.positions = positions; a.starts = starts; a.lengths_after = lengths_after;
  a.taken_after = taken_after;
  return oq::kv_assign_dispatch(a, as_stream(stream));
}

int oq_kv_write(const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride,
                int dtype, const int64_t *slots, int64_t tokens, const oq_kv_cache *cache, void *stream) {
  oq::KvWriteArgs a{};
  if (const int status = kv_cache_of("kv_write", cache, a.cache)) return status;
  if (!known_dtype(dtype)) return fail(OQ_ERR_INVALID, "kv_write: dtype=%d", dtype);
  if (const int status = kv_vectors_fit("kv_write", tokens, cache, oq::kv_write_threads(cache->head_dim))) return status;
  if (tokens == 0) return OQ_OK;
  if (k == nullptr || v == nullptr || slots == nullptr) return fail(OQ_ERR_INVALID, "kv_write: null pointer");
  a.k = k; a.v = v; a.slots = slots; a.tokens = tokens;
  a.k_token_stride = k_token_stride; a.k_head_stride = k_head_stride; a.v_token_stride = v_token_stride; a.v_head_stride = v_head_stride;
  a.k_wide = vectors_wide(k, k_token_stride, k_head_stride, dtype);
  a.v_wide = vectors_wide(v, v_token_stride, v_head_stride, dtype);
  return oq::kv_write_dispatch(a, static_cast<int>(cache->head_dim), dtype, as_stream(stream));
}

int oq_kv_read(const int64_t *slots, int64_t tokens, const oq_kv_cache *cache, void *k, void *v, int dtype, void *stream) {
  oq::KvReadArgs a{};
  if (const int status = kv_cache_of("kv_read", cache, a.cache)) return status;
  if (!known_dtype(dtype)) return fail(OQ_ERR_INVALID, "kv_read: dtype=%d", dtype);
  if (const int status = kv_vectors_fit("kv_read", tokens, cache, oq::kv_read_threads(cache->head_dim))) return status;
  if (tokens == 0) return OQ_OK;
  if (k == nullptr || v == nullptr || slots == nullptr) return fail(OQ_ERR_INVALID, "kv_read: null pointer");
  if (!aligned(k, 16) || !aligned(v, 16)) return fail(OQ_ERR_INVALID, "kv_read: the outputs are not aligned to 16 bytes");
  a.slots = slots; a.k = k; a.v = v; a.tokens = tokens;
  return oq::kv_read_dispatch(a, static_cast<int>(cache->head_dim), dtype, as_stream(stream));
}

namespace {
int attend(const void *q, int q_dtype, int64_t tokens, int64_t heads, int64_t q_token_stride, int64_t q_head_stride, const oq_kv_cache *cache,
           const int32_t *table, int64_t table_stride, int64_t table_width, const int32_t *lengths, const int32_t *starts, int64_t requests, int causal,
           const uint64_t *masks, int mask_words, int64_t window, float scale, int64_t max_length, int64_t max_new, void *out, float *lse,
           void *workspace, uint64_t workspace_bytes, void *stream) {
  oq::KvAttendArgs a{};
  if (const int status = kv_cache_of("kv_attend", cache, a.cache)) return status;
  if (!known_dtype(q_dtype)) return fail(OQ_ERR_INVALID, "kv_attend: q_dtype=%d", q_dtype);
  if (const int status = kv_attend_shape(a, tokens, heads, table_width, requests, window)) return status;
  if (starts == nullptr && tokens != requests) return fail(OQ_ERR_INVALID, "kv_attend: tokens=%lld requests=%lld and no starts", (long long)tokens, (long long)requests);
  if (window > 0 && !causal) return fail(OQ_ERR_INVALID, "kv_attend: a window needs causal attention");
  if (requests > 1 && table_stride < table_width) return fail(OQ_ERR_INVALID, "kv_attend: table_stride=%lld table_width=%lld", (long long)table_stride, (long long)table_width);
  if (tokens == 0) return OQ_OK;
  if (q == nullptr || out == nullptr || (requests > 0 && lengths == nullptr) || (requests > 0 && table_width > 0 && table == nullptr))
    return fail(OQ_ERR_INVALID, "kv_attend: null pointer");
  if (!aligned(out, 16) || !aligned(workspace, 16)) return fail(OQ_ERR_INVALID, "kv_attend: the output or the workspace is not aligned to 16 bytes");
  const int dim = static_cast<int>(cache->head_dim);
  a.q = q; a.q_dtype = q_dtype; a.q_token_stride = q_token_stride; a.q_head_stride = q_head_stride;
  a.q_wide = vectors_wide(q, q_token_stride, q_head_stride, q_dtype);
  a.table = table; a.table_stride = table_stride; a.lengths = lengths; a.starts = starts; a.causal = causal != 0; a.scale = scale;
  a.masks = masks; a.mask_words = mask_words;
  a.out = out; a.lse = lse;
  const uint64_t needed = oq::kv_attend_plan(a, dim, max_length, most_queries(tokens, starts != nullptr, max_new), workspace);
  if (!oq::kv_attend_fits(a, dim)) return fail(OQ_ERR_UNSUPPORTED, "kv_attend: tokens=%lld heads=%lld requests=%lld exceed the grid", (long long)tokens, (long long)heads, (long long)requests);
  if (workspace == nullptr || workspace_bytes < needed) a.few.target = a.many.target = 0;
  return oq::kv_attend_dispatch(a, dim, as_stream(stream));
}
}  // namespace

int oq_kv_attend(const void *q, int q_dtype, int64_t tokens, int64_t heads, int64_t q_token_stride, int64_t q_head_stride,
                 const oq_kv_cache *cache, const int32_t *table, int64_t table_stride, int64_t table_width, const int32_t *lengths,
                 const int32_t *starts, int64_t requests, int causal, int64_t window, float scale, int64_t max_length, int64_t max_new,
                 void *out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream) {
  return attend(q, q_dtype, tokens, heads, q_token_stride, q_head_stride, cache, table, table_stride, table_width, lengths, starts, requests, causal, nullptr, 0,
                window, scale, max_length, max_new, out, lse, workspace, workspace_bytes, stream);
}

int oq_kv_attend_tree(const void *q, int q_dtype, int64_t tokens, int64_t heads, int64_t q_token_stride, int64_t q_head_stride,
                      const oq_kv_cache *cache, const int32_t *table, int64_t table_stride, int64_t table_width, const int32_t *lengths,
                      const int32_t *starts, int64_t requests, const uint64_t *masks, int64_t mask_words, int64_t window, float scale,
                      int64_t max_length, int64_t max_new, void *out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream) {
  if (mask_words < 1) return fail(OQ_ERR_INVALID, "kv_attend_tree: mask_words=%lld", (long long)mask_words);
  if (mask_words > oq::kKvMaskWords) return fail(OQ_ERR_UNSUPPORTED, "kv_attend_tree: mask_words=%lld (at most %d)", (long long)mask_words, oq::kKvMaskWords);
  if (tokens > 0 && (masks == nullptr || !aligned(masks, 8))) return fail(OQ_ERR_INVALID, "kv_attend_tree: no masks, or not aligned to 8 bytes");
  return attend(q, q_dtype, tokens, heads, q_token_stride, q_head_stride, cache, table, table_stride, table_width, lengths, starts, requests, 1, masks,
                static_cast<int>(mask_words), window, scale, max_length, max_new, out, lse, workspace, workspace_bytes, stream);
}

namespace {
uint64_t attend_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size, int64_t table_width, int64_t requests,
                                int has_starts, int q_dtype, int64_t mask_words, int64_t window, int64_t max_length, int64_t max_new) {
  static const int32_t some = 0;
  static const uint64_t mask = 0;
  oq::KvAttendArgs a{};
  a.q_dtype = q_dtype;
  a.masks = mask_words > 0 ? &mask : nullptr;  // (as the starts)
  a.mask_words = static_cast<int>(mask_words);
  a.cache.page_shift = page_shift_of(page_size);
  if (a.cache.page_shift < 0 || !known_head_dim(head_dim) || kv_heads < 1 || kv_heads > 65535) return 0;
  a.cache.heads = static_cast<int>(kv_heads);
  if (kv_attend_shape(a, tokens, heads, table_width, requests, window) != OQ_OK || tokens == 0) return 0;
  a.starts = has_starts ? &some : nullptr;  // (asked whether it is there, not read)
  const uint64_t bytes = oq::kv_attend_plan(a, static_cast<int>(head_dim), max_length, most_queries(tokens, has_starts != 0, max_new), nullptr);
  return oq::kv_attend_fits(a, static_cast<int>(head_dim)) ? bytes : 0;
}
}  // namespace

uint64_t oq_kv_attend_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                      int64_t table_width, int64_t requests, int has_starts, int64_t window, int64_t max_length,
                                      int64_t max_new) {
  return attend_workspace_bytes(tokens, heads, kv_heads, head_dim, page_size, table_width, requests, has_starts, OQ_F32, 0, window, max_length, max_new);
}

uint64_t oq_kv_attend_tree_workspace_bytes(int q_dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                                           int64_t table_width, int64_t requests, int has_starts, int64_t mask_words, int64_t window,
                                           int64_t max_length, int64_t max_new) {
  if (!known_dtype(q_dtype) || mask_words < 1 || mask_words > oq::kKvMaskWords) return 0;
  return attend_workspace_bytes(tokens, heads, kv_heads, head_dim, page_size, table_width, requests, has_starts, q_dtype, mask_words, window, max_length, max_new);
}

// ---- norms and rotary positions ----

namespace {
// No more values at once than 16 bytes hold of the smaller type, or 8, where these vectors begin.
void qk_fit_piece(oq::QkNormRotary &how, const void *x, int64_t token_stride, int64_t head_stride, int dtype) {
  for (; how.piece > 1; how.piece = how.piece == 8 ? 4 : 1) {
    const int bytes = how.piece * oq::dtype_size(dtype) < 16 ? how.piece * oq::dtype_size(dtype) : 16, per = bytes / oq::dtype_size(dtype);
    if (aligned(x, bytes) && token_stride % per == 0 && head_stride % per == 0) return;
  }
}

// How the pairs of heads of `dim` are normed and turned; an error status where the plan is none.
int qk_plan_of(const char *what, const oq_qk_norm_rotary_plan *p, int64_t dim, oq::QkNormRotary &how) {
  if (p == nullptr) return fail(OQ_ERR_INVALID, "%s: no plan", what);
  if ((p->cos == nullptr) != (p->sin == nullptr)) return fail(OQ_ERR_INVALID, "%s: cosines and sines go together", what);
  const int64_t rotary = p->cos != nullptr ? p->rotary_dim : 0;
  if (p->cos != nullptr && (rotary < 2 || rotary % 2 != 0 || rotary > dim || p->rows < 0))
    return fail(OQ_ERR_INVALID, "%s: rotary_dim=%lld (even, 2 to %lld) rows=%lld", what, (long long)p->rotary_dim, (long long)dim, (long long)p->rows);
  if (p->rows > 0x7fffffffLL) return fail(OQ_ERR_UNSUPPORTED, "%s: rows=%lld", what, (long long)p->rows);
  if (!aligned(p->cos, 4) || !aligned(p->sin, 4)) return fail(OQ_ERR_INVALID, "%s: the tables are not aligned to their entries", what);
  if (p->norm == 0 && (p->q_weight != nullptr || p->k_weight != nullptr)) return fail(OQ_ERR_INVALID, "%s: weights without a norm", what);
  if ((p->q_weight != nullptr || p->k_weight != nullptr) && !known_dtype(p->weight_dtype)) return fail(OQ_ERR_INVALID, "%s: weight_dtype=%d", what, p->weight_dtype);
  if (p->norm != 0 && !(p->eps >= 0.0f && p->eps <= 3.402823466e38f)) return fail(OQ_ERR_INVALID, "%s: eps=%g", what, p->eps);
  how.cos = p->cos; how.sin = p->sin; how.positions = p->positions; how.rows = p->rows;
  how.half = static_cast<int>(rotary / 2);
  how.table_wide = how.half % 8 == 0 && aligned(p->cos, 16) && aligned(p->sin, 16);
  how.weight[0] = p->q_weight; how.weight[1] = p->k_weight; how.weight_dtype = p->weight_dtype;
  how.norm = p->norm != 0; how.interleaved = p->interleaved != 0; how.eps = p->eps; how.by_dim = static_cast<float>(1.0 / static_cast<double>(dim));
  // Eight values at once where a head's parts are multiples of eight pairs, four where they are of four; the vectors' alignment has its say below.
  how.piece = dim % 16 == 0 && (how.interleaved || how.half % 8 == 0) ? 8 : dim % 8 == 0 && (how.interleaved || how.half % 4 == 0) ? 4 : 1;
  qk_fit_piece(how, p->q_weight, 0, 0, p->weight_dtype);
  qk_fit_piece(how, p->k_weight, 0, 0, p->weight_dtype);
  return OQ_OK;
}

// One side's tensors, and the workgroups of `threads` that they take.
int qk_side_of(const char *what, const void *x, int64_t token_stride, int64_t head_stride, int64_t heads, int dtype, int64_t tokens, int64_t dim,
               oq::QkNormRotary &how, void *out, int threads, oq::QkSide &side, uint32_t &blocks) {
  if (tokens < 0 || heads < 1 || heads > 65535) return fail(OQ_ERR_INVALID, "%s: tokens=%lld heads=%lld", what, (long long)tokens, (long long)heads);
  if (tokens > 0x3fffffffLL || tokens * heads > 0x3fffffffLL) return fail(OQ_ERR_UNSUPPORTED, "%s: tokens=%lld heads=%lld exceed the grid", what, (long long)tokens, (long long)heads);
  if (tokens > 0 && (x == nullptr || out == nullptr)) return fail(OQ_ERR_INVALID, "%s: null pointer", what);
  if (!aligned(out, 16)) return fail(OQ_ERR_INVALID, "%s: the outputs are not aligned to 16 bytes", what);
  side.x = x; side.out = out; side.token_stride = token_stride; side.head_stride = head_stride;
  side.heads = static_cast<int>(heads); side.each = tokens * heads <= oq::kQkAlone ? 1 : oq::kQkHeads;
  side.groups = (side.heads + side.each - 1) / side.each;
  side.magic = static_cast<uint32_t>(((1ull << 32) + side.groups - 1) / side.groups);
  qk_fit_piece(how, x, token_stride, head_stride, dtype);
  const int64_t count = oq::qk_blocks(tokens, side.groups, static_cast<int>(dim), threads);
  if (count > oq::kKvMostThreads / threads / 2) return fail(OQ_ERR_UNSUPPORTED, "%s: tokens=%lld heads=%lld exceed the grid", what, (long long)tokens, (long long)heads);
  blocks = static_cast<uint32_t>(count);
  return OQ_OK;
}
}  // namespace

int oq_qk_norm_rotary(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t heads, const void *k, int64_t k_token_stride,
                      int64_t k_head_stride, int64_t kv_heads, int dtype, int64_t tokens, int64_t head_dim, const oq_qk_norm_rotary_plan *plan,
                      void *q_out, void *k_out, void *stream) {
  oq::QkArgs a{};
  if (!known_dtype(dtype)) return fail(OQ_ERR_INVALID, "qk_norm_rotary: dtype=%d", dtype);
  if (head_dim < 2 || head_dim % 2 != 0) return fail(OQ_ERR_INVALID, "qk_norm_rotary: head_dim=%lld (even)", (long long)head_dim);
  if (head_dim > oq::kQkMostDim) return fail(OQ_ERR_UNSUPPORTED, "qk_norm_rotary: head_dim=%lld (at most %d)", (long long)head_dim, oq::kQkMostDim);
  if (const int status = qk_plan_of("qk_norm_rotary", plan, head_dim, a.how)) return status;
  if (const int status = qk_side_of("qk_norm_rotary", q, q_token_stride, q_head_stride, heads, dtype, tokens, head_dim, a.how, q_out, oq::kQkThreads, a.side[0], a.q_blocks)) return status;
  if (const int status = qk_side_of("qk_norm_rotary", k, k_token_stride, k_head_stride, kv_heads, dtype, tokens, head_dim, a.how, k_out, oq::kQkThreads, a.side[1], a.k_blocks)) return status;
  if (tokens == 0) return OQ_OK;
  a.tokens = tokens;
  a.dim = static_cast<int>(head_dim);
  return oq::qk_norm_rotary_dispatch(a, dtype, as_stream(stream));
}

int oq_kv_append(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t heads, const void *k, int64_t k_token_stride,
                 int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride, int dtype, const int64_t *slots,
                 int64_t tokens, const oq_qk_norm_rotary_plan *plan, const oq_kv_cache *cache, void *q_out, void *stream) {
  oq::KvAppendArgs a{};
  if (const int status = kv_cache_of("kv_append", cache, a.write.cache)) return status;
  if (!known_dtype(dtype)) return fail(OQ_ERR_INVALID, "kv_append: dtype=%d", dtype);
  const int threads = oq::kv_write_threads(cache->head_dim);
  if (const int status = kv_vectors_fit("kv_append", tokens, cache, 2 * threads)) return status;
  if (const int status = qk_plan_of("kv_append", plan, cache->head_dim, a.how)) return status;
  if (const int status = qk_side_of("kv_append", q, q_token_stride, q_head_stride, heads, dtype, tokens, cache->head_dim, a.how, q_out, threads, a.q, a.q_blocks)) return status;
  if (tokens == 0) return OQ_OK;
  if (k == nullptr || v == nullptr || slots == nullptr) return fail(OQ_ERR_INVALID, "kv_append: null pointer");
  oq::KvWriteArgs &w = a.write;
  w.k = k; w.v = v; w.slots = slots; w.tokens = tokens;
  w.k_token_stride = k_token_stride; w.k_head_stride = k_head_stride; w.v_token_stride = v_token_stride; w.v_head_stride = v_head_stride;
  qk_fit_piece(a.how, k, k_token_stride, k_head_stride, dtype);
  w.v_wide = vectors_wide(v, v_token_stride, v_head_stride, dtype);
  a.kv_blocks = static_cast<uint32_t>((tokens + oq::kKvGroup - 1) / oq::kKvGroup * cache->kv_heads);
  return oq::kv_append_dispatch(a, static_cast<int>(cache->head_dim), dtype, as_stream(stream));
}

// ---- trees of drafted tokens ----

int oq_kv_tree(const int32_t *parents, const int32_t *starts, const int32_t *lengths, int64_t requests, int64_t tokens, int64_t mask_words,
               int32_t *positions, uint64_t *masks, void *stream) {
  if (requests < 0 || tokens < 0 || mask_words < 1)
    return fail(OQ_ERR_INVALID, "kv_tree: requests=%lld tokens=%lld mask_words=%lld", (long long)requests, (long long)tokens, (long long)mask_words);
  if (mask_words > oq::kKvMaskWords || requests > 0xffffff || tokens > 0x3fffffffLL)
    return fail(OQ_ERR_UNSUPPORTED, "kv_tree: requests=%lld tokens=%lld mask_words=%lld (at most %d)", (long long)requests, (long long)tokens, (long long)mask_words, oq::kKvMaskWords);
  if (tokens == 0) return OQ_OK;
  if (parents == nullptr || starts == nullptr || (requests > 0 && lengths == nullptr) || positions == nullptr || masks == nullptr)
    return fail(OQ_ERR_INVALID, "kv_tree: null pointer");
  if (!aligned(masks, 8)) return fail(OQ_ERR_INVALID, "kv_tree: the masks are not aligned to 8 bytes");
  return oq::kv_tree_dispatch({parents, starts, lengths, static_cast<int>(requests), static_cast<int>(mask_words), tokens, positions, masks}, as_stream(stream));
}

namespace {
// No two parts of the caches may share memory: two wavefronts would move the same entries, one of them what the other has moved already.  Parts sorted by where they
// begin, four a cache (eight caches 1 us of the host, 64, which one launch takes, 6).
int keep_caches_apart(const oq_kv_cache *caches, int64_t count) {
  struct Part {
    uintptr_t begin, end;
    int64_t cache;
  };
  Part few[4 * 16];
  const std::unique_ptr<Part[]> many(count > 16 ? new (std::nothrow) Part[4 * count] : nullptr);
  Part *const parts = count > 16 ? many.get() : few;
  if (parts == nullptr) return fail(OQ_ERR_UNSUPPORTED, "kv_keep: no memory to look %lld caches over", (long long)count);
  const uint64_t vectors = static_cast<uint64_t>(caches->pages) * caches->kv_heads * caches->page_size, codes = vectors * (caches->head_dim / 2), scales = vectors * 2;
  for (int64_t i = 0; i < count; ++i) {
    const auto put = [&](int part, const void *p, uint64_t bytes) { parts[4 * i + part] = {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, i}; };
    put(0, caches[i].k_codes, codes);
    put(1, caches[i].v_codes, codes);
    put(2, caches[i].k_scales, scales);
    put(3, caches[i].v_scales, scales);
  }
  std::sort(parts, parts + 4 * count, [](const Part &a, const Part &b) { return a.begin < b.begin; });
  for (int64_t i = 1; i < 4 * count; ++i) {  // (in front of the first that overlaps, each begins behind the one before)
    if (parts[i].begin >= parts[i - 1].end) continue;
    for (int64_t a = 1; a < count; ++a) {
      for (int64_t b = 0; b < a; ++b) {
        if (caches[a].k_codes == caches[b].k_codes) return fail(OQ_ERR_INVALID, "kv_keep: cache %lld is cache %lld again", (long long)a, (long long)b);
      }
    }
    return fail(OQ_ERR_INVALID, "kv_keep: parts of cache %lld and cache %lld share memory", (long long)parts[i - 1].cache, (long long)parts[i].cache);
  }
  return OQ_OK;
}
}  // namespace

int oq_kv_keep(const int32_t *kept, int64_t most, const int32_t *lengths, const int32_t *starts, const int64_t *slots, int64_t requests, int64_t tokens,
               const oq_kv_cache *caches, int64_t cache_count, const int32_t *table, int64_t table_stride, int64_t table_width, int32_t *free_pages,
               int64_t free_count, const int32_t *taken, int32_t *lengths_after, int32_t *taken_after, void *stream) {
  if (most < 0 || requests < 0 || tokens < 0 || cache_count < 1 || table_width < 0 || free_count < 0 || (table != nullptr && requests > 1 && table_stride < table_width))
    return fail(OQ_ERR_INVALID, "kv_keep: most=%lld requests=%lld tokens=%lld caches=%lld table_width=%lld table_stride=%lld free_count=%lld", (long long)most,
                (long long)requests, (long long)tokens, (long long)cache_count, (long long)table_width, (long long)table_stride, (long long)free_count);
  if (caches == nullptr) return fail(OQ_ERR_INVALID, "kv_keep: no cache");
  oq::KvCache first{}, other{};
  if (const int status = kv_cache_of("kv_keep", caches, first)) return status;
  for (int64_t i = 1; i < cache_count; ++i) {
    if (const int status = kv_cache_of("kv_keep", caches + i, other)) return status;
    if (other.pages != first.pages || other.heads != first.heads || other.page_shift != first.page_shift || caches[i].head_dim != caches[0].head_dim)
      return fail(OQ_ERR_INVALID, "kv_keep: cache %lld is of another shape than the first", (long long)i);
  }
  if (most > oq::kKvMostKept || requests > oq::kKvMaxRequests || tokens > 0x3fffffffLL || table_width > 0x7fffffffLL || free_count > 0x7fffffffLL)
    return fail(OQ_ERR_UNSUPPORTED, "kv_keep: most=%lld (at most %d) requests=%lld (at most %d) tokens=%lld", (long long)most, oq::kKvMostKept, (long long)requests,
                oq::kKvMaxRequests, (long long)tokens);
  const bool pages = taken != nullptr;
  if (pages != (taken_after != nullptr) || (pages ? requests > 0 && table_width > 0 && table == nullptr : table != nullptr) || (free_count > 0 && free_pages == nullptr))
    return fail(OQ_ERR_INVALID, "kv_keep: block table, free pages and their count go together");
  if (requests == 0 && !pages) return OQ_OK;
  if ((requests > 0 && (lengths == nullptr || starts == nullptr || lengths_after == nullptr || (most > 0 && kept == nullptr))) || (tokens > 0 && slots == nullptr))
    return fail(OQ_ERR_INVALID, "kv_keep: null pointer");
  if (requests > 0) {
    if (const int status = keep_caches_apart(caches, cache_count)) return status;
  }
  oq::KvKeepArgs a{};
  a.kept = kept; a.lengths = lengths; a.starts = starts; a.slots = slots; a.tokens = tokens; a.pages = first.pages; a.table_stride = table_stride;
  a.requests = static_cast<int>(requests); a.most = static_cast<int>(most); a.heads = first.heads; a.page_shift = first.page_shift;
  a.table_width = static_cast<int>(table_width); a.free_count = static_cast<int>(free_count);
  a.table = table; a.taken = taken; a.free_pages = free_pages; a.lengths_after = lengths_after; a.taken_after = taken_after;
  for (int64_t at = 0; at < cache_count; at += oq::kKvKeepCaches) {
    a.counts = at == 0;
    a.caches = static_cast<int>(cache_count - at < oq::kKvKeepCaches ? cache_count - at : oq::kKvKeepCaches);
    for (int i = 0; i < a.caches; ++i) a.cache[i] = {caches[at + i].k_codes, caches[at + i].v_codes, caches[at + i].k_scales, caches[at + i].v_scales};
    if (oq::kv_keep_blocks(a) == 0) break;  // (no requests: the first launch has made the counts)
    if (oq::kv_keep_blocks(a) > oq::kKvMostThreads / 256) return fail(OQ_ERR_UNSUPPORTED, "kv_keep: requests=%lld kv_heads=%d exceed the grid", (long long)requests, a.heads);
    if (const int status = oq::kv_keep_dispatch(a, static_cast<int>(caches->head_dim), as_stream(stream))) return status;
  }
  return OQ_OK;
}

}  // extern "C"
