/*
 * orbitquant_hip.h - C ABI of the MI355X (gfx950) quantized-linear forward.
 *
 * One shared library, plain pointers and sizes, no framework types.  Every
 * pointer is a DEVICE pointer unless a comment says otherwise; the library
 * borrows them for the duration of the call and keeps nothing.  Work is
 * enqueued on `stream` (a hipStream_t passed as void*; NULL = the null stream)
 * and the call returns without synchronizing, so calls may be captured into a
 * HIP graph.  Return value: OQ_OK or an oq_status error; `oq_last_error()`
 * gives the text of the last error raised on the calling thread.
 *
 * The entry points replace, for AMD GPUs, the operators the reference's native
 * package registers (paths relative to the reference checkout):
 *   native-kernels/orbitquant-packed-matmul/torch-ext/torch_binding.cpp:7-66
 *   native-kernels/orbitquant-packed-matmul/torch-ext/torch_binding.h:11-92
 * and the kernels behind them in
 *   native-kernels/orbitquant-packed-matmul/orbitquant_packed_matmul_cuda/packed_matmul.cu
 */
#ifndef ORBITQUANT_HIP_H
#define ORBITQUANT_HIP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
  OQ_OK = 0,
  OQ_ERR_INVALID = 1,     /* an argument is out of its documented range        */
  OQ_ERR_UNSUPPORTED = 2, /* valid request this build has no kernel for        */
  OQ_ERR_LAUNCH = 3       /* the HIP runtime rejected a launch / attribute set */
} oq_status;

typedef enum { OQ_F32 = 0, OQ_F16 = 1, OQ_BF16 = 2 } oq_dtype;

/* How activation codes are stored. */
typedef enum {
  OQ_CODES_U8 = 0,    /* one code per byte, [M, K]                                   */
  OQ_CODES_NIBBLE = 1 /* two codes per byte, even k in the low nibble, [M, K/2];     */
                      /* needs levels <= 16 and even K (packed_matmul.cu:648-656)    */
} oq_code_format;

/* What oq_rotate_quantize writes to `values_out`. */
typedef enum {
  OQ_VALUES_NONE = 0,
  OQ_VALUES_SCALED = 1,  /* centroid[code] * ||x||, rounded to x's dtype, [M, K]     */
                         /* (quantize_activations_cpu contract, torch_binding.h:28-37) */
  OQ_VALUES_UNIT_BF16 = 2 /* bf16(centroid[code]), [M, K]; the token norm stays in   */
                          /* norms_out and is applied by the matmul epilogue         */
} oq_values_mode;

/* Library / device probe.  Returns OQ_OK when a gfx950 device is current. */
int oq_device_ok(void);
const char *oq_last_error(void);
const char *oq_version(void);

/*
 * Fused RPBH rotate + per-token quantize.
 * Replaces quantize_activations_packed_w4 / quantize_activations_int8 /
 * quantize_activations_cpu (torch_binding.cpp:13-31,47-66; kernels
 * packed_matmul.cu:581-742; semantics src/orbitquant/functional.py:16-22):
 *
 *   s      = ||fp32(x_row)||_2                     (fixed summation order, see below)
 *   unit   = fp32(x_row) / (s + eps)               (IEEE division)
 *   y      = unit[perm] * signs                    (gather, exact)
 *   y      = blockwise FWHT(y), block `block`, butterfly distance 1,2,4,...
 *   rot    = y * inv_sqrt_block                    (one fp32 multiply)
 *   code   = #{ j : boundaries[j] < rot }          (ties to the lower code)
 *
 * Sum of squares order: the row is zero-padded to a multiple of 2048 and viewed
 * as [passes][256 lanes][8]; per (pass, lane) the eight squares are added as
 * ((s0+s1)+(s2+s3))+((s4+s5)+(s6+s7)); each lane adds its passes left to right;
 * the 256 lane sums are reduced by a balanced binary tree in lane order.  No
 * operation is contracted into an FMA.
 *
 * x            [M, K] of x_dtype, row-major, contiguous
 * perm         int32 [K], signs int8 [K] (+1/-1)
 * boundaries   fp32 [levels-1], ascending;  2 <= levels <= 256
 * centroids    fp32 [levels]; only read when values_mode != OQ_VALUES_NONE (else may be NULL)
 * block        power of two dividing K;  K <= 16384
 * rotate_plan  NULL, or the plan oq_rotate_plan_build made from these perm, signs, boundaries,
 *              levels, K, block and inv_sqrt_block: launches of more than 16 rows, and fewer where a row
 *              has several blocks or blocks of 1024 to 4096, then take the plan-based kernel (a third of
 *              the instructions, the same results bit for bit)
 * codes_out    NULL or [M, K] u8 / [M, K/2] u8 per code_format
 * values_out   NULL or per values_mode
 * norms_out    fp32 [M]: the raw norm s (no eps); may be NULL
 */
int oq_rotate_quantize(const void *x, int x_dtype, int64_t M, int64_t K,
                       const int32_t *perm, const int8_t *signs,
                       const float *boundaries, const float *centroids, int levels,
                       int64_t block, float eps, float inv_sqrt_block, const void *rotate_plan,
                       void *codes_out, int code_format,
                       void *values_out, int values_mode,
                       float *norms_out, void *stream);

/*
 * The rotate plan: everything the rotate+quantize kernel can know about a layer before it sees
 * a token (the permutation as gather offsets, the signs by position, the boundaries folded with
 * inv_sqrt_block, the bucketize tables), built once per layer by one small launch and kept by
 * the caller in device memory next to the layer's other constants: oq_rotate_plan_bytes(K)
 * bytes, 16-byte aligned.  No counterpart in the reference, whose kernels re-derive all of it per
 * row (packed_matmul.cu:581-657).  A plan is only valid for the arguments it was built from,
 * and for the library that built it; a call that passes a plan built for another K, block or levels, or
 * by a library of another layout, writes no codes, and NaN for the norms.
 */
uint64_t oq_rotate_plan_bytes(int64_t K);
int oq_rotate_plan_build(const int32_t *perm, const int8_t *signs, const float *boundaries, int levels,
                         int64_t K, int64_t block, float inv_sqrt_block, void *plan_out, void *stream);

/* The same launch, which also copies perm and signs to perm_copy int32 [K] and signs_copy int8 [K]: for a caller whose
 * constants came to the device in one buffer and that wants them in memory of their own. */
int oq_rotate_plan_build_copy(const int32_t *perm, const int8_t *signs, const float *boundaries, int levels, int64_t K,
                              int64_t block, float inv_sqrt_block, void *plan_out, int32_t *perm_copy, int8_t *signs_copy,
                              void *stream);

/*
 * The weight side of a layer on the GPU: what the packed matmuls read, made from a float weight
 * matrix.  Replaces the reference's device-side weight quantization
 * (src/orbitquant/layers.py:102-125,159-222; src/orbitquant/kernels/triton_cuda.py:926-1039,2740-2935).
 * Per output row:
 *
 *   r      = ||fp32(w_row)||_2                     (the summation order of oq_rotate_quantize)
 *   rot    = blockwise FWHT(fp32(w_row)[perm] * signs) * inv_sqrt_block
 *   unit   = rot / max(r, eps)                     (IEEE division; note the order: rotate, scale, divide)
 *   idx    = #{ j : boundaries[j] < unit }
 *
 * packed_out is the flat little-endian bit stream of idx[N, K], `bits` per index
 * (ceil(N*K*bits/8) bytes; src/orbitquant/packing/bitpack.py:8-46), row_norms_out is bf16(r) [N].
 * A zero row keeps r = 0, so it dequantizes to exact zeros.
 *
 * w            [N, K] of w_dtype, row-major, 16-byte aligned;  K a multiple of 8, K <= 16384
 * rotate_plan  the plan oq_rotate_plan_build made from the layer's perm and signs with THESE
 *              boundaries, levels, K, block and inv_sqrt_block.  Its bucketize table is used where it is
 *              one over `boundaries`; a plan of the same perm, signs, levels, K and block over others (the
 *              layer's activation plan, say) gives the same indices from a search (14336 x 4096 into four bits:
 *              99 us instead of 78)
 * boundaries   fp32 [levels-1] of the weight codebook;  2 <= levels <= 2^bits, 1 <= bits <= 8
 * block        power of two dividing K, 8 <= block <= 4096
 */
int oq_quantize_weight(const void *w, int w_dtype, int64_t N, int64_t K, const void *rotate_plan,
                       const float *boundaries, int levels, int64_t block, float eps, float inv_sqrt_block,
                       int bits, uint8_t *packed_out, uint16_t *row_norms_out, void *stream);

/*
 * The same, on f(x) instead of x, for an elementwise function f of a 16-bit
 * input given as a table: input_map[bits of x] = bits of f(x), 65536 entries of
 * the same dtype as x, 16-byte aligned, on the device.  The result is what
 * oq_rotate_quantize returns for the tensor f(x), bit for bit; f(x) is never
 * written to memory.  x_dtype must be OQ_F16 or OQ_BF16.  rotate_plan: as for
 * oq_rotate_quantize (bf16 rows into codes take the plan-based kernel with it).
 *
 * No counterpart in the reference's extension: there the activation between two
 * quantized linears (the GELU of an MLP, functional calls in the model code) is
 * a separate elementwise kernel that writes f(x) and the quantizer reads it
 * back; the table is how a caller hands that function to this kernel without
 * changing its results (fill it by applying the framework's own f to all
 * 65536 bit patterns).
 */
int oq_rotate_quantize_mapped(const void *x, int x_dtype, const uint16_t *input_map,
                              int64_t M, int64_t K,
                              const int32_t *perm, const int8_t *signs,
                              const float *boundaries, const float *centroids, int levels,
                              int64_t block, float eps, float inv_sqrt_block, const void *rotate_plan,
                              void *codes_out, int code_format,
                              void *values_out, int values_mode,
                              float *norms_out, void *stream);

/*
 * Sets (value != NULL) or clears one of the library's experiment switches, the OQ_* environment
 * variables that pick a launch shape or turn a kernel variant off (OQ_GEMM_TILE, OQ_GEMM_WG_SPLIT,
 * OQ_GEMV_CFG, OQ_NO_TOKEN_LINEAR, ...).  The library reads the environment once per process;
 * tests and measurements that compare variants inside one process change a switch through this
 * call.  Results stay correct under every setting; only which kernel computes them changes.
 * Not thread-safe against running calls.  No counterpart in the reference.
 * Refused (OQ_ERR_INVALID) unless the process was started with ORBITQUANT_DEBUG=1 in its
 * environment: a serving process cannot have its kernels, and so the bits of its results,
 * switched under it.
 */
int oq_debug_override(const char *name, const char *value);

/*
 * Packed-weight linear on quantized activations (the fused hot path):
 *
 *   out[m,n] = (sum_k c_a[code[m,k]] * c_w[idx[n,k]]) * s[m] * r_w[n] + bias[n]
 *
 * Replaces matmul_packed_w4a4_int8 (torch_binding.cpp:39-46; packed_matmul.cu:744-1009)
 * for every weight width, with exact (bf16-rounded) centroids instead of the
 * int8 surrogate.  M <= 64 takes the streaming small-M kernel (the weights are read and
 * decoded once, sixteen token rows per matrix instruction, up to four blocks of sixteen per
 * workgroup), larger M the MFMA tile kernel.  A token row's result does not depend on the
 * rows computed with it as long as the call stays within 64 rows.  A problem with few output
 * tiles and many K-steps (some hundred tokens on a short-and-long matrix) is shared between
 * workgroups along K when the caller provides a workspace for the fp32 partial tiles, and a large
 * problem (some thousand tokens) is decoded once into the workspace and multiplied from there.  A
 * shared K is added in parts, so the last bits of such a result depend on the workspace; a decoded
 * problem gives the same bits as without:
 *
 * workspace    NULL, or a device buffer of at least oq_packed_linear_workspace_bytes(...) bytes, 16-byte
 *              aligned, that this call may overwrite (calls on one stream are ordered and may share one).
 *              The library allocates nothing: as in the reference, whose Python wrapper owns every
 *              allocation (torch-ext/orbitquant_packed_matmul/__init__.py:130-160), kernels borrow all
 *              pointers.  NULL, or too small: the single launch.  Which kernel runs depends on the
 *              arguments alone, so a call captured into a graph computes what the eager call does, bit
 *              for bit.
 *
 * codes        activation codes in code_format (see oq_rotate_quantize)
 * token_norms  fp32 [M]
 * act_centroids fp32 [2^a_bits]
 * packed_w     flat little-endian bit stream of idx[N,K], value v at bits [v*w_bits, v*w_bits+w_bits)
 *              (src/orbitquant/packing/bitpack.py:8-46); w_bits in [1, 8]: 2, 3, 4, 6 and 8 take the
 *              tiled and streaming kernels, the other widths the shape-agnostic kernel
 * row_norms    bf16 [N] (raw uint16 bit patterns)
 * w_centroids  fp32 [2^w_bits]
 * bias         NULL or [N] of bias_dtype
 * out          [M, N] of out_dtype (OQ_BF16, OQ_F16 or OQ_F32)
 */
int oq_packed_linear(const void *codes, int code_format, const float *token_norms,
                     const float *act_centroids, int a_bits,
                     const uint8_t *packed_w, int w_bits, const uint16_t *row_norms,
                     const float *w_centroids, const void *bias, int bias_dtype,
                     int64_t M, int64_t N, int64_t K, void *out, int out_dtype,
                     void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * Bytes of workspace oq_packed_linear (and _mapped, oq_quantized_linear, and each member of a group)
 * can make use of for this shape; 0 when it takes a single launch anyway.  No counterpart in the
 * reference (its wrapper sizes its own temporaries).
 */
uint64_t oq_packed_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int code_format, int a_bits);

/*
 * What of it holds partial tiles of a K shared between workgroups: 0 for a problem that would be decoded into
 * the workspace, and so the size to fall back on when that much memory is not there.
 */
uint64_t oq_packed_linear_least_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int code_format, int a_bits);

/*
 * oq_packed_linear for 4-bit codes (two per byte) on both sides whose codebooks are int8 tables, summed in
 * int32 on the int8 matrix instructions:
 *
 *   out[m,n] = (sum_k act_table[code[m,k]] * w_table[idx[n,k]]) * (s[m] * scale) * r_w[n] + bias[n]
 *
 * (matmul_packed_w4a4_int8, torch_binding.cpp:39-46.)  act_table and w_table: int8 [16].  For the shapes that
 * oq_packed_linear_int8_workspace_bytes gives a size for, with a workspace of at least that size; OQ_ERR_UNSUPPORTED
 * for the others (0), which oq_packed_linear, with its workspace, is about as fast or faster on.
 */
int oq_packed_linear_int8(const void *codes, const float *token_norms, float scale, const int8_t *act_table,
                          const uint8_t *packed_w, const uint16_t *row_norms, const int8_t *w_table, const void *bias,
                          int bias_dtype, int64_t M, int64_t N, int64_t K, void *out, int out_dtype, void *workspace,
                          uint64_t workspace_bytes, void *stream);
uint64_t oq_packed_linear_int8_workspace_bytes(int64_t M, int64_t N, int64_t K);

/*
 * `count` packed linears on the SAME activation codes (the q, k and v projections of an attention
 * block, the gate and up projections of an MLP): out[i] = oq_packed_linear(codes, ..., packed_w[i],
 * w_bits[i], row_norms[i], w_centroids[i], bias[i], M, N[i], K), bit for bit.  The argument arrays
 * (count entries each, read during the call only) live in host memory and hold device pointers;
 * `bias` may be NULL (no matrix has one) or hold NULL entries.  For at most 32 tokens, nibble
 * codes, 2-, 3- or 4-bit weights and two to four matrices the whole group is ONE launch of the
 * streaming kernel (at decode sizes a launch is mostly fixed cost); any other group runs as
 * `count` launches.  No counterpart in the reference, whose layers each call
 * matmul_packed_* on their own (src/orbitquant/layers.py:1079-1455); it replaces `count`
 * consecutive calls of oq_packed_linear.
 */
int oq_packed_linear_group(const void *codes, int code_format, const float *token_norms,
                           const float *act_centroids, int a_bits, int count,
                           const uint8_t *const *packed_w, const int *w_bits,
                           const uint16_t *const *row_norms, const float *const *w_centroids,
                           const void *const *bias, int bias_dtype, int64_t M, const int64_t *N,
                           int64_t K, void *const *out, int out_dtype,
                           void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * oq_packed_linear followed by an elementwise function of the 16-bit outputs given as a
 * table (output_map[bits of y] = bits of f(y), 65536 entries of the output dtype, 16-byte
 * aligned, on the device): out = f(linear) bit for bit, f(...) applied before the store
 * (tile and streaming kernels: where they store; other kernels: by a small elementwise launch).  out_dtype
 * must be OQ_F16 or OQ_BF16.  No counterpart in the reference, like oq_rotate_quantize_mapped:
 * it is the activation that follows a linear, without its kernel.
 */
int oq_packed_linear_mapped(const void *codes, int code_format, const float *token_norms,
                            const float *act_centroids, int a_bits,
                            const uint8_t *packed_w, int w_bits, const uint16_t *row_norms,
                            const float *w_centroids, const void *bias, int bias_dtype,
                            int64_t M, int64_t N, int64_t K, void *out, int out_dtype,
                            const uint16_t *output_map, void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * The whole quantized-linear forward in one call: oq_rotate_quantize (through
 * `input_map` when it is not NULL, see oq_rotate_quantize_mapped) followed by
 * oq_packed_linear, with the same results bit for bit.  It is the native form of the
 * reference layer's forward (src/orbitquant/layers.py:1079-1455: quantize_activations_*
 * then matmul_packed_*), which exists there only as Python glue between two ops.
 *
 * One token (M == 1) of a 16-bit dtype with a_bits <= 4, w_bits 2, 3 or 4, K a multiple of
 * 128 up to 8192, N up to 8192 and 16-byte aligned operands is a SINGLE launch: every workgroup
 * of the streaming kernel quantizes the token itself while its weight loads are in flight, so
 * decoding pays one launch per linear and the scratch buffers are not touched.  Callers that
 * cannot tell in advance pass scratch always; NULL scratch is an error only when it is
 * needed.  Every other shape is the two launches, with the codes
 * ([M, K/2] bytes when a_bits <= 4 and K is even, else [M, K]) and norms (fp32 [M]) passing
 * through the caller's scratch buffers (16-byte aligned).
 *
 * `rotate_plan` (NULL for none): see oq_rotate_quantize.
 *
 * `output_map` (NULL for none) is a table like `input_map`, of the OUTPUT dtype (16-bit
 * only), applied to every output value before it is stored: out = f(linear(x)) bit for bit
 * what f applied to the stored result of the plain call gives.  The tile kernels look the
 * values up in their epilogue, the small-M kernels where they store; the shape-agnostic kernels are
 * followed by a tiny elementwise launch.  It is the cheaper place for the activation between two linears (a
 * lookup per output value in a kernel that is waiting for its stores, instead of a lookup
 * per input value in the quantizer, which has no such slack).
 */
int oq_quantized_linear(const void *x, int x_dtype, const uint16_t *input_map,
                        int64_t M, int64_t K,
                        const int32_t *perm, const int8_t *signs,
                        const float *boundaries, const float *act_centroids, int a_bits,
                        int64_t block, float eps, float inv_sqrt_block, const void *rotate_plan,
                        const uint8_t *packed_w, int w_bits, const uint16_t *row_norms,
                        const float *w_centroids, const void *bias, int bias_dtype, int64_t N,
                        void *codes_scratch, float *norms_scratch,
                        void *out, int out_dtype, const uint16_t *output_map,
                        void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * oq_quantized_linear for `count` linears that read the same input (q, k and v of an attention
 * block; gate and up of an MLP): the input is quantized once into the caller's scratch buffers
 * (required; sizes as for oq_quantized_linear), then oq_packed_linear_group.  out[i] equals what
 * oq_quantized_linear gives for matrix i, bit for bit.  Arrays as in oq_packed_linear_group.
 * No counterpart in the reference (see oq_packed_linear_group).
 */
int oq_quantized_linear_group(const void *x, int x_dtype, const uint16_t *input_map,
                              int64_t M, int64_t K,
                              const int32_t *perm, const int8_t *signs, const float *boundaries,
                              const float *act_centroids, int a_bits,
                              int64_t block, float eps, float inv_sqrt_block, const void *rotate_plan,
                              int count, const uint8_t *const *packed_w, const int *w_bits,
                              const uint16_t *const *row_norms, const float *const *w_centroids,
                              const void *const *bias, int bias_dtype, const int64_t *N,
                              void *codes_scratch, float *norms_scratch,
                              void *const *out, int out_dtype,
                              void *workspace, uint64_t workspace_bytes, void *stream);

/*
 * oq_quantized_linear for callers that cannot allocate device memory or bring a workspace:
 * code running under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc.  No counterpart in the reference.  Same arguments as oq_quantized_linear without
 * the two scratch pointers, and the results of oq_quantized_linear without a workspace (with one,
 * the order of the additions can differ, see oq_packed_linear): codes and norms pass through a buffer
 * of OQ_STATIC_SCRATCH_BYTES that is part of the library's device image (every GPU the library
 * runs on holds its own copy until the process ends).  The call allocates and frees nothing.
 * Shapes whose codes ([M, K/2] bytes for a_bits <= 4 and even K, else [M, K], rounded up to
 * 256) plus norms (4 M bytes) do not fit are refused with OQ_ERR_UNSUPPORTED.  All calls on one
 * GPU share the buffer: calls that may overlap there (different streams, or graphs replayed
 * concurrently) race, and the buffer keeps the previous call's contents (every byte a call
 * reads it has written itself first).  The buffer's address on a device is looked up the
 * first time that device is current in oq_device_ok() or in this call; callers that capture
 * graphs call oq_device_ok() once beforehand.
 */
#define OQ_STATIC_SCRATCH_BYTES (8u << 20)
int oq_quantized_linear_static(const void *x, int x_dtype, const uint16_t *input_map,
                               int64_t M, int64_t K,
                               const int32_t *perm, const int8_t *signs,
                               const float *boundaries, const float *act_centroids, int a_bits,
                               int64_t block, float eps, float inv_sqrt_block, const void *rotate_plan,
                               const uint8_t *packed_w, int w_bits, const uint16_t *row_norms,
                               const float *w_centroids, const void *bias, int bias_dtype, int64_t N,
                               void *out, int out_dtype, const uint16_t *output_map, void *stream);

/*
 * Packed-weight matmul on float activations:
 *
 *   out[m,n] = (sum_k x[m,k] * c_w[idx[n,k]]) * r_w[n] + bias[n]      (out in x's dtype)
 *
 * Replaces matmul_packed_weight (torch_binding.cpp:7-12,32-38; packed_matmul.cu:1335-1713).
 * bits in [1, 8].  token_scale: NULL, or fp32 [M] multiplied into row m (lets the
 * caller pass unit-norm bf16 centroids plus token norms).
 * workspace: NULL, or oq_matmul_packed_weight_workspace_bytes(...) bytes of device memory, 16-byte aligned,
 * that the call may overwrite.  With it, bf16 activations (from two tokens on; one token on large matrices)
 * and fp16 activations (from nine tokens on) are first rewritten into the matrix core's operand order
 * (2 * M * K bytes, rows padded to 32) and the tile kernel reads that copy; where it is faster (large problems,
 * weights of six and eight bits) the weights are decoded into the workspace too.  Without it every wavefront stages
 * its own rows through LDS (bf16: no buffer, the same sums, 10-15 % slower on large problems) or the workgroup does
 * (fp16: sums in another order).  The library allocates nothing.
 */
int oq_matmul_packed_weight(const void *x, int x_dtype, const float *token_scale,
                            const uint8_t *packed_w, int bits, const uint16_t *row_norms,
                            const float *w_centroids, const void *bias, int bias_dtype,
                            int64_t M, int64_t N, int64_t K, void *out, int out_dtype,
                            void *workspace, uint64_t workspace_bytes, void *stream);

/* Bytes of workspace oq_matmul_packed_weight can make use of for this shape (0: none). */
uint64_t oq_matmul_packed_weight_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_bits, int x_dtype);

/*
 * Packed INT4 group-scaled linear on bf16 activations (the AdaLN modulation linears):
 *
 *   w[n,k]   = bf16( (q[n,k] - 8) * float(scales[n, k / group_size]) )
 *   out[m,n] = bf16( sum_k x[m,k] * w[n,k] + float(bias[n]) )          (fp32 accumulation)
 *
 * Replaces matmul_packed_adaln_int4_cpu (torch_binding.cpp:47-66) and the reference's Triton
 * kernel for it (src/orbitquant/kernels/triton_cuda.py:682-819) on AMD GPUs.
 *
 * x             bf16 [M, K] (raw bit patterns), row-major
 * packed_weight 4-bit q, two per byte, low nibble first, rows padded to whole groups:
 *               [N, groups * group_size / 2] bytes with groups = ceil(K / group_size)
 *               (src/orbitquant/adaln.py:17-35)
 * scales        bf16 [N, groups]
 * bias          NULL or bf16 [N]
 * out           bf16 [M, N]
 * K a multiple of 8, group_size a multiple of 8 and a 16-byte aligned x take the streaming
 * kernel, anything else a shape-agnostic one.
 */
int oq_matmul_packed_adaln_int4(const uint16_t *x, const uint8_t *packed_weight, const uint16_t *scales,
                                const uint16_t *bias, int64_t M, int64_t N, int64_t K, int64_t group_size,
                                uint16_t *out, void *stream);

/*
 * The weight side of the AdaLN linears on the GPU: group-wise round-to-nearest INT4
 * (src/orbitquant/adaln.py:17-35 `quantize_adaln_weight_int4`; the reference runs it as torch
 * operations on whatever device holds the weight):
 *
 *   scale[n,g] = max(max_k |w[n,k]|, 1e-12) / 7            over the group's k, fp32, IEEE division
 *   q[n,k]     = clamp(round_half_even(w[n,k] / scale[n,g]), -8, 7) + 8      (padding beyond K: 8)
 *
 * w          [N, K] of w_dtype (OQ_F32 / OQ_F16 / OQ_BF16), row-major
 * packed_out [N * groups * group_size / 2] bytes, low nibble first, groups = ceil(K / group_size)
 * scales_out fp32 [N, groups] (the module stores them rounded to bf16)
 * group_size even.
 */
int oq_quantize_adaln_weight(const void *w, int w_dtype, int64_t N, int64_t K, int64_t group_size, uint8_t *packed_out,
                             float *scales_out, void *stream);

/*
 * Unpack a little-endian bit stream into one index per byte (debug / tests;
 * the GPU twin of unpack_lowbit, src/orbitquant/packing/bitpack.py:63-97).
 */
int oq_unpack_lowbit(const uint8_t *packed, int bits, int64_t count, uint8_t *out, void *stream);

/*
 * The inverse of oq_unpack_lowbit: values[i] (its low `bits` bits) into bits [i * bits, (i + 1) * bits)
 * of a little-endian stream of ceil(count * bits / 8) bytes, unused tail bits zero.
 * Replaces pack_lowbit (src/orbitquant/packing/lowbit.py) and its Triton form
 * (src/orbitquant/kernels/triton_cuda.py:878-899, 2681-2710) on AMD GPUs.  bits in [1, 8].
 */
int oq_pack_lowbit(const uint8_t *values, int bits, int64_t count, uint8_t *packed_out, void *stream);

/*
 * The dense form of a packed weight, in the rotated basis the layer multiplies in:
 *   out[n,k] = centroids[index[n,k]] * float(row_norms[n])        (one fp32 product, then rounded to out_dtype)
 * Replaces dequantize_packed_weight_with_triton (src/orbitquant/kernels/triton_cuda.py:523-547,
 * 1538-1571; fp32 out there) for the reference's `dequant_bf16` debug mode.
 * packed_weight  N * K indices of `bits` bits, one stream over the whole matrix
 * row_norms      bf16 [N];  centroids fp32 [2^bits];  out [N, K] of out_dtype.
 */
int oq_dequantize_packed_weight(const uint8_t *packed_weight, int bits, const uint16_t *row_norms, const float *centroids,
                                int64_t N, int64_t K, void *out, int out_dtype, void *stream);

/*
 * ---- The 4-bit key/value cache of a serving program and the attention that reads it (no counterpart in the reference) ----
 *
 * A token's key or value of one head, x[D], is held as y = H(signs * x), H the unnormalised Walsh-Hadamard transform
 * (butterfly distance 1, 2, 4, ...), in fp32:
 *   a    = bf16(max|y| * fp32(1/6)), 0 where that is below 2^-126, NaN where y has an infinity or a NaN
 *   code = the E2M1 value (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign: bit 3) nearest to y * (1 / a), ties to the even code
 * and stands for x^ = signs * H(a * code) / D.  The struct is host memory, read during the call.  Pages hold page_size
 * tokens; a slot is page * page_size + place in the page.
 */
typedef struct {
  uint8_t *k_codes;     /* [pages, kv_heads, page_size, D/2]; byte j: dimension 2j in the low half, 2j+1 in the high half */
  uint16_t *k_scales;   /* bf16 [pages, kv_heads, page_size]                                                                */
  uint8_t *v_codes;     /* [pages, kv_heads, D/2, page_size]: the same bytes, a page's tokens side by side                 */
  uint16_t *v_scales;   /* bf16 [pages, kv_heads, page_size]                                                                */
  const int8_t *signs;  /* [D], +1/-1; all five 16-byte aligned                                                               */
  int64_t pages;        /* 1 .. 2^31 - 1                                                                                    */
  int64_t kv_heads;     /* 1 .. 65535                                                                                       */
  int64_t page_size;    /* a power of two, 16 .. 1024                                                                       */
  int64_t head_dim;     /* D: 64, 128 or 256                                                                                */
} oq_kv_cache;

/*
 * Pages and slots for the new tokens of a batch.  Request r holds lengths[r] tokens in the first ceil(lengths[r] /
 * page_size) pages of its row of the block table and gets new_lengths[r] more (negative counts are taken as 0); the
 * pages this needs are taken from the front of free_pages in request order, behind the *taken that are already given out.
 *
 * lengths, new_lengths  int32 [requests], requests <= 8192
 * table        int32 [requests, table_width], rows table_stride apart: the entries of new pages are written, -1 where
 *              the free list has run out; columns beyond the table are dropped
 * free_pages   int32 [free_count]; taken int32 [1]
 * slots        int64 [tokens], positions int32 [tokens]: of the new tokens, request by request; a token without a page
 *              has the slot -1, and what lies behind the last token has both -1
 * starts       int32 [requests + 1]: where a request's tokens begin
 * lengths_after int32 [requests] = lengths + new_lengths; taken_after int32 [1], at most free_count
 * No output may overlap an input other than the table itself.  Sums of new tokens below 2^31.
 */
int oq_kv_assign(const int32_t *lengths, const int32_t *new_lengths, int64_t requests, int32_t *table,
                 int64_t table_stride, int64_t table_width, const int32_t *free_pages, int64_t free_count,
                 const int32_t *taken, int64_t page_size, int64_t tokens, int64_t *slots, int32_t *positions,
                 int32_t *starts, int32_t *lengths_after, int32_t *taken_after, void *stream);

/*
 * Keys and values [tokens, kv_heads, D] of dtype into the cache at slots[token]; slots that are negative or beyond the
 * last page are skipped.  No slot twice in one call.  Strides in elements; the last dimension is contiguous.
 * (This call, oq_kv_read and oq_kv_attend are OQ_ERR_UNSUPPORTED where a launch would have 2^32 threads: 2^28 vectors of a head.)
 */
int oq_kv_write(const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
                int64_t v_head_stride, int dtype, const int64_t *slots, int64_t tokens, const oq_kv_cache *cache,
                void *stream);

/* What the cache holds at slots[token], as [tokens, kv_heads, D] of dtype, contiguous, 16-byte aligned; zeros for slots
 * that are negative or beyond the last page. */
int oq_kv_read(const int64_t *slots, int64_t tokens, const oq_kv_cache *cache, void *k, void *v, int dtype, void *stream);

/*
 * Attention of q [tokens, heads, D] over the cache; heads a multiple of kv_heads, head h reads key head h / (heads /
 * kv_heads).  Request r holds lengths[r] tokens (new ones included, already written), at the pages of its row of the
 * block table, and its queries are the last of them: tokens starts[r] .. starts[r+1] - 1 of q, or token r where starts is
 * NULL (tokens = requests then).  A query at position p sees the cached positions <= p (causal) or all of them, of these
 * the last `window` if window > 0 (causal only), and none whose page is missing (-1, or not one of the cache's).
 *
 *   out = sum_t softmax_t(scale * q . k^_t) v^_t        of q's dtype, [tokens, heads, D], contiguous, 16-byte aligned
 *   lse = ln sum_t e^(scale * q . k^_t)                 NULL or fp32 [tokens, heads]
 * A query that sees nothing, and a token that belongs to no request, gets zeros (lse -inf).  starts[0] is 0.
 *
 * max_length   the longest of the lengths as far as the caller knows, -1 if it does not; max_new likewise the largest number of
 *              a request's queries (1 without starts).  They choose launch shapes: a wrong one costs time, never a result's correctness.
 * workspace    NULL, or oq_kv_attend_workspace_bytes(...) bytes, 16-byte aligned: the keys are then cut into parts where
 *              there are few rows.  Without it (or with less) the call runs uncut.
 */
int oq_kv_attend(const void *q, int q_dtype, int64_t tokens, int64_t heads, int64_t q_token_stride,
                 int64_t q_head_stride, const oq_kv_cache *cache, const int32_t *table, int64_t table_stride,
                 int64_t table_width, const int32_t *lengths, const int32_t *starts, int64_t requests, int causal,
                 int64_t window, float scale, int64_t max_length, int64_t max_new, void *out, float *lse,
                 void *workspace, uint64_t workspace_bytes, void *stream);
uint64_t oq_kv_attend_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                      int64_t page_size, int64_t table_width, int64_t requests, int has_starts,
                                      int64_t window, int64_t max_length, int64_t max_new);

/*
 * Norms of queries and keys for each head, and their rotary positions, in one pass (no counterpart in the reference).
 *
 * The D values of a head are D/2 pairs: 2p and 2p+1 (interleaved), or p and p + R/2 of the first R and p and p + (D-R)/2 of
 * the rest (R = rotary_dim, 0 without tables; p and p + D/2 then).  In fp32, every product and sum rounded by itself:
 *   s  = sum of squares: the two of a pair, then pairs 4, 2, 1 apart of each eight, then eights 1, 2, 4, ... apart
 *   y  = (x * (1 / sqrt(s * fp32(1/D) + eps))) * w              where norm is set; w = 1 where there is no weight
 *   (y0, y1) -> (y0 c - y1 s, y1 c + y0 s)                      of the first R/2 pairs; c, s: the position's row of the tables
 * and rounded once to the output's type.  Squares are fp32: norms are right for values below 2^59 where mean square + eps is a normal fp32
 * number (2^-126 and more; with eps = 0 smaller heads lose digits and then become infinite, and one of zeros NaN, as 0 / 0 is).
 * The struct is host memory, read during the call.
 */
typedef struct {
  const float *cos, *sin;    /* [rows, rotary_dim / 2], contiguous; both NULL: nothing is turned                                   */
  int64_t rows, rotary_dim;  /* even, 2 .. D                                                                                       */
  const int32_t *positions;  /* [tokens]: rows of the tables; a token at a negative one is not turned, one behind them becomes NaN.  NULL: token t has row t */
  const void *q_weight;      /* [D] of weight_dtype, or NULL                                                                       */
  const void *k_weight;      /* the same                                                                                           */
  int weight_dtype;
  int norm;                  /* 0: no norm (and no weights)                                                                        */
  float eps;                 /* >= 0                                                                                               */
  int interleaved;
} oq_qk_norm_rotary_plan;

/*
 * q [tokens, heads, D] and k [tokens, kv_heads, D] of dtype -> q_out and k_out, contiguous, 16-byte aligned.  D even, 2 .. 512.
 * Strides in elements; the last dimension is contiguous.  No output may overlap an input.
 */
int oq_qk_norm_rotary(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t heads, const void *k,
                      int64_t k_token_stride, int64_t k_head_stride, int64_t kv_heads, int dtype, int64_t tokens,
                      int64_t head_dim, const oq_qk_norm_rotary_plan *plan, void *q_out, void *k_out, void *stream);

/*
 * The same for q, and keys and values into the cache at slots[token] as oq_kv_write puts them, the key normed and turned on the
 * way: its codes are those of the fp32 result, which is not rounded in between.  One launch.
 */
int oq_kv_append(const void *q, int64_t q_token_stride, int64_t q_head_stride, int64_t heads, const void *k,
                 int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride,
                 int64_t v_head_stride, int dtype, const int64_t *slots, int64_t tokens,
                 const oq_qk_norm_rotary_plan *plan, const oq_kv_cache *cache, void *q_out, void *stream);

/*
 * ---- Trees of drafted tokens over the cache ----
 * A request's new tokens are a tree instead of a chain: token i hangs on token parents[i] < i of the request's new ones, or on what the
 * request has cached already (negative, or not less than i).
 *
 * parents    int32 [tokens]; starts int32 [requests + 1] and lengths int32 [requests] as oq_kv_assign gives them (starts, lengths_after)
 * positions  int32 [tokens]: of token i, its depth (0 for one that hangs on the cached ones) behind the request's cached tokens
 * masks      uint64 [tokens, mask_words], mask_words 1 .. 4: bit j % 64 of word j / 64 is set for token i itself and those it hangs on
 * A request with more new tokens than 64 * mask_words is a prompt: positions one behind the other, masks of zeros (which
 * oq_kv_attend_tree does not look at).  Tokens of no request have position -1 and zeros.
 */
int oq_kv_tree(const int32_t *parents, const int32_t *starts, const int32_t *lengths, int64_t requests, int64_t tokens,
               int64_t mask_words, int32_t *positions, uint64_t *masks, void *stream);

/*
 * oq_kv_attend (causal) where a query sees of its request's new tokens those whose bit is set in its mask, whichever these are: any masks will
 * do, its own token is seen only if its bit is set.  It sees all tokens before the new ones.  Of what it sees, the last `window`
 * in the cache's order if window > 0.  A request with more new tokens than 64 * mask_words is causal.  masks 8-byte aligned.
 * workspace: NULL, or oq_kv_attend_tree_workspace_bytes(...) bytes, as for oq_kv_attend.
 */
int oq_kv_attend_tree(const void *q, int q_dtype, int64_t tokens, int64_t heads, int64_t q_token_stride,
                      int64_t q_head_stride, const oq_kv_cache *cache, const int32_t *table, int64_t table_stride,
                      int64_t table_width, const int32_t *lengths, const int32_t *starts, int64_t requests,
                      const uint64_t *masks, int64_t mask_words, int64_t window, float scale, int64_t max_length,
                      int64_t max_new, void *out, float *lse, void *workspace, uint64_t workspace_bytes, void *stream);
uint64_t oq_kv_attend_tree_workspace_bytes(int q_dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                           int64_t page_size, int64_t table_width, int64_t requests, int has_starts,
                                           int64_t mask_words, int64_t window, int64_t max_length, int64_t max_new);

/*
 * After the step: of each request's new tokens those of an accepted path stay, as if they had been its only ones.
 *
 * kept       int32 [requests, most], most <= 256: of the request's new tokens, rising; the list ends at the first entry that does not rise, is
 *            not one of them (-1, say), has no slot or would go where there is none.  The i-th kept token's entries go to the i-th new token's slot
 *            OQ_KV_KEEP_ALL as a list's first entry: all of the request's new tokens stay, however many they are (a prompt in a step with trees)
 * lengths, starts, slots   as oq_kv_assign gave them for the step (lengths_after, starts, slots [tokens])
 * caches     host memory: the caches of cache_count layers, of one shape, all moved in one launch (for every 64 of them);
 *            a cache that layers share stands there once, and no two parts of caches share memory (OQ_ERR_INVALID)
 * table, free_pages, taken NULL, or as oq_kv_assign left them (taken: taken_after): pages behind the kept tokens go back onto the free
 *            list, in front of those that it gives out next; the table is not changed, its columns behind the kept pages
 *            stand for nothing.  Requests <= 8192.  The pages that oq_kv_assign drew for columns behind the table's end go back too, in a call
 *            for all of its requests; but for a step in which the list ran out and no column of the table got a page: which pages
 *            were drawn is not known then.  (A table with room for every new token never has such pages.)
 * lengths_after int32 [requests]: without the forgotten tokens; taken_after int32 [1]
 * No slot twice in slots.  No output may overlap an input other than the caches and free_pages.
 */
enum { OQ_KV_KEEP_ALL = -2 };
int oq_kv_keep(const int32_t *kept, int64_t most, const int32_t *lengths, const int32_t *starts, const int64_t *slots,
               int64_t requests, int64_t tokens, const oq_kv_cache *caches, int64_t cache_count, const int32_t *table,
               int64_t table_stride, int64_t table_width, int32_t *free_pages, int64_t free_count,
               const int32_t *taken, int32_t *lengths_after, int32_t *taken_after, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* ORBITQUANT_HIP_H */
