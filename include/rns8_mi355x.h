/* MI355X extensions to the rns8 C ABI: the device-resident hot path.
 *
 * The reference ABI (rns8/rns8.h) takes and returns host memory and ends
 * every call with a device synchronization, so each GEMM pays PCIe transfers.
 * These entry points run the same pack -> plane GEMM -> Garner stages on
 * operands that already live in HBM, enqueue their kernels on a caller
 * stream and return without synchronizing. They have no counterpart in the
 * reference; they are what a caller that chains GEMMs on the GPU (or a
 * benchmark measuring the kernels rather than PCIe) binds. They reuse the
 * same handles, validation and kernels as the host entry points.
 *
 * Conventions
 *   - `stream` is a hipStream_t passed as void*; NULL selects the context's
 *     own stream, which waits for no other. Work is ordered on that stream
 *     only. The device's default stream, whose handle is NULL elsewhere, is
 *     RNS8_MI355X_DEFAULT_STREAM here (hipStreamLegacy's value).
 *   - Device pointers must be accessible from the context's device.
 *   - Range violations are reported through `d_status`: a device uint32_t
 *     that the caller zeroes before the call; the export kernel sets it
 *     nonzero if any cell violates the contract. The output contents of such
 *     a call are unspecified (the host exports keep `dst` untouched instead).
 *   - Validation failures return before anything is enqueued.
 */
#ifndef RNS8_MI355X_H
#define RNS8_MI355X_H

#include <stdint.h>

#include "rns8/rns8.h"

#ifdef __cplusplus
extern "C" {
#endif

#define RNS8_MI355X_DEFAULT_STREAM ((void*)1)

/* Prefix a plan created from `desc` would select (validation and prefix
 * selection of rns8_create_plan, reference api_plan_public_api.inc:3-73 and
 * api_plan_schedule.inc:263-278), without a context or device. Finite
 * semantics report 0. */
RNS8_API rns8_status rns8_mi355x_select_prefix(const rns8_gemm_desc* desc, uint32_t* out_prefix);

/* The schedule rns8_create_plan would build for `desc`, without a context or
 * device: the same results as rns8_get_plan_schedule_info and
 * rns8_get_plan_tile_schedule on that plan (reference rns8.h:683-691,
 * api_plan_schedule.inc:109-279, api_plan_public_api.inc:80-160), including
 * per-tile bounded schedules. `entries` may be NULL to query the count. */
RNS8_API rns8_status rns8_mi355x_plan_schedule(
    const rns8_gemm_desc* desc,
    rns8_plan_schedule_info* info,
    rns8_plan_tile_schedule_entry* entries,
    uint64_t capacity,
    uint64_t* written);

/* Device-source variants of rns8_pack_i64 / rns8_pack_u64 / rns8_pack_finite_u8
 * (reference rns8.h:848-911): `d_src` is device memory, row stride `ld`
 * elements. For exact-wide matrices the magnitude proof is the one the
 * reference's host pack builds (per-row and per-column maxima, sums,
 * absolute sums, extremes and deviation sums, reference exact_range.hpp
 * :52-78), computed on the GPU; so every later admission equals the one
 * the reference makes for the same values. At prefix 9 and up the call does
 * not synchronize; below, it reads max |x| back before writing anything. */
RNS8_API rns8_status rns8_mi355x_pack_i64_device(
    rns8_context* ctx,
    rns8_matrix* matrix,
    const int64_t* d_src,
    int64_t ld,
    uint64_t source_version,
    void* stream);
RNS8_API rns8_status rns8_mi355x_pack_u64_device(
    rns8_context* ctx,
    rns8_matrix* matrix,
    const uint64_t* d_src,
    int64_t ld,
    uint64_t source_version,
    void* stream);
RNS8_API rns8_status rns8_mi355x_pack_finite_u8_device(
    rns8_context* ctx,
    rns8_matrix* matrix,
    uint16_t modulus,
    const uint8_t* d_src,
    int64_t ld,
    uint64_t source_version,
    void* stream);

/* Asynchronous rns8_gemm_rns / rns8_gemm_finite_u8 (reference rns8.h:988,
 * 1098): same validation and admission, kernels enqueued on `stream`.
 * Exact-wide admission: the call decides on k * maxA * maxB, from maxima the
 * host already holds, and does not synchronize when that bound fits. When it
 * does not fit, the reference's refined bound (the minimum of its candidate
 * bounds for every output cell, from the operands' per-row and per-column
 * summaries) is computed on the device and read back before the call
 * returns: the call then synchronizes `stream`. */
RNS8_API rns8_status rns8_mi355x_gemm_rns_async(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_matrix* A,
    const rns8_matrix* B,
    rns8_matrix* C,
    rns8_workspace* workspace,
    void* stream);
RNS8_API rns8_status rns8_mi355x_gemm_finite_u8_async(
    rns8_context* ctx,
    const rns8_plan* plan,
    uint16_t modulus,
    const rns8_matrix* A,
    const rns8_matrix* B,
    rns8_matrix* C,
    rns8_workspace* workspace,
    void* stream);

/* rns8_mi355x_gemm_rns_async for bounded int64 / uint64 plans (global or
 * per-tile bounds) without a workspace, for callers that cannot allocate:
 * code under HIP graph capture, tight serving loops, harnesses that forbid
 * allocation. No counterpart in the reference. The call allocates nothing,
 * on the device or the host: split-K residues (shapes with few output tiles
 * and a long K) go to a static per-device scratch array of 4 MiB that the
 * library holds until the process ends (its address is looked up when a
 * context is created). Plans whose split-K residues exceed 4 MiB return
 * RNS8_WORKSPACE_TOO_SMALL;
 * exact-wide plans return RNS8_UNSUPPORTED_BACKEND (their admission may read
 * a device bound back and keeps its proofs in host memory). Every call on one device shares that device's
 * scratch: calls that overlap on one device (on different streams, or from
 * several threads) race and must be ordered by the caller; calls ordered on
 * one stream do not. Results equal rns8_mi355x_gemm_rns_async's. */
RNS8_API rns8_status rns8_mi355x_gemm_rns_noalloc(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_matrix* A,
    const rns8_matrix* B,
    rns8_matrix* C,
    void* stream);

/* Stream-ordered rns8_gemm_rns_grouped / rns8_gemm_finite_u8_grouped
 * (reference rns8.h:1061-1065, 1139-1144): the same validation, the group
 * enqueued on `stream` as one persistent launch per 65536-K block and up to
 * 32 tasks. */
RNS8_API rns8_status rns8_mi355x_gemm_rns_grouped_async(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_grouped_gemm_task* tasks,
    uint32_t task_count,
    void* stream);
RNS8_API rns8_status rns8_mi355x_gemm_finite_u8_grouped_async(
    rns8_context* ctx,
    const rns8_plan* plan,
    uint16_t modulus,
    const rns8_grouped_gemm_task* tasks,
    uint32_t task_count,
    void* stream);

/* Fused native-input GEMM for bounded int64 / uint64 plans: C's residue
 * planes straight from native device operands (m x k at row stride lda, k x n
 * at row stride ldb, in elements), the pack folded into the GEMM's operand
 * loads, enqueued on `stream` (reference hip_direct_gemm_native_kernels.cuh:
 * 9-193, its native-operand GEMM behind the oneshot path,
 * hip_backend_gemm_native_prefix.inc). Offered for outputs small enough that
 * the product is split along K, with 16-byte aligned operands and even row
 * strides below 2^21 elements; returns RNS8_UNSUPPORTED_BACKEND otherwise
 * (such plans pack their operands once and multiply with rns8_gemm_rns). The
 * plan's declared bound covers the result exactly as for rns8_gemm_rns. */
RNS8_API rns8_status rns8_mi355x_gemm_native_i64_async(
    rns8_context* ctx,
    const rns8_plan* plan,
    const int64_t* d_A,
    int64_t lda,
    const int64_t* d_B,
    int64_t ldb,
    rns8_matrix* C,
    rns8_workspace* workspace,
    void* stream);
RNS8_API rns8_status rns8_mi355x_gemm_native_u64_async(
    rns8_context* ctx,
    const rns8_plan* plan,
    const uint64_t* d_A,
    int64_t lda,
    const uint64_t* d_B,
    int64_t ldb,
    rns8_matrix* C,
    rns8_workspace* workspace,
    void* stream);

/* Device-destination variants of the exports (reference rns8.h:1146-1242). */
RNS8_API rns8_status rns8_mi355x_export_i64_device(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_matrix* C,
    int64_t* d_dst,
    int64_t ld,
    uint32_t* d_status,
    void* stream);
RNS8_API rns8_status rns8_mi355x_export_u64_device(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_matrix* C,
    uint64_t* d_dst,
    int64_t ld,
    uint32_t* d_status,
    void* stream);
RNS8_API rns8_status rns8_mi355x_export_exact_wide_signed_limbs_device(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_matrix* C,
    uint64_t* d_dst,
    int64_t ld,
    uint32_t limb_count,
    uint32_t* d_status,
    void* stream);
RNS8_API rns8_status rns8_mi355x_export_exact_wide_unsigned_limbs_device(
    rns8_context* ctx,
    const rns8_plan* plan,
    const rns8_matrix* C,
    uint64_t* d_dst,
    int64_t ld,
    uint32_t limb_count,
    uint32_t* d_status,
    void* stream);
RNS8_API rns8_status rns8_mi355x_export_finite_u8_device(
    rns8_context* ctx,
    const rns8_plan* plan,
    uint16_t modulus,
    const rns8_matrix* C,
    uint8_t* d_dst,
    int64_t ld,
    void* stream);

/* Layout of a resident matrix's planes in HBM ("rns8_mi355x_planes_v1"):
 * plane p, row r, column c lives at d_planes + p*plane_pitch + r*row_pitch + c
 * as a centered int8 residue; padding bytes are zero. Lets device code read
 * or produce residue planes directly. */
RNS8_API rns8_status rns8_mi355x_get_matrix_planes(
    const rns8_matrix* matrix,
    void** d_planes,
    int64_t* row_pitch,
    int64_t* plane_pitch,
    uint32_t* plane_count);

/* One row or column of an exact-wide matrix's magnitude proof, as
 * little-endian 64-bit words (reference rns8_exact_axis_range,
 * internal.hpp:72-86). */
typedef struct rns8_mi355x_exact_axis {
  uint64_t max_magnitude[4]; /* unsigned 256-bit */
  uint64_t absolute_sum[4];  /* unsigned 256-bit */
  uint64_t sum[2];           /* signed 128-bit, two's complement */
  uint64_t minimum[2];       /* signed 128-bit */
  uint64_t maximum[2];       /* signed 128-bit */
  uint64_t deviation_sum[2]; /* unsigned 128-bit */
} rns8_mi355x_exact_axis;

#define RNS8_MI355X_EXACT_AXES_NATIVE 0u  /* a pack's summaries: every field */
#define RNS8_MI355X_EXACT_AXES_CARRIED 1u /* a GEMM result's: max_magnitude, absolute_sum */
#define RNS8_MI355X_EXACT_AXES_NONE 2u    /* no per-axis summaries */

/* The magnitude proof an exact-wide matrix carries into later GEMMs
 * (reference exact_range.hpp:51-171): its bound (max |x| of a packed
 * operand, the proven bound of a GEMM result) into bound[0..3] as an
 * unsigned 256-bit integer, the kind of its axes, and rows[desc.rows] /
 * cols[desc.cols] (either may be NULL; untouched for
 * RNS8_MI355X_EXACT_AXES_NONE). A result's own summaries are computed when
 * first needed, here on the context's stream. Synchronizes. No counterpart
 * in the reference's C API (its proof is internal state). Returns
 * RNS8_INVALID_ARGUMENT for matrices without an exact-wide proof. */
RNS8_API rns8_status rns8_mi355x_get_exact_proof(
    rns8_context* ctx,
    const rns8_matrix* matrix,
    uint64_t bound[4],
    uint32_t* axes_kind,
    rns8_mi355x_exact_axis* rows,
    rns8_mi355x_exact_axis* cols);

/* ---- operators of language models around the 8-bit product --------------------
 *
 * The linear layer in 8-bit integers with a scale for each token and each
 * channel, the norms around a residual block, and the log-probabilities of
 * given tokens, each with its gradients. No counterpart in the reference.
 * They share these rules:
 *   - Every operator takes its arguments in one struct: struct_size and
 *     abi_version as in the other structs of this library, device pointers,
 *     and row strides (ld*) in elements. The device writes only the columns
 *     named and reads no others of floating operands; 8-bit operands may be
 *     read in whole aligned 16-byte chunks, whose other bytes do not matter. A
 *     stride may be any value from the row length on, and no pointer needs more
 *     alignment than its element type. Outputs must not overlap inputs unless
 *     stated.
 *   - `dtype` is the type of the floating operands marked `dtype` below.
 *     Sums, statistics and scales are computed and kept in 32 bits; an output
 *     is rounded once, to nearest even.
 *   - A call enqueues kernels on `stream` (NULL: the context's own stream) and
 *     returns. It allocates nothing and never synchronizes, so it may be
 *     captured into a graph. Operators that need scratch memory take
 *     `workspace` and `workspace_bytes`; the size for a call comes from the
 *     `_workspace` query of its name (which reads the struct's sizes, strides
 *     and pointers, not device memory) and a smaller one returns
 *     RNS8_WORKSPACE_TOO_SMALL. A workspace holds nothing between calls; calls
 *     that may overlap need one each. It is 16-byte aligned.
 *   - A size of zero rows is a valid call that leaves nothing to do (gradients
 *     summed over rows are then written as zeros).
 *   - Missing pointers, negative sizes, strides below the row length, unknown
 *     types and flags return RNS8_INVALID_ARGUMENT; sizes past the limits
 *     stated return RNS8_UNSUPPORTED_BACKEND. Nothing is enqueued then.
 *   - The same inputs give the same bytes on every run: no result depends on
 *     the order in which workgroups finish. */
#define RNS8_MI355X_F32 0u
#define RNS8_MI355X_F16 1u
#define RNS8_MI355X_BF16 2u

/* Quantization to 8 bits. A row v of 32-bit values becomes bytes q in
 * [-127, 127] and one scale, v ~ q * scale:
 *   amax = max |v|, scale = amax / 127, q = round_to_even(v * (127 / amax)).
 * A row whose amax is below 2^-100 gives q = 0 and scale = 0. A row that holds
 * an infinity or a NaN gives q = 0 and scale = NaN, so that whatever is
 * computed from it is NaN too.
 *   - rns8_mi355x_quantize_rows: v = x[r][c] * multiplier[c], one scale for
 *     each of `rows` rows; q is rows x cols. Bytes from cols up to
 *     min(ldq, cols rounded up to 16) are written as zeros (so a product may
 *     take the padded length as its k).
 *   - rns8_mi355x_quantize_columns: v = x[r][c] * multiplier[r], one scale for
 *     each of `cols` columns; q is written transposed, cols x rows, with the
 *     same zeros after each of its rows. `sums`, if given, receives the sum of
 *     x over the rows for each column (the gradient of a bias).
 * cols >= 1; sizes below 2^31. */
typedef struct rns8_mi355x_quantize_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t rows;
  int64_t cols;
  const void* x; /* dtype, rows x cols */
  int64_t ldx;
  const float* multiplier; /* or NULL: 1 */
  int8_t* q;
  int64_t ldq;
  float* scale;
  float* sums;     /* quantize_columns only; or NULL */
  void* workspace; /* quantize_columns only */
  uint64_t workspace_bytes;
} rns8_mi355x_quantize_args;

RNS8_API rns8_status rns8_mi355x_quantize_rows(rns8_context* ctx, const rns8_mi355x_quantize_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_quantize_columns(
    rns8_context* ctx,
    const rns8_mi355x_quantize_args* args,
    void* stream);
RNS8_API rns8_status rns8_mi355x_quantize_columns_workspace(const rns8_mi355x_quantize_args* args, uint64_t* bytes);

/* The product of 8-bit matrices with scales:
 *   out[i][j] = a_scale[i] * b_scale[j] * sum_k a[i][k] b(k, j) + bias[j],
 * the sum exact in integers for every k (bytes may be -128) and rounded once to
 * 32 bits, so a row of out is the same whatever other rows a call has. b is stored n x k (RNS8_MI355X_B_CHANNELS: one row for each output
 * channel, the usual layout of weights) or k x n (RNS8_MI355X_B_INNER). Any of
 * a_scale, b_scale (1) and bias (0) may be NULL. m, n >= 0, k >= 0 (an empty
 * sum is zero); m below 2^31, n below 2^31 - 256, k (and n where b is k x n) at
 * most 2^23 - 16, lda and ldb below 2^23. Products of more
 * than 64 rows read operands in place whose pointers and strides are multiples
 * of 16 and copy others into the workspace first, and one of the two where b is
 * n x k and k is no multiple of 16. Products of fewer rows may read in place
 * at any alignment. */
#define RNS8_MI355X_B_CHANNELS 0u
#define RNS8_MI355X_B_INNER 1u
typedef struct rns8_mi355x_gemm_i8_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t m;
  int64_t n;
  int64_t k;
  const int8_t* a; /* m x k */
  int64_t lda;
  const int8_t* b;
  int64_t ldb;
  uint32_t b_layout;
  uint32_t reserved; /* 0 */
  const float* a_scale; /* m, or NULL */
  const float* b_scale; /* n, or NULL */
  const float* bias;    /* n, or NULL */
  void* out;            /* dtype, m x n */
  int64_t ldo;
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_gemm_i8_args;

RNS8_API rns8_status rns8_mi355x_gemm_i8_scaled(rns8_context* ctx, const rns8_mi355x_gemm_i8_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_gemm_i8_scaled_workspace(const rns8_mi355x_gemm_i8_args* args, uint64_t* bytes);

/* A linear layer on floating activations: x's rows are quantized as by
 * rns8_mi355x_quantize_rows (no multiplier) and multiplied with 8-bit weights
 * w (n x k, w_scale[n]):
 *   out[i][j] = x_scale[i] * w_scale[j] * sum_k q[i][k] w[j][k] + bias[j].
 * x_q (m x k at stride ldq, zeros after each row as there) and x_scale[m] receive
 * the quantized rows if given (both or neither): what the backward pass reads.
 * k >= 1; n below 2^31 - 256, k below 2^23 - 16, ldw and ldq below 2^23. */
typedef struct rns8_mi355x_linear_i8_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t m;
  int64_t n;
  int64_t k;
  const void* x; /* dtype, m x k */
  int64_t ldx;
  const int8_t* w; /* n x k */
  int64_t ldw;
  const float* w_scale; /* n */
  const float* bias;    /* n, or NULL */
  void* out;            /* dtype, m x n */
  int64_t ldo;
  int8_t* x_q; /* m x k, or NULL */
  int64_t ldq;
  float* x_scale; /* m, or NULL */
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_linear_i8_args;

RNS8_API rns8_status rns8_mi355x_linear_i8(rns8_context* ctx, const rns8_mi355x_linear_i8_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_linear_i8_workspace(const rns8_mi355x_linear_i8_args* args, uint64_t* bytes);

/* Its gradients, also in 8-bit products, the roundings to 8 bits passed
 * straight through: dy's rows are quantized with the channels' scales folded
 * in, its columns with the tokens' scales folded in, and
 *   dx[i][k] = g_scale[i] * sum_j gq[i][j] w[j][k],   gq, g_scale: rows of dy[i][j] * w_scale[j]
 *   dw[j][k] = h_scale[j] * sum_i hq[i][j] x_q[i][k], hq, h_scale: columns of dy[i][j] * x_scale[i]
 *   dbias[j] = sum_i dy[i][j].
 * dw is the gradient of the weights w * w_scale. dx, dw and dbias may each be
 * NULL (not all three); x_q and x_scale may be NULL without dw, w and w_scale
 * without dx. With dx n, and with dw or dbias m, stays below 2^23 - 16, and with dx
 * or dw k at most that; ldq and ldw below 2^23. */
typedef struct rns8_mi355x_linear_i8_backward_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t m;
  int64_t n;
  int64_t k;
  const void* dy; /* dtype, m x n */
  int64_t lddy;
  const int8_t* x_q; /* m x k */
  int64_t ldq;
  const float* x_scale; /* m */
  const int8_t* w;      /* n x k */
  int64_t ldw;
  const float* w_scale; /* n */
  void* dx;             /* dtype, m x k */
  int64_t lddx;
  float* dw; /* n x k */
  int64_t lddw;
  float* dbias; /* n */
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_linear_i8_backward_args;

RNS8_API rns8_status rns8_mi355x_linear_i8_backward(
    rns8_context* ctx,
    const rns8_mi355x_linear_i8_backward_args* args,
    void* stream);
RNS8_API rns8_status rns8_mi355x_linear_i8_backward_workspace(
    const rns8_mi355x_linear_i8_backward_args* args,
    uint64_t* bytes);

/* The norms after and before a residual block, for each row (token):
 *   f = x * r1 * post_weight,  r1 = 1 / sqrt(mean(x^2) + eps)   (RNS8_MI355X_NORM_POST; otherwise f = x)
 *   h = residual_scale * residual + branch_scale * gate * f
 *   y = h * r2 * pre_weight,   r2 = 1 / sqrt(mean(h^2) + eps)   (RNS8_MI355X_NORM_PRE)
 * x is the block's output, h the residual stream after it and y what the next
 * block reads; y is computed from h before h is rounded. residual, gate and
 * the weights may be NULL (0, 1 and 1). gate has one row for all tokens
 * (ldgate == 0) or one for each. With NORM_PRE at least one of y and q is
 * given: q (stride ldq) and q_scale receive y quantized as by
 * rns8_mi355x_quantize_rows. h may be NULL with NORM_PRE, and may be x or
 * residual itself (in place, at equal strides). rstd, if given, receives r1
 * (rows values) and then r2 (rows values) for the backward pass. Rows are at
 * most 32768 long. Their sums of squares are 32-bit values: one past 2^128 gives
 * r = 0, and with eps = 0 one that vanishes (values below 1e-22) r = infinity. */
#define RNS8_MI355X_NORM_POST 1u
#define RNS8_MI355X_NORM_PRE 2u
typedef struct rns8_mi355x_block_norm_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t rows;
  int64_t cols;
  uint32_t flags;
  float eps;
  float branch_scale;
  float residual_scale;
  const void* x; /* dtype, rows x cols */
  int64_t ldx;
  const void* residual; /* dtype, rows x cols, or NULL */
  int64_t ldresidual;
  const void* gate; /* dtype, or NULL */
  int64_t ldgate;
  const void* post_weight; /* dtype, cols, or NULL */
  const void* pre_weight;  /* dtype, cols, or NULL */
  void* h;                 /* dtype, rows x cols */
  int64_t ldh;
  void* y; /* dtype, rows x cols, or NULL */
  int64_t ldy;
  int8_t* q; /* rows x cols, or NULL */
  int64_t ldq;
  float* q_scale; /* rows; with q */
  float* rstd;    /* 2 x rows, or NULL */
} rns8_mi355x_block_norm_args;

RNS8_API rns8_status rns8_mi355x_block_norm(
    rns8_context* ctx,
    const rns8_mi355x_block_norm_args* args,
    void* stream);

/* Its gradients, from the forward pass's inputs and rstd, dy (the gradient of
 * y; with NORM_PRE) and dh (the gradient that h receives from elsewhere, or
 * NULL: 0; one of dy and dh is needed). h is computed again from the inputs.
 * Outputs, each NULL if not wanted: dx, dresidual and, where the gate has a row
 * for each token, dgate in dtype; dgate of a one-row gate, dpost_weight and
 * dpre_weight summed over the rows in 32 bits. */
typedef struct rns8_mi355x_block_norm_backward_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t rows;
  int64_t cols;
  uint32_t flags;
  float eps;
  float branch_scale;
  float residual_scale;
  const void* x;
  int64_t ldx;
  const void* residual;
  int64_t ldresidual;
  const void* gate;
  int64_t ldgate;
  const void* post_weight;
  const void* pre_weight;
  const float* rstd; /* 2 x rows */
  const void* dy;    /* dtype, rows x cols, or NULL */
  int64_t lddy;
  const void* dh; /* dtype, rows x cols, or NULL */
  int64_t lddh;
  void* dx; /* dtype, rows x cols */
  int64_t lddx;
  void* dresidual; /* dtype, rows x cols */
  int64_t lddresidual;
  void* dgate; /* float[cols] (ldgate == 0) or dtype, rows x cols */
  int64_t lddgate;
  float* dpost_weight; /* cols */
  float* dpre_weight;  /* cols */
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_block_norm_backward_args;

RNS8_API rns8_status rns8_mi355x_block_norm_backward(
    rns8_context* ctx,
    const rns8_mi355x_block_norm_backward_args* args,
    void* stream);
RNS8_API rns8_status rns8_mi355x_block_norm_backward_workspace(
    const rns8_mi355x_block_norm_backward_args* args,
    uint64_t* bytes);

/* Log-probabilities of given tokens, for each row of logits, z = scale * logits:
 *   lse = log(sum exp(z)), logp = z[target] - lse, entropy = -sum p log p, p = exp(z - lse),
 * and the `top` most likely tokens: top_ids (int32) in falling order of their
 * logits, equal ones (0 and -0 are equal) by rising index, and top_logp, their
 * log-probabilities. A logit of -infinity is a token ruled out: it takes no
 * part in the sums. A row of nothing else gives lse = -infinity, logp =
 * -infinity and entropy 0. A NaN or +infinity in a row makes its lse, logp and
 * entropy NaN; NaNs come first among the alternatives. A target below 0 or
 * not below vocab asks for none: logp is 0. logp, entropy, lse and the
 * alternatives may each be NULL (targets too, without logp). top <= 64 and
 * top <= vocab; vocab below 2^31; scale finite and above 0. */
typedef struct rns8_mi355x_logprobs_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t rows;
  int64_t vocab;
  const void* logits; /* dtype, rows x vocab */
  int64_t ldl;
  const int64_t* targets; /* rows */
  float scale;
  uint32_t top;
  float* logp;      /* rows */
  float* entropy;   /* rows */
  float* lse;       /* rows */
  int32_t* top_ids; /* rows x top, dense */
  float* top_logp;  /* rows x top, dense */
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_logprobs_args;

RNS8_API rns8_status rns8_mi355x_token_logprobs(
    rns8_context* ctx,
    const rns8_mi355x_logprobs_args* args,
    void* stream);
RNS8_API rns8_status rns8_mi355x_token_logprobs_workspace(const rns8_mi355x_logprobs_args* args, uint64_t* bytes);

/* The gradient of logp and entropy, from the forward pass's lse and entropy:
 *   dlogits[v] = scale * (dlogp * ([v = target] - p[v]) - dentropy * p[v] * (log p[v] + entropy)).
 * Ruled-out tokens and rows without a finite lse from ruled-out tokens alone
 * get 0; a row whose lse is NaN gets NaN throughout; a row whose target asks for none has no gradient from logp. dlogp and
 * dentropy may be NULL (0; not both); entropy may be NULL without dentropy.
 * dlogits may be logits itself, at an equal stride. */
typedef struct rns8_mi355x_logprobs_backward_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t rows;
  int64_t vocab;
  const void* logits; /* dtype, rows x vocab */
  int64_t ldl;
  const int64_t* targets; /* rows; with dlogp */
  float scale;
  uint32_t reserved;       /* 0 */
  const float* lse;        /* rows */
  const float* entropy;    /* rows; with dentropy */
  const float* dlogp;      /* rows, or NULL */
  const float* dentropy;   /* rows, or NULL */
  void* dlogits;           /* dtype, rows x vocab */
  int64_t lddl;
} rns8_mi355x_logprobs_backward_args;

RNS8_API rns8_status rns8_mi355x_token_logprobs_backward(
    rns8_context* ctx,
    const rns8_mi355x_logprobs_backward_args* args,
    void* stream);

/* ---- operators on 4-bit microscaled matrices ("MX4") ---------------------------
 *
 * A block of 32 neighbouring values of a row (the last of a row may have fewer)
 * shares one power of two, and each value has 4 bits:
 *   v ~ level * 2^e,  level in {0, 1/2, 1, 3/2, 2, 3, 4, 6} with a sign,
 *   e = floor(log2(max |v|)) - 2, at least -127,
 * level the nearest to v / 2^e, of two as near the one with the even code, at most
 * 6. A code is the level's index above plus 8 for a sign, e is held as the byte e +
 * 127. A block that holds an infinity or a NaN gives codes 0 and the byte 255,
 * which makes whatever is computed from it NaN. (These are the OCP microscaling
 * formats' MXFP4 elements and scales.)
 *
 * An MX4 matrix of rows x cols is one buffer of RNS8_MI355X_MX4_BYTES(rows, cols)
 * bytes, 16-byte aligned, in the order in which the matrix cores take it: units
 * of 16 rows x 256 columns, 2176 bytes each, the units of 16 rows one after the
 * other. Column c of row r of a unit has its code in the 4 bits (the low ones
 * where c is even) of byte 1024 (c / 128) + 16 L + (c % 32) / 2 and its scale in
 * byte 2048 + 2 L + c / 128, L = r % 16 + 16 ((c % 128) / 32). What lies past the
 * matrix in its units is zeros. 16 rows at a multiple of 16 are themselves an MX4
 * matrix, and matrices of as many rows, a multiple of 16, one after the other are one of
 * all their rows: one call packs, rounds or reads them.
 *
 * The rules of the operators above hold here too. rows and cols of an MX4 matrix
 * are below 2^31 - 256 and those that a product sums over at most 2^23. */
#define RNS8_MI355X_MX4_UNIT 2176
#define RNS8_MI355X_MX4_BYTES(rows, cols) \
  (((uint64_t)(rows) + 15u) / 16u * (((uint64_t)(cols) + 255u) / 256u) * RNS8_MI355X_MX4_UNIT)

/* Floating rows to MX4 and back.
 *   - rns8_mi355x_quantize_mx4: q receives x (rows x cols), q_t its transpose (cols
 *     x rows, blocks along the rows of x); either may be NULL, not both.
 *   - rns8_mi355x_dequantize_mx4: x receives the values of q (rows x cols), NaN
 *     for blocks whose scale is 255; q_t is NULL.
 * Values that MX4 holds are unchanged by a quantization (their blocks' scales may
 * be smaller than they were). rows >= 0, cols >= 1. */
typedef struct rns8_mi355x_mx4_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t rows;
  int64_t cols;
  void* x; /* dtype, rows x cols; quantize_mx4 only reads it */
  int64_t ldx;
  uint8_t* q;   /* MX4, rows x cols */
  uint8_t* q_t; /* MX4, cols x rows */
} rns8_mi355x_mx4_args;

RNS8_API rns8_status rns8_mi355x_quantize_mx4(rns8_context* ctx, const rns8_mi355x_mx4_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_dequantize_mx4(rns8_context* ctx, const rns8_mi355x_mx4_args* args, void* stream);

/* Rows as checkpoints hold them into q: `data` has the codes, two to a byte (an
 * even column in the low bits; ceil(cols / 2) bytes of a row are read), `scale`
 * the scales' bytes (ceil(cols / 32) of a row). Both have strides in bytes and any
 * alignment. rows >= 0, cols >= 1. */
typedef struct rns8_mi355x_pack_mx4_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype; /* 0: there are no floating operands */
  int64_t rows;
  int64_t cols;
  const uint8_t* data;
  int64_t ldd;
  const uint8_t* scale;
  int64_t lds;
  uint8_t* q; /* MX4, rows x cols */
} rns8_mi355x_pack_mx4_args;

RNS8_API rns8_status rns8_mi355x_pack_mx4(rns8_context* ctx, const rns8_mi355x_pack_mx4_args* args, void* stream);

/* The product of MX4 matrices:
 *   out[i][j] = sum_k a[i][k] b[j][k] + bias[j],
 * b with one row for each output channel. Products of two codes are exact, sums
 * are 32-bit. m, n, k >= 0 (an empty sum is zero). */
typedef struct rns8_mi355x_gemm_mx4_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t m;
  int64_t n;
  int64_t k;
  const uint8_t* a;  /* MX4, m x k */
  const uint8_t* b;  /* MX4, n x k */
  const float* bias; /* n, or NULL */
  void* out;         /* dtype, m x n */
  int64_t ldo;
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_gemm_mx4_args;

RNS8_API rns8_status rns8_mi355x_gemm_mx4(rns8_context* ctx, const rns8_mi355x_gemm_mx4_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_gemm_mx4_workspace(const rns8_mi355x_gemm_mx4_args* args, uint64_t* bytes);

/* A linear layer: x's rows rounded as by rns8_mi355x_quantize_mx4, times MX4
 * weights w (n x k), with bias. k >= 1. */
typedef struct rns8_mi355x_linear_mx4_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t m;
  int64_t n;
  int64_t k;
  const void* x; /* dtype, m x k */
  int64_t ldx;
  const uint8_t* w;  /* MX4, n x k */
  const float* bias; /* n, or NULL */
  void* out;         /* dtype, m x n */
  int64_t ldo;
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_linear_mx4_args;

RNS8_API rns8_status rns8_mi355x_linear_mx4(rns8_context* ctx, const rns8_mi355x_linear_mx4_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_linear_mx4_workspace(const rns8_mi355x_linear_mx4_args* args, uint64_t* bytes);

/* Its gradients, in MX4 products too, the roundings passed straight through. R is
 * the rounding along rows, so that each product sums over blocks of its own:
 *   dx = R(dy) R(w^T)^T, R(w^T) the MX4 matrix w_t (k x n),
 *   dw = R(dy^T) R(x^T)^T,  dbias[j] = sum_i dy[i][j].
 * dx, dw and dbias may each be NULL (not all three); x may be NULL without dw, w_t
 * without dx. n, k >= 1. */
typedef struct rns8_mi355x_linear_mx4_backward_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t m;
  int64_t n;
  int64_t k;
  const void* dy; /* dtype, m x n */
  int64_t lddy;
  const void* x; /* dtype, m x k */
  int64_t ldx;
  const uint8_t* w_t; /* MX4, k x n */
  void* dx;           /* dtype, m x k */
  int64_t lddx;
  float* dw; /* n x k */
  int64_t lddw;
  float* dbias; /* n */
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_linear_mx4_backward_args;

RNS8_API rns8_status rns8_mi355x_linear_mx4_backward(
    rns8_context* ctx,
    const rns8_mi355x_linear_mx4_backward_args* args,
    void* stream);
RNS8_API rns8_status rns8_mi355x_linear_mx4_backward_workspace(
    const rns8_mi355x_linear_mx4_backward_args* args,
    uint64_t* bytes);

/* A mixture-of-experts layer for few tokens, its experts' weights MX4 matrices:
 *   scores[t][e] = sum_c x[t][c] router[e][c]              (64-bit sums, then 32 bits)
 *   ids[t]: the `top` experts of the largest scores, falling, of equal ones the
 *     lower index first (a NaN counts as the largest),
 *   weights[t][s] = exp(scores[t][ids[t][s]]) / sum_e exp(scores[t][e]), with
 *     RNS8_MI355X_EXPERTS_NORMALIZE the sum over the chosen experts alone,
 *   out[t] = sum_s weights[t][s] down[e] (silu(gate[e] x[t]) * (up[e] x[t])),  e = ids[t][s],
 *   silu(v) = v / (1 + exp(-v)).
 * x is not rounded: few tokens wait for the weights alone. Sums are 32-bit; x and the
 * hidden values keep their bits (up to 24, of those worth 2^-133 and more), and a
 * weight past float's range is infinite. Without a router, ids and weights are inputs:
 * an id below 0 or not below `experts` is a slot that adds nothing (its expert is
 * elsewhere), and an expert that a token has twice counts twice. With one they are
 * outputs, and each may be NULL. gate and up hold one inner x width matrix for each
 * expert, down one width x inner, one after the other. A score that is NaN or
 * +infinity, or a value of a token that is not finite, makes that token's row alone NaN
 * (or infinite); an expert whose score is -infinity beside a finite one has weight 0.
 * tokens at most 64, experts at most 1024, top at most 16 and at most `experts`, width
 * and inner at most 65536. */
#define RNS8_MI355X_EXPERTS_NORMALIZE 1u
typedef struct rns8_mi355x_experts_mx4_args {
  uint64_t struct_size;
  uint32_t abi_version;
  uint32_t dtype;
  int64_t tokens;
  int64_t experts;
  int64_t width;
  int64_t inner;
  uint32_t top;
  uint32_t flags;
  const void* x; /* dtype, tokens x width */
  int64_t ldx;
  const void* router; /* dtype, experts x width, or NULL */
  int64_t ldrouter;
  const uint8_t* gate; /* MX4, experts of inner x width */
  const uint8_t* up;   /* MX4, experts of inner x width */
  const uint8_t* down; /* MX4, experts of width x inner */
  void* out;           /* dtype, tokens x width */
  int64_t ldo;
  int32_t* ids;   /* tokens x top, dense */
  float* weights; /* tokens x top, dense */
  void* workspace;
  uint64_t workspace_bytes;
} rns8_mi355x_experts_mx4_args;

RNS8_API rns8_status rns8_mi355x_experts_mx4(rns8_context* ctx, const rns8_mi355x_experts_mx4_args* args, void* stream);
RNS8_API rns8_status rns8_mi355x_experts_mx4_workspace(const rns8_mi355x_experts_mx4_args* args, uint64_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* RNS8_MI355X_H */
