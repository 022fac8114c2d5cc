/*
 * gyro_ops: operators around the MoE layers, on the engine of gyro_moe.h (libgyro_moe.so).
 *
 * No counterpart in the reference: products with 4-bit matrices, the residual step's norms and the log
 * probabilities of an answer, on rows in device memory of the engine's GPU. They need no layer. A call queues its
 * launches on `stream` and does not wait, allocate or copy; `stream` is a hipStream_t of the engine's device as HIP
 * means it, and the caller's current device is left as it was. NULL is the device's null stream. (To
 * gm_forward_decode_noalloc NULL is the engine's compute stream, which is not ordered with the null stream, and the
 * null stream hipStreamLegacy.) gm_linear, gm_block_norm and gm_logprobs may be captured into a HIP graph; a kernel that no
 * call has used yet is loaded by its first call, which a capture refuses, so call once (or gm_load_operators) before.
 * The calls that load, add or release wait and allocate, and belong outside captures. n = 0 does nothing. Calls on one
 * engine are serialised by the caller, as all of gyro_moe.h's; what they queue may overlap where its outputs and
 * workspaces are apart. All return 0 or a negative code; gm_last_error describes the failure.
 */
#ifndef GYRO_OPS_H
#define GYRO_OPS_H

#include "gyro_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { GM_F32 = 0, GM_BF16 = 1, GM_F16 = 2 };

/* Rows in device memory: row t starts `stride` values after row t - 1; values of a row are neighbours. Any
 * alignment to the type's size is taken (16-byte aligned rows are read faster). Output rows must not overlap. */
typedef struct gm_rows {
    void *data;
    uint64_t stride;
    uint32_t type; /* GM_F32, GM_BF16, GM_F16 */
    uint32_t reserved;
} gm_rows;

/* Loads the operators' kernels that are not loaded yet. */
GM_API int gm_load_operators(gm_engine *e);

/* A 4-bit matrix W of `rows` rows of `cols` values, in groups of `group` neighbours of a row that share a scale s
 * and, where the format has one, a minimum m (binary16 both), of 4-bit values q:
 *   GM_MATRIX_Q4_0    GGUF Q4_0 blocks at quants: W = s (q - 8), group 32
 *   GM_MATRIX_Q4_1    GGUF Q4_1 blocks at quants: W = s q + m, group 32
 *   GM_MATRIX_Q4      quants [rows][cols / 2], value 2 i in the low bits of byte i; scales and mins
 *                     [rows][cols / group], group 32, 64 or 128: W = s q + m, or s (q - 8) with mins NULL
 * cols is a multiple of group. With up_quants given (up_scales and up_mins as the format has them) the matrix
 * is a gated pair of two such matrices. Host memory, read before the call returns. */
enum { GM_MATRIX_Q4_0 = 0, GM_MATRIX_Q4_1 = 1, GM_MATRIX_Q4 = 2 };
typedef struct gm_matrix_desc {
    uint32_t format, rows, cols, group;
    const void *quants, *scales, *mins;
    const void *up_quants, *up_scales, *up_mins;
} gm_matrix_desc;
/* Uploads a matrix (at most 4 GiB in the device's layout: half a byte per value and the scales, of rows in
 * sixteens and columns in 128s) and returns its index. */
GM_API int gm_add_matrix(gm_engine *e, const gm_matrix_desc *desc, uint32_t *out_index);
/* Frees a matrix once the device's work is done; its index may come again. A graph captured with it may not be
 * replayed any more. */
GM_API int gm_release_matrix(gm_engine *e, uint32_t matrix);
/* y[t] = act(scale W x[t]) for n tokens, x [n][cols], y [n][rows]; with accumulate, the sum is added to y
 * (after act, in fp32). A gated pair: y[t] = scale silu(G x[t]) * (U x[t]), act GM_ACT_NONE. Activations and sums
 * are fp32 whatever the types (products are exact in them); y is rounded once. Activations
 * are below 2^116 in magnitude (a group's sums of products with 0 .. 31 stay in range then); of fp32 and bf16 ones below
 * 2^-103 what is below 2^-126 counts as zero. Of a token with an activation that is not finite no output is (a NaN or an
 * infinity). Two or more rows of x are at most 2^24 values apart, n at most 2^18; y must not overlap x. */
enum { GM_ACT_NONE = 0, GM_ACT_SILU = 1, GM_ACT_SIGMOID = 2 };
GM_API int gm_linear(gm_engine *e, uint32_t matrix, const gm_rows *x, uint32_t n, const gm_rows *y, uint32_t act,
                     uint32_t accumulate, float scale, void *stream);

/* The residual step between two blocks, on n rows of E <= 16384 values:
 *   a = h / sqrt(mean(h^2) + post_eps) * post_weight  with `post`, else h (no weight: ones)
 *   v = x + scale gate a             (no h: v = x)
 *   out = v;  normed = v / sqrt(mean(v^2) + pre_eps) * pre_weight
 * in fp32, normed from the unrounded v. gate: GM_GATE_NONE; one value per token (value t at t * stride), per
 * channel [E], or per value; through a sigmoid with gate_act GM_ACT_SIGMOID. out or normed may be absent (data NULL),
 * not both. out may be x's rows, normed h's, of the same type and stride (another layout at the same address is refused);
 * outputs overlap nothing else. Weights fp32 [E], on the device. */
enum { GM_GATE_NONE = 0, GM_GATE_TOKEN = 1, GM_GATE_CHANNEL = 2, GM_GATE_VALUE = 3 };
typedef struct gm_block_norm_desc {
    uint32_t E, post, gate_kind, gate_act;
    gm_rows h, x, out, normed, gate;
    const float *post_weight, *pre_weight;
    float post_eps, pre_eps, scale;
    uint32_t reserved;
} gm_block_norm_desc;
GM_API int gm_block_norm(gm_engine *e, const gm_block_norm_desc *desc, uint32_t n, void *stream);

/* Of each of n rows of V logits x, with z = scale x (scale > 0: an inverse temperature) and p = softmax(z), in fp32:
 *   logprobs[t][j]  log p of tokens[t][j] (int32, or int64 with tokens_64), j < given <= 64: 0 for a
 *                   negative token (none given), NaN for one >= V
 *   entropy[t]      -sum p log p (absent: NULL)
 *   top_ids[t][k], top_logprobs[t][k]  the `top` <= 64 largest logits, equal ones by id, and their log p
 * A logit of -infinity has p = 0. A row of nothing but those has log p -infinity everywhere and entropy 0; one with a NaN or
 * +infinity has NaN for both (top_ids still order the logits, NaNs first). Strides count values. The
 * workspace (256-byte aligned; may be NULL where gm_logprobs_workspace is 0) holds nothing between calls; calls that may
 * overlap, replayed graphs among them, take one each. */
typedef struct gm_logprobs_desc {
    gm_rows logits;
    uint32_t V, given, top, tokens_64;
    float scale;
    uint32_t reserved;
    const void *tokens;
    uint64_t tokens_stride;
    float *logprobs;
    uint64_t logprobs_stride;
    float *entropy;
    uint32_t *top_ids;
    float *top_logprobs;
    uint64_t top_stride;
    void *workspace;
    uint64_t workspace_bytes;
} gm_logprobs_desc;
/* Bytes that suffice for every call of up to n rows (few rows are split over more groups than many, and take more of them
 * than n rows may). */
GM_API uint64_t gm_logprobs_workspace(uint32_t n, uint32_t V, uint32_t top);
GM_API int gm_logprobs(gm_engine *e, const gm_logprobs_desc *desc, uint32_t n, void *stream);

#ifdef __cplusplus
}
#endif
#endif
