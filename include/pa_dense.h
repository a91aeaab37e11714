/*
 * pa_dense.h -- the dense side around the paged-attention path, for an
 * end-to-end decoder step: RMSNorm or LayerNorm (with the residual add fused
 * in), the SwiGLU activation, and the linear projections (skinny-M for
 * decode steps, a tiled GEMM for prompt chunks), and the same projections over
 * MXFP8 rows and weights.  Conventions as pa.h (device
 * pointers, stream-ordered, PA_OK or a negative pa_status); dtype
 * PA_DTYPE_F32 or PA_DTYPE_BF16, math in f32.
 */
#ifndef VLLM_LITE_AMD_PA_DENSE_H
#define VLLM_LITE_AMD_PA_DENSE_H

#include "pa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* RmsNorm::forward (crates/model/src/components/norm/rms_norm.rs:26-50) with
 * the decoder block's residual add fused in front
 * (crates/model/src/components/decoder_block/mod.rs:157-198):
 *   if add != NULL:  residual[r] += add[r]        (rounded to dtype, in place)
 *   out[r] = residual[r] / sqrt(mean(residual[r]^2) + eps) * weight
 * residual / add / out [rows, hidden] (contiguous), weight [hidden]. */
int32_t pa_rms_norm(void* out, void* residual, const void* add, const void* weight,
                    int32_t rows, int32_t hidden, float eps, int32_t dtype, pa_stream_t stream);

/* LnLayerNorm::forward (crates/model/src/components/norm/layer_norm.rs:26-39,
 * candle_nn::LayerNorm with the mean removed and an affine bias), the norm the
 * reference's decoder blocks are built with
 * (crates/model/src/components/decoder_block/factory.rs:42-46), with the
 * residual add fused in front as in pa_rms_norm:
 *   if add != NULL:  residual[r] += add[r]        (rounded to dtype, in place)
 *   mu = mean(residual[r]);  var = mean((residual[r] - mu)^2)
 *   out[r] = (residual[r] - mu) / sqrt(var + eps) * weight + bias
 * bias may be NULL (the zero bias).  Shapes as pa_rms_norm. */
int32_t pa_layer_norm(void* out, void* residual, const void* add, const void* weight,
                      const void* bias, int32_t rows, int32_t hidden, float eps, int32_t dtype,
                      pa_stream_t stream);

/* The SwiGLU activation of swiglu_forward
 * (crates/model/src/components/mlp/swiglu.rs:18-31) on a fused gate|up
 * projection output:  out[r][i] = silu(gate_up[r][i]) * gate_up[r][inter + i],
 * silu(x) = x / (1 + e^-x).  gate_up [rows, 2 * inter], out [rows, inter]. */
int32_t pa_silu_mul(void* out, const void* gate_up, int32_t rows, int32_t inter, int32_t dtype,
                    pa_stream_t stream);

/* Activation epilogues and flags of pa_linear. */
enum { PA_ACT_NONE = 0, PA_ACT_SILU_MUL = 1 };
enum { PA_LINEAR_RMS_IN = 1, PA_LINEAR_ADD_OUT = 2 };

/* The decoder's linear projections for the few-row batches of a decode step
 * (candle_nn::Linear as the reference's attention and MLP use it: the QKV
 * projection with bias, crates/model/src/components/attention/rope_gqa.rs:261-302,
 * the output projection, and the MLP's gate/up/down projections,
 * crates/model/src/components/mlp/swiglu.rs:18-31), plus the tied LM head:
 *   act PA_ACT_NONE:      out[r][n] = sum_k x[r][k] * weight[n][k] (+ bias[n])
 *   act PA_ACT_SILU_MUL:  weight is the fused gate|up matrix [2 N, K] and
 *                         out[r][n] = silu(g) * u with g, u the gate / up
 *                         outputs of column n rounded to bf16 (pa_silu_mul on
 *                         the unfused projection's output); bias must be NULL.
 * x [rows, K], weight [N or 2 N, K], out [rows, N], all contiguous bf16 and
 * 16-byte aligned, bias [N] or NULL; K (in_features) and N (out_features)
 * as the kernel below needs.  f32 accumulation.
 * packed = 1: weight is in the layout of pa_linear_pack (rows N or 2 N).
 * flags (0 or a combination):
 *   PA_LINEAR_RMS_IN   the rows of x are RMS-normalised on the fly: the result
 *                      is multiplied by 1 / sqrt(mean_k(x[r][k]^2) + eps) (the
 *                      decoder's RMSNorm, crates/model/src/components/norm/
 *                      rms_norm.rs:26-50, in front of the projection); the
 *                      norm weight is folded into the weight's columns by
 *                      pa_linear_pack's col_scale;
 *   PA_LINEAR_ADD_OUT  out is the residual stream and is updated in place,
 *                      out[r][n] = bf16(out[r][n] + bf16(y[r][n])) (the
 *                      decoder block's residual add); not with SwiGLU.
 * workspace: NULL, or pa_linear_workspace_size() bytes (256-byte aligned)
 * whose first bytes hold counters that must be ZERO before the first call
 * that uses it (e.g. hipMemset once after allocating it); every call leaves
 * them zero again.  With it, long-K projections over few output tiles (the
 * MLP down projection of a decode step) split K over several workgroups per
 * tile, the last to finish summing the partial tiles in a fixed order (the
 * result does not depend on their timing).  Calls that may run at the same
 * time need distinct workspaces.  Without it one workgroup takes each tile.
 * Three kernels behind the one entry point:
 *  - rows <= 64 (decode steps), packed or row-major weights: the skinny
 *    kernel, where the weights dominate the traffic (they are re-read once
 *    per 32 rows); K a multiple of 32, N of 16;
 *  - rows <= 32, packed weights of at least 65,536 rows (the LM head), no
 *    bias, activation or residual add, K <= 992: a persistent kernel that
 *    holds X in LDS and streams the weight tiles over all CUs (the
 *    workspace is not used);
 *  - rows > 64 (prompt chunks), or an N the skinny tiles do not divide, with
 *    row-major weights, no PA_LINEAR_RMS_IN and K a multiple of 64: a tiled
 *    GEMM on the matrix cores (six tilings from 64 x 64 to 256 x 256 output
 *    tiles, chosen from rows, N and K; K staged through LDS in steps of 64
 *    or 128; any N, with SwiGLU a multiple of 64; the workspace is not used).
 *    Some tilings sum K in two or four interleaved parts, so the order of a
 *    row's f32 sums, and with it the last bit of an output, may depend on
 *    rows, N and K (equal calls give equal bits).
 * Other shapes return PA_ERR_UNSUPPORTED, as does any dtype but bf16. */
int32_t pa_linear(void* out, const void* x, const void* weight, const void* bias, int32_t rows,
                  int32_t out_features, int32_t in_features, int32_t act, int32_t packed,
                  int32_t flags, float eps, void* workspace, size_t workspace_bytes,
                  int32_t dtype, pa_stream_t stream);

/* Workspace bytes pa_linear's K split uses for this shape (0: none; the call
 * then needs no workspace).  No reference counterpart. */
size_t pa_linear_workspace_size(int32_t rows, int32_t out_features, int32_t in_features,
                                int32_t act);

/* Repacks a row-major bf16 weight [rows, cols] (rows a multiple of 16, cols
 * of 32) into the fragment order pa_linear reads with packed = 1: every
 * 16-row x 32-column MFMA operand fragment becomes one contiguous kilobyte,
 * the fragments of a 16-row tile consecutive along the columns.  col_scale
 * [cols] (bf16) or NULL: each column is multiplied by it (rounded to bf16),
 * which folds a norm weight in front of the projection.  Same size as the
 * input; packed and weight must not overlap.  No reference counterpart: a
 * load-time layout step for the weights pa_linear streams. */
int32_t pa_linear_pack(void* packed, const void* weight, const void* col_scale, int32_t rows,
                       int32_t cols, int32_t dtype, pa_stream_t stream);

/* The decode step's QKV projection with RoPE and the KV-cache write fused
 * into its epilogue: pa_linear (bf16, act none, optional PA_LINEAR_RMS_IN and
 * bias) over a weight packed by pa_linear_pack_qkv, followed in the same pass
 * by what pa_rope_reshape_and_cache does to its output
 * (crates/model/src/components/attention/rope_gqa.rs:280-302,
 * crates/model/src/components/positional/rope.rs:335-568):
 *   out [rows, (num_heads + 2 num_kv_heads) head_dim]: the projection, q and k
 *       columns rotated by position (inv_freq [head_dim / 2], positions [rows]),
 *       v columns as projected; identical to pa_linear followed by
 *       pa_rope_reshape_and_cache on the q / k / v views of its output;
 *   k_cache / v_cache: token r's rotated k and its v written to slot
 *       slot_mapping[r] (skipped when outside [0, num_blocks * 16)).
 * head_dim and in_features multiples of 32; flags 0 or PA_LINEAR_RMS_IN.
 * weight, bias: the fused QKV weight [(Hq + 2 Hkv) head_dim, in_features]
 * (bias in the original row order).  No reference counterpart as one call. */
int32_t pa_linear_rope_cache(void* out, const void* x, const void* weight, const void* bias,
                             int32_t rows, int32_t num_heads, int32_t num_kv_heads,
                             int32_t head_dim, int32_t in_features, int32_t flags, float eps,
                             const int64_t* positions, const int64_t* slot_mapping,
                             const float* inv_freq, void* k_cache, void* v_cache,
                             int32_t num_blocks, int32_t dtype, pa_stream_t stream);

/* pa_linear_pack for pa_linear_rope_cache's weight: the fused QKV weight
 * [(num_heads + 2 num_kv_heads) head_dim, cols], with the rows of each query
 * and key head reordered so that the two members (i, i + head_dim / 2) of
 * each rotation pair land in the same wavefront; col_scale as pa_linear_pack.
 * No reference counterpart: a load-time layout step. */
int32_t pa_linear_pack_qkv(void* packed, const void* weight, const void* col_scale,
                           int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                           int32_t cols, int32_t dtype, pa_stream_t stream);

/* ---------------------------------------------------------------------- */
/* The projections in MXFP8                                               */
/* ---------------------------------------------------------------------- */

/* MXFP8 (the OCP microscaling format with E4M3 elements): a row's columns go
 * in blocks of 32 with one power-of-two scale each, the format that the matrix
 * cores multiply directly.  No counterpart in the reference, whose FP8 is a KV
 * cache type with codes of its own (PA_DTYPE_FP8_E4M3); here the codes are OCP
 * E4M3 (bias 7, +-448 the largest, 0x7F / 0xFF NaN, no infinities).
 *   a = the largest |y| among the block's finite values
 *   e = the smallest integer >= -127 with a <= 448 * 2^e; scale byte e + 127
 *   code = y * 2^-e rounded to the nearest E4M3 value, ties to even; NaN and
 *          +-inf become NaN codes
 * so no finite value saturates, and a value is its code times 2^(byte - 127).
 * Columns are padded to Kp, the next multiple of 128, with zero codes.
 *   rows     codes [rows, Kp] uint8; scales [Kp / 128][R][4] uint8, R = rows
 *            rounded up to 16: byte b of (s, r) scales columns 128 s + 32 b ..
 *            + 31 of row r.  The scales of rows behind `rows` are neither
 *            written nor used.
 *   weights  [N, K], N padded to Np, the next multiple of 16, with zero rows:
 *            codes [Np / 16][Kp / 128][8][16][16], 16-row x 128-column
 *            fragments of 2 KB in the order of the matrix instructions'
 *            operands: chunk c of row r holds columns 16 c .. 16 c + 15;
 *            scales [Np / 16][Kp / 128][16][4].
 * Code arrays are 16-byte aligned, scale arrays 4-byte. */

/* Kp: the bytes of one row of codes. */
size_t pa_mx_row_bytes(int32_t cols);
/* Bytes of the scales of `rows` MXFP8 rows, and of a weight of `rows` rows. */
size_t pa_mx_scale_bytes(int32_t rows, int32_t cols);
/* Bytes of the codes of a weight of `rows` rows. */
size_t pa_mx_weight_bytes(int32_t rows, int32_t cols);

/* Quantises rows to MXFP8 (the attention's output in front of an MXFP8 O
 * projection): x [rows, cols] of dtype with x_stride elements between rows
 * (0 = cols, else at least cols), any alignment; codes and scales as above.
 * x does not overlap them. */
int32_t pa_quantize_mx(uint8_t* codes, uint8_t* scales, const void* x, int32_t rows,
                       int32_t cols, int64_t x_stride, int32_t dtype, pa_stream_t stream);

/* pa_rms_norm with an MXFP8 output:
 *   if add != NULL:  sum[r] = residual[r] + add[r]  (rounded to dtype)
 *   y[r] = s / sqrt(mean(s^2) + eps) * weight,  s = sum[r], or residual[r]
 *   codes, scales = MXFP8 of y (f32, not rounded in between)
 * residual / add / sum [rows, hidden] and weight [hidden] contiguous, of dtype;
 * sum is needed with add only and may be residual itself (in place), but
 * overlaps nothing otherwise. */
int32_t pa_rms_norm_mx(uint8_t* codes, uint8_t* scales, void* sum, const void* residual,
                       const void* add, const void* weight, int32_t rows, int32_t hidden,
                       float eps, int32_t dtype, pa_stream_t stream);

/* Quantises a weight [rows, cols] of dtype (contiguous) into the weight layout
 * above: a load-time step. */
int32_t pa_linear_mx_pack(uint8_t* codes, uint8_t* scales, const void* weight, int32_t rows,
                          int32_t cols, int32_t dtype, pa_stream_t stream);

/* pa_linear on MXFP8 rows and weights:
 *   act PA_ACT_NONE:      out[r][n] = sum_k x[r][k] * weight[n][k]
 *                                     (+ bias[n]) (+ residual[r][n])
 *   act PA_ACT_SILU_MUL:  weight is the gate|up matrix [2 N, K], N a multiple
 *                         of 32, out[r][n] = silu(g) * u of the two products of
 *                         column n; bias and residual must be NULL.
 * out_scales NULL: out [rows, N] bf16, contiguous, 16-byte aligned, rounded
 * once, from the f32 result.  out_scales given (PA_ACT_SILU_MUL only): the
 * result goes out as MXFP8 rows, codes to out, for the projection after it.
 *   bias [N] or NULL, residual [rows, N] (16-byte aligned) or NULL, bf16,
 *   contiguous; residual may be out itself (the residual stream updated in
 *   place), but out overlaps no other argument.
 * The sums are f32, over groups of 16 columns whose exact products the matrix
 * instructions align to the group's largest, cutting them off (towards zero) 13
 * binary places below its leading one.  A product loses less than 2^-13 of the
 * group's largest, so a group is off by less than 2^-9 of it and a result by
 * less than the sum of that over the K / 16 groups.  The losses have the signs of
 * the products: where these are mixed they add up as the root of their squares
 * (normal values, K 896 to 16384: 2^-16 of the result's root mean square, well
 * below the bf16 rounding unless terms cancel).  silu is off by up to (1.5 |g| +
 * 8) 2^-24 of it and 0 below -87.3, where it is less than 2^-119.  The scales of
 * an MXFP8 output are those of these results: where a block's largest value lies
 * that near to a border it may take the neighbouring scale.
 * Any rows, N (with PA_ACT_NONE) and K up to 2^22; PA_ERR_UNSUPPORTED where
 * the outputs' tiles would need 2^32 threads (no such arrays fit a GPU, but for
 * the last few of 2^31 rows).  The order of a row's f32
 * sums, and with it the last bit of an output, may depend on rows, N and K
 * (equal calls give equal bits). */
int32_t pa_linear_mx(void* out, uint8_t* out_scales, const uint8_t* x, const uint8_t* x_scales,
                     const uint8_t* weight, const uint8_t* weight_scales, const void* bias,
                     const void* residual, int32_t rows, int32_t out_features,
                     int32_t in_features, int32_t act, pa_stream_t stream);

/* Greedy sampling's argmax_logits (crates/traits/src/sampling.rs:439-453) on
 * every row of a logit matrix: out[r] = the first column holding the row's
 * largest value, comparing with `>` from -inf, so NaN never wins and a row
 * with no value above -inf (or cols == 0) gives 0.  logits [rows, cols] with
 * row_stride elements between rows (0 = cols); out [rows] int64 (device). */
int32_t pa_argmax(int64_t* out, const void* logits, int32_t rows, int32_t cols,
                  int64_t row_stride, int32_t dtype, pa_stream_t stream);

/* Draws a token from each row of a logit matrix.  With the row's settings T =
 * temperature, k = top_k, p = top_p, m = min_p and u = uniform, x its logits and
 * M the largest:
 *   w_i = exp((x_i - M) / T): 1 where x_i = M (also +inf), 0 for -inf; NaN is no
 *         value and never drawn
 *   top-k (0 < k < cols): the k largest are kept, of equal ones the first
 *   top-p (p < 1): of those, in descending order (equal ones by index), the
 *         shortest run whose weights sum to p times the sum of all of them or
 *         more; one at least
 *   min-p (m > 0): of those the ones with w_i >= m, and the largest
 *   out[r] = the first kept i, in the order of the columns, whose weights up to
 *         and with it sum to more than u times the sum of all kept
 * T not above 0: the argmax of pa_argmax.  A row without a value above -inf gives
 * 0.  u is in [0, 1): below 0 and NaN count as 0, 1 and more draw the last.
 *   uniform [rows] f32; temperature, top_p, min_p [rows] f32 and top_k [rows]
 *   int32, each may be NULL (1, off, off, off); all device
 *   logits  [rows, cols] of dtype with row_stride elements between rows (0 =
 *           cols), rows at any element; cols up to 2^22, rows up to 65535
 *   out     [rows] int64 (device)
 * Weights are formed in f64 and summed exactly in units of 2^-min(51, 62 - b), b =
 * max(1, ceil(log2 cols)), of the largest: the draw is that of the formula but for
 * borders closer than a few of those times cols, and does not depend on the order
 * of anything.
 * workspace: pa_sample_workspace_size() bytes, 16-byte aligned, with any contents;
 * calls that may overlap need workspaces of their own.
 * The reference samples on the host (crates/core/src/sampling.rs). */
int32_t pa_sample(int64_t* out, const void* logits, const float* uniform,
                  const float* temperature, const int32_t* top_k, const float* top_p,
                  const float* min_p, int32_t rows, int32_t cols, int64_t row_stride,
                  void* workspace, size_t workspace_bytes, int32_t dtype, pa_stream_t stream);

/* Workspace bytes of pa_sample (0, and workspace may be NULL, from 512 rows on). */
size_t pa_sample_workspace_size(int32_t rows);

#ifdef __cplusplus
}
#endif

#endif /* VLLM_LITE_AMD_PA_DENSE_H */
