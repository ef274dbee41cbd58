/*
 * pixelsplat_ops.h -- C ABI of libpixelsplat_ops.so (MI355X / gfx950): the operators of image-transformer blocks.
 *
 * The conventions are those of pixelsplat_hip.h: plain pointers and sizes, every buffer is DEVICE memory owned by the
 * caller, `stream` is a hipStream_t passed as void*, the library keeps no state between calls, never throws, aborts or
 * synchronises, and returns 0 or a negative PsStatus.  Launches go to the calling thread's current device, which has to
 * be the tensors' own.
 *
 * Tensors have one of three element types; arithmetic is fp32 (sums over many elements fp32 or fp64), results are
 * rounded to nearest even.  All of it is deterministic: the same inputs give the same bits.
 */
#ifndef PIXELSPLAT_OPS_H
#define PIXELSPLAT_OPS_H

#include "pixelsplat_hip.h" /* PsStatus */

#ifdef __cplusplus
extern "C" {
#endif

#define PS_DTYPE_F32 0
#define PS_DTYPE_BF16 1
#define PS_DTYPE_F16 2

#define PS_ACT_NONE 0
#define PS_ACT_RELU 1
#define PS_ACT_SILU 2 /* z sigmoid(z)                 */
#define PS_ACT_GELU 3 /* z (1 + erf(z / sqrt 2)) / 2  */
#define PS_ACT_SIGMOID 4

/* Group norm with an activation, channels last: x [samples][rows][channels] (unit channel stride, strides of samples
 * and rows in elements), y = act((x - mean) rstd gamma + beta) with mean and variance over the rows and the
 * channels / groups channels of a (sample, group); y and dx are contiguous and 16-byte aligned.  gamma, beta
 * [channels] in the tensors' type, or fp32 when param_f32; either may be NULL (1 and 0).  mean, rstd [samples][groups]
 * fp32 are what the backward needs of the forward.  d_gamma / d_beta are in the parameters' type, NULL when not
 * wanted.  channels <= 8192, samples <= 65535, rows * channels < 2^31 (else PS_ERR_UNSUPPORTED).
 * workspace: ps_group_norm_workspace_bytes(desc, backward) bytes, 16-byte aligned, its contents are not kept. */
typedef struct PsGroupNormDesc {
  int32_t samples, rows, channels, groups;
  int32_t dtype, activation, param_f32;
  float eps;
  int64_t x_sample_stride, x_row_stride;
  int64_t dy_sample_stride, dy_row_stride; /* backward only */
} PsGroupNormDesc;
size_t ps_group_norm_workspace_bytes(const PsGroupNormDesc* desc, int32_t backward);
int ps_group_norm_forward(const PsGroupNormDesc* desc, const void* x, const void* gamma, const void* beta, void* y,
                          float* mean, float* rstd, void* workspace, size_t workspace_bytes, void* stream);
int ps_group_norm_backward(const PsGroupNormDesc* desc, const void* x, const void* dy, const void* gamma,
                           const void* beta, const float* mean, const float* rstd, void* dx, void* d_gamma,
                           void* d_beta, void* workspace, size_t workspace_bytes, void* stream);

/* Gated projection of a feed-forward block, h = act(x w_gate^T + b_gate) * (x w_up^T + b_up): x [rows][dim], weights
 * [hidden][dim] (one row stride for both), biases [hidden] in the tensors' type, each may be NULL; h [rows][hidden]
 * contiguous.  dim and the strides of x and of the weights are whole numbers of 16-byte chunks and the three
 * matrices are 16-byte aligned (else PS_ERR_BAD_ARG); hidden is any number.  No projection is written to memory,
 * except gate, up [rows][hidden] fp32 (the projections with their biases) where they are not NULL: fp32 training
 * hands them to the backward, 16-bit types compute them again and take NULL there.
 * Backward: every output may be NULL.  dx [rows][dim], dw [hidden][dim], db [hidden], contiguous.  h, dx and dw are
 * 16-byte aligned. */
typedef struct PsGatedLinearDesc {
  int32_t rows, dim, hidden;
  int32_t dtype, activation;
  int32_t reserved; /* 0 */
  int64_t x_row_stride, w_row_stride, dh_row_stride;
} PsGatedLinearDesc;
int ps_gated_linear_forward(const PsGatedLinearDesc* desc, const void* x, const void* w_gate, const void* w_up,
                            const void* b_gate, const void* b_up, void* h, float* gate, float* up, void* stream);
size_t ps_gated_linear_backward_workspace_bytes(const PsGatedLinearDesc* desc);
int ps_gated_linear_backward(const PsGatedLinearDesc* desc, const void* x, const void* w_gate, const void* w_up,
                             const void* b_gate, const void* b_up, const float* gate, const float* up, const void* dh,
                             void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, void* workspace,
                             size_t workspace_bytes, void* stream);

/* Attention over a grid of grid_h x grid_w tokens (numbered by rows) with a learned relative position bias:
 *   s = scale q.k + table[bucket_map[key row - query row + grid_h - 1][key column - query column + grid_w - 1]][head]
 *   out = softmax(s over the keys whose key_mask is not 0) v; a row without keys is zero.
 * The queries are the tokens query_start .. query_start + queries - 1, the keys and values all tokens.  q, k, v, d_out
 * are read at strides (batch, head, token; elements, unit stride within a row of dim); their rows start on 16 bytes
 * and hold whole 16-byte chunks.  out, dq [batch][queries][heads][dim] and dk, dv [batch][keys][heads][dim] are
 * contiguous.  key_mask [batch][keys] bytes or NULL: the rows of k and v of masked keys are not read.  bucket_map
 * [2 grid_h - 1][2 grid_w - 1]; an entry outside 0 .. buckets - 1 is an offset without bias.  table [buckets][heads] in
 * the tensors' type, or fp32 when table_f32.
 * For the backward the forward leaves bias [heads][offsets] fp32 (always written), stats [2][batch][heads][queries
 * rounded up to 64] fp32 and out_f32 (the unrounded out; fp32 tensors hand `out` itself to the backward and NULL to the
 * forward); stats and out_f32 are NULL where no backward follows.  Backward: each output may be NULL.
 * dim <= 128, keys <= 2^20, grid_w <= 512 unless grid_h is 1, token strides < 2^24, batch * heads < 2^24 and
 * batch * heads * tokens / 32 < 2^26, tokens rounded up to whole tiles (else PS_ERR_UNSUPPORTED). */
typedef struct PsRelativeAttentionDesc {
  int32_t batch, heads, queries, query_start, grid_h, grid_w, dim;
  int32_t dtype, buckets, table_f32;
  float scale;
  int32_t reserved; /* 0 */
  int64_t q_strides[3], k_strides[3], v_strides[3], do_strides[3];
  int64_t mask_stride; /* of a batch element */
} PsRelativeAttentionDesc;
#define PS_FORWARD 0
#define PS_BACKWARD 1          /* with d_table: grows with queries x keys */
#define PS_BACKWARD_NO_TABLE 2 /* d_table is NULL */
size_t ps_relative_attention_workspace_bytes(const PsRelativeAttentionDesc* desc, int32_t pass);
int ps_relative_attention_forward(const PsRelativeAttentionDesc* desc, const void* q, const void* k, const void* v,
                                  const uint8_t* key_mask, const int32_t* bucket_map, const void* table, void* out,
                                  float* out_f32, float* stats, float* bias, void* workspace, size_t workspace_bytes,
                                  void* stream);
int ps_relative_attention_backward(const PsRelativeAttentionDesc* desc, const void* q, const void* k, const void* v,
                                   const uint8_t* key_mask, const int32_t* bucket_map, const float* bias,
                                   const float* out_f32, const float* stats, const void* d_out, void* dq, void* dk, void* dv,
                                   void* d_table, void* workspace, size_t workspace_bytes, void* stream);

/* "pixelsplat_ops gfx950 | <file>:<hash> ...", as ps_build_info of pixelsplat_hip.h. */
const char* ps_ops_build_info(void);

#ifdef __cplusplus
}
#endif
#endif
