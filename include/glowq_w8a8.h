/*
 * glowq_w8a8.h - C ABI of the B200 (sm_100a) 8-bit linear and of the norms in front of it
 *
 *     y[t, o] = s_t * w_o * sum_k c[t, k] q[o, k]  +  alpha * sum_j r[t, j] L[o, j]  (+ bias_o),    r = x . R^T
 *
 * c: int8 codes of a token's activations with one fp32 scale s_t per token; q: int8 codes of the weights with one fp32 scale w_o per
 * output channel.  The sums of products are exact (32-bit integers); scales, correction and bias are applied in fp32 and the result is
 * rounded once.  The reference project has no 8-bit path; these entry points stand beside those of glowq_w4a16.h, live in the same
 * library and follow its conventions: device pointers, memory owned by the caller, no allocation, no synchronisation, GLOWQ_* status
 * codes, no exceptions, no CPU fallback.  Nothing here needs a workspace except the gradients of the layer norm.
 */
#ifndef GLOWQ_W8A8_H_
#define GLOWQ_W8A8_H_

#include "glowq_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types.  (The first two have the values of GLOWQ_OUT_F16 and GLOWQ_OUT_F32.) */
enum { GLOWQ_F16 = 0, GLOWQ_F32 = 1, GLOWQ_BF16 = 2 };

/* Norms of glowq_w8a8_rows_t. */
enum { GLOWQ_NORM_NONE = 0, GLOWQ_NORM_LAYER = 1, GLOWQ_NORM_RMS = 2 };

/* Rows of an [M, K] matrix in front of a linear: an optional residual add and norm, and codes or the normalised rows.
 *     h = round(x + residual)                                            (residual NULL: h = x)
 *     LAYER  v = round(fma((h - mean) * rstd, weight, bias))             mean, rstd of h: taken in 64 bits, rounded to fp32 once
 *     RMS    v = round(weight * round(h * rstd))                         (the arithmetic of the models' RMSNorm modules)
 *     NONE   v = h
 *     scale = fp32(max |v| / 127),  code = the integer nearest to v / scale, ties to even, exactly, within [-127, 127]
 * "round" is to the matrix's own type.  A row of zeros has scale 0 and codes 0.  A row with a NaN or an infinity has scale NaN and
 * codes 0, so that every output of that token is NaN.  Strides are in elements; rows have unit column stride; no output overlaps an
 * input or another output.  At most 2^30 rows and 2^29 columns, here and in the layer norm's gradients. */
typedef struct glowq_w8a8_rows {
  const void* x;          /* [M, x_stride]                                                       */
  const void* residual;   /* [M, residual_stride] or NULL                                        */
  const void* weight;     /* [K] of the norm; NULL with GLOWQ_NORM_NONE                          */
  const void* bias;       /* [K] of the layer norm; NULL otherwise                               */
  void* hidden;           /* [M, hidden_stride] receives h, or NULL; only with a residual        */
  void* y;                /* [M, y_stride] receives v (glowq_layer_norm_forward), else NULL      */
  int8_t* codes;          /* [M, code_stride] (glowq_w8a8_quantize), else NULL                   */
  float* scales;          /* [M] with codes                                                      */
  float* mean;            /* [M] or NULL (layer norm's statistics for its gradients)             */
  float* rstd;            /* [M] or NULL                                                         */
  void* stream;
  double eps;
  int64_t x_stride, residual_stride, hidden_stride, y_stride, code_stride;
  int32_t M, K;
  int32_t dtype;          /* GLOWQ_F16 / GLOWQ_F32 / GLOWQ_BF16: x, residual, weight, bias, hidden, y */
  int32_t norm;           /* GLOWQ_NORM_*                                                        */
  int32_t constant;       /* nonzero: the codes are weights, which a product launched behind this call may read early */
  int32_t reserved;       /* must be 0                                                           */
} glowq_w8a8_rows_t;

int glowq_w8a8_quantize(const glowq_w8a8_rows_t* rows);
int glowq_layer_norm_forward(const glowq_w8a8_rows_t* rows);

/* Gradients of the layer norm y = LN(h) * weight + bias, where h may itself be an output (residual form):
 *     g = dy * weight,  xh = (h - mean) * rstd,  dx = rstd * (g - mean_k(g) - xh * mean_k(g xh)) + dh
 *     dweight = sum_t dy xh,  dbias = sum_t dy           (fp32 sums in an order that the sizes and the rows'
 *                                                           places within 16 bytes fix; rounded once)
 * dweight and dbias may be NULL together; dx may be NULL.  `workspace`: glowq_layer_norm_workspace_bytes(), any contents. */
typedef struct glowq_layer_norm_grad {
  const void* h;
  const void* dy;
  const void* dh;         /* gradient of h as an output, or NULL */
  const void* weight;
  const float* mean;
  const float* rstd;
  void* dx;
  void* dweight;
  void* dbias;
  void* workspace;
  size_t workspace_bytes;
  void* stream;
  int64_t h_stride, dy_stride, dh_stride, dx_stride;
  int32_t M, K, dtype;
  int32_t reserved;       /* must be 0 */
} glowq_layer_norm_grad_t;

size_t glowq_layer_norm_workspace_bytes(int M, int K);
int glowq_layer_norm_backward(const glowq_layer_norm_grad_t* grad);

/* Added to r_mode below. */
enum { GLOWQ_W8A8_FRESH = 16 };

/* One linear.  With `x` set the call first quantises x into `codes` and `scales` (which are then scratch of the caller's); with r_mode
 * GLOWQ_R_COMPUTE it computes r = r_x . R^T (rounded to fp16, as the W4A16 path holds it) into `r`; GLOWQ_R_LOAD takes r as it is.
 * Alignment: codes, weight, r_x, R, L and r begin on 16 bytes and their row strides are multiples of 16 bytes (what lies behind
 * column K is never used).  r and r_x are fp16: where a token's values or its r pass 65504 its corrected outputs are infinite or NaN,
 * whatever x_dtype.  out and bias need the alignment of their elements.  K <= 131071 (exact sums); rank <= 1024; at most 2^22
 * tokens and 2^29 channels.
 * `weight`, `weight_scales`, `bias`, L and R are constants: they may be read before what is in front of this call on the stream is complete
 * and visible, whoever launched it.  Where the kernel, copy or call right in front made one of them, add GLOWQ_W8A8_FRESH to r_mode
 * (glowq_w8a8_quantize with `constant` is complete for all that is launched behind it). */
typedef struct glowq_w8a8_linear {
  const void* x;                /* [M, x_stride] of x_dtype, or NULL: codes and scales are there already */
  int8_t* codes;                /* [M, code_stride]                                                      */
  float* scales;                /* [M]                                                                   */
  const int8_t* weight;         /* [OC, weight_stride]                                                   */
  const float* weight_scales;   /* [OC]                                                                  */
  const float* bias;            /* [OC] or NULL                                                          */
  const void* r_x;              /* fp16 [M, r_x_stride]; GLOWQ_R_COMPUTE                                 */
  const void* R;                /* fp16 [rank, R_stride]; GLOWQ_R_COMPUTE                                */
  void* r;                      /* fp16 [M, r_stride]                                                    */
  const void* L;                /* fp16 [OC, L_stride]                                                   */
  void* out;                    /* [M, out_stride] of out_dtype                                          */
  void* stream;
  int64_t x_stride, code_stride, weight_stride, r_x_stride, R_stride, r_stride, L_stride, out_stride;
  int32_t M, K, OC, rank;
  int32_t x_dtype, out_dtype, r_mode;
  float alpha;
  int64_t reserved;             /* must be 0 */
} glowq_w8a8_linear_t;

int glowq_w8a8_linear(const glowq_w8a8_linear_t* linear);

/* The right factor's product alone: r of the call above, for linears that share one. */
int glowq_w8a8_right_factor(const glowq_w8a8_linear_t* linear);

/* Whether a wait of the 8-bit kernels ran out on the current device since the last call (synchronises `stream`): GLOWQ_OK or
 * GLOWQ_ERR_DEVICE_TIMEOUT. */
int glowq_w8a8_read_status(void* stream);

#ifdef __cplusplus
}
#endif
#endif /* GLOWQ_W8A8_H_ */
