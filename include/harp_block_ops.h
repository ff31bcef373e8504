/*
 * harp_block_ops.h — C ABI of the MI355X (gfx950) kernels around the attention
 * block: the residual addition with its RMSNorm (forward and backward), 8-bit
 * rows (quantise, norm + quantise, dequantise), and products of 8-bit rows
 * (Linear layers, and the q/k/v producer with QK RMSNorm and RoPE).
 *
 * HARP's model normalises the hidden states with an RMSNorm in front of the
 * attention and the feed-forward of its blocks and adds their results to the
 * residual stream (src/models/z_image/module/block.py; factors per sample and
 * gates, where a block has them, are the caller's), and runs its Linear
 * layers through xhblas_gemm (gemm/bgemm/bgemm.h:20-26) in bf16; the 8-bit
 * forms have no reference counterpart.  libharp_ra.so exports the functions
 * declared here next to those of harp_ring_attn.h and harp_qk_norm_rope.h.
 *
 * Conventions (as there): plain device pointers of the current device, row
 * strides ("ld") in elements, unit stride along a row, asynchronous on the
 * given HIP stream (NULL = default stream), int status (HARP_BLK_OK = 0) and
 * harp_blk_last_error() for the message.  Nothing is allocated; arguments are
 * checked on the host before any device call.  Matrices need the alignment of
 * their elements only; input rows may repeat (ld 0), output rows may not
 * overlap (ld >= cols).  rows == 0 (or M == 0) does nothing.
 *
 * An 8-bit row is cols int8 values in -127 .. 127 with one fp32 scale: it
 * stands for value * scale.  Rows start 16-byte aligned (ld a multiple of 16
 * bytes).  scale = max|row| / 127, values to nearest, ties to even; a row of
 * zeros has scale 0; a row with an infinity or a NaN (of a norm: whose results
 * are not finite) has scale NaN and values 0, so that whatever reads it is NaN.
 */
#ifndef HARP_BLOCK_OPS_H
#define HARP_BLOCK_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifndef HARP_BLK_API
#define HARP_BLK_API __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

enum {
  HARP_BLK_OK = 0,
  HARP_BLK_EINVAL = 1,       /* bad pointer, size, stride, alignment or dtype */
  HARP_BLK_EUNSUPPORTED = 2, /* valid request that the library does not handle (e.g. cols > 32768) */
  HARP_BLK_ENOMEM = 3,       /* workspace too small */
  HARP_BLK_ELAUNCH = 4       /* HIP launch or runtime error */
};

enum { HARP_BLK_F32 = 0, HARP_BLK_BF16 = 1 };

/*
 * h = x + residual, rounded to the residual's type (x_dtype, r_dtype: F32 or
 * BF16), y = h / sqrt(mean(h^2) + eps) * weight in x's type.  residual NULL:
 * h is x, and is not written (h must be NULL).  weight: [cols] of w_dtype or
 * NULL for ones.  rstd ([rows] fp32, may be NULL): 1 / sqrt(mean(h^2) + eps).
 * 1 <= cols <= 32768.  y and h must not overlap the inputs.
 */
HARP_BLK_API int harp_blk_add_rms_norm_forward(const void* x, int64_t ld_x, int x_dtype, const void* residual,
                                               int64_t ld_residual, int r_dtype, const void* weight, int w_dtype,
                                               float eps, void* y, int64_t ld_y, void* h, int64_t ld_h, float* rstd,
                                               int rows, int cols, void* stream);

/*
 * Its backward.  dy: gradient of y (x_dtype); dh: gradient of h (h_dtype),
 * NULL for zeros; h: the normalised input that the forward wrote (or x);
 * dx in x_dtype; dresidual in h_dtype, or NULL (where the types agree it
 * equals dx); grad_weight [cols] of gw_dtype, or NULL.  workspace:
 * harp_blk_backward_workspace_bytes() bytes of device memory, 16-byte aligned,
 * needed (and written) only with grad_weight; its sums are taken in an order
 * that the sizes alone fix.  rows == 0 clears nothing: grad_weight is not
 * written.
 */
HARP_BLK_API int harp_blk_add_rms_norm_backward(const void* dy, int64_t ld_dy, int x_dtype, const void* dh,
                                                int64_t ld_dh, const void* h, int64_t ld_h, int h_dtype,
                                                const void* weight, int w_dtype, const float* rstd, void* dx,
                                                int64_t ld_dx, void* dresidual, int64_t ld_dresidual,
                                                void* grad_weight, int gw_dtype, int rows, int cols, void* workspace,
                                                size_t workspace_bytes, void* stream);

/* Device bytes the backward needs for its weight gradient; (size_t)-1 for sizes it does not take. */
HARP_BLK_API size_t harp_blk_backward_workspace_bytes(int rows, int cols);

/*
 * 8-bit rows of the norm's result: h as above, q [rows, cols] int8 (ld_q a
 * multiple of 16 and >= cols rounded up to 16; the bytes from cols up to that
 * are written as zeros), scales [rows] fp32.  The result is quantised from
 * fp32, without a rounding to 16 bits before.
 */
HARP_BLK_API int harp_blk_add_rms_norm_int8(const void* x, int64_t ld_x, int x_dtype, const void* residual,
                                            int64_t ld_residual, int r_dtype, const void* weight, int w_dtype,
                                            float eps, void* h, int64_t ld_h, int8_t* q, int64_t ld_q, float* scales,
                                            int rows, int cols, void* stream);

/* 8-bit rows of x (q and scales as above). */
HARP_BLK_API int harp_blk_quantize_int8(const void* x, int64_t ld_x, int x_dtype, int8_t* q, int64_t ld_q,
                                        float* scales, int rows, int cols, void* stream);

/* out = values * scales, in out_dtype.  1 <= cols <= 2^30. */
HARP_BLK_API int harp_blk_dequantize_int8(const int8_t* q, int64_t ld_q, const float* scales, void* out,
                                          int64_t ld_out, int out_dtype, int rows, int cols, void* stream);

/*
 * A Linear layer on 8-bit rows:
 *   y[m][n] = (sum_k x[m][k] * w[n][k]) * x_scales[m] * w_scales[n] + bias[n]
 * x [M, K] and w [N, K] int8, rows 16-byte aligned (ld_x, ld_w multiples of
 * 16, >= K rounded up to 16, <= 2^22; the bytes from K up to there may be read
 * but count for nothing); bias [N] of bias_dtype or NULL; y of y_dtype.  The
 * sums are exact 32-bit integers: 1 <= K <= 65536; M, N <= 2^30.
 */
HARP_BLK_API int harp_blk_linear_int8(const int8_t* x, int64_t ld_x, const float* x_scales, const int8_t* w,
                                      int64_t ld_w, const float* w_scales, const void* bias, int bias_dtype, void* y,
                                      int64_t ld_y, int y_dtype, int M, int N, int K, void* stream);

/* One projection of harp_blk_qkv_int8. */
typedef struct {
  const int8_t* weight; /* [n_out, k_dim] 8-bit rows */
  int64_t ld_weight;    /* bytes, a multiple of 16, >= k_dim rounded up to 16 */
  const float* weight_scales;
  void* y;              /* [batch * seq, n_out] bf16 */
  int64_t ld_y;
  const void* norm_weight; /* [128] QK RMSNorm weight over each head's 128 features, or NULL: plain projection */
  int norm_weight_dtype;
  float eps;
} harp_blk_qkv_out_t;

/*
 * Up to three projections of the same 8-bit rows x [batch * seq, k_dim], heads
 * of 128 features (n_out a multiple of 128); the outputs with a norm weight
 * are normalised per head and, with freqs (the RoPE table of
 * harp_qk_norm_rope.h: rows of 128 floats, strides multiples of 4, 16-byte
 * aligned), rotated.  fp32 throughout, one rounding to bf16 at the end.
 */
HARP_BLK_API int harp_blk_qkv_int8(const int8_t* x, int64_t ld_x, const float* x_scales, int batch, int seq, int k_dim,
                                   int n_out, const float* freqs, int64_t f_stride_b, int64_t f_stride_s,
                                   const harp_blk_qkv_out_t* outs, int n_outs, void* stream);

HARP_BLK_API const char* harp_blk_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* HARP_BLOCK_OPS_H */
