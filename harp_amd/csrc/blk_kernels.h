// Parameter blocks and launchers of the kernels around the attention block:
// the residual addition with its RMSNorm, 8-bit rows, and the products of
// 8-bit rows (internal to libharp_ra.so; the C ABI is in
// include/harp_block_ops.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace harp_blk {

constexpr int kF32 = 0, kBf16 = 1, kNone = 2;  // element types (kNone: no such tensor)

constexpr int kMaxCols = 1 << 15;  // a row of the norm fits the registers of one block

// h = x + residual (rounded to the residual's type), y = h / rms(h) * weight.
struct NormParams {
  int rows, cols;
  const void* x;  // [rows, cols], row stride ldx
  int64_t ldx;
  int x_dtype;
  const void* res;  // residual, or NULL: h is x and is not written
  int64_t ldr;
  int r_dtype;  // of the residual and of h
  void* h;      // [rows, cols] x + residual (NULL = not written)
  int64_t ldh;
  const void* w;  // [cols], NULL = ones
  int w_dtype;
  float eps;
  void* y;  // [rows, cols] in x's type; the forward only
  int64_t ldy;
  float* rstd;  // [rows] 1 / rms, NULL = not written
  // 8-bit rows instead of y: q[r][c] * scale[r] is about y
  int8_t* q;
  int64_t ldq;  // bytes, a multiple of 16: rows are written up to the next multiple of 16 (zeros behind cols)
  float* scale;
};

// dx = d(loss)/d(x) for dy = d(loss)/d(y) and dh = d(loss)/d(h).
struct NormBwdParams {
  int rows, cols;
  const void* dy;  // in x's type
  int64_t ldy;
  int x_dtype;
  const void* dh;  // in h's type, NULL = zeros
  int64_t lddh;
  const void* h;  // the normalised input
  int64_t ldh;
  int h_dtype;
  const void* w;
  int w_dtype;
  const float* rstd;
  void* dx;  // in x's type
  int64_t lddx;
  void* dres;  // in h's type; NULL = not written (it equals dx where the types do)
  int64_t lddr;
  float* wpart;  // [bwd_blocks(rows, cols)][cols] sums of dy * h * rstd over a block's rows, NULL = not needed
};

int bwd_blocks(int rows, int cols);

hipError_t launch_norm(const NormParams& p, hipStream_t stream);       // y
hipError_t launch_norm_rows8(const NormParams& p, hipStream_t stream);  // q, scale of y
hipError_t launch_quantize(const NormParams& p, hipStream_t stream);    // q, scale of x
hipError_t launch_norm_backward(const NormBwdParams& p, hipStream_t stream);
hipError_t launch_wgrad(const float* wpart, int blocks, int cols, void* gw, int gw_f32, hipStream_t stream);
// out[r][c] = q[r][c] * scale[r]
hipError_t launch_dequantize(const int8_t* q, int64_t ldq, const float* scale, void* out, int64_t ldo, int o_dtype,
                             int rows, int cols, hipStream_t stream);

// ---------------------------------------------------------------------------
constexpr int kMaxOuts8 = 3;
constexpr int kKTile8 = 128;  // bytes of K per unit of the kinds' measured times

// One product y = (x w^T) * x_scale * w_scale + bias of 8-bit rows.
struct Prod8Out {
  const int8_t* w;  // [N, K], row stride ldw bytes
  int64_t ldw;
  const float* w_scale;  // [N]
  const void* bias;      // [N] or NULL
  int bias_f32;
  void* y;  // [M, N] bf16 or fp32, row stride ldy elements
  int64_t ldy;
  int y_f32;
  const void* norm_w;  // QK RMSNorm weight [128] over each 128 features, NULL = no norm
  int norm_w_f32;
  float eps;
};

struct Prod8Params {
  const int8_t* x;  // [M, K], row stride ldx bytes
  int64_t ldx;
  const float* x_scale;  // [M]
  int M, N, K;
  int S;               // tokens of one batch entry (rows of the RoPE table)
  int m_base;          // x's first row among the call's tokens (0, or set by launch_prod8)
  const float* freqs;  // RoPE table of the normed outputs, fp32 (cos, sin) pairs; NULL = none
  int64_t f_stride_b, f_stride_s;
  int n_outs;
  Prod8Out out[kMaxOuts8];
};

hipError_t launch_prod8(const Prod8Params& p, hipStream_t stream);

}  // namespace harp_blk
