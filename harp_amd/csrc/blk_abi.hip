// C ABI of the kernels around the attention block: argument validation and
// kernel sequencing.  See include/harp_block_ops.h.
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <string>

#include "../../include/harp_block_ops.h"
#include "blk_kernels.h"

using namespace harp_blk;

static_assert(HARP_BLK_F32 == kF32 && HARP_BLK_BF16 == kBf16, "the kernels' element types");

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}
int ok() {
  g_last_error.clear();
  return HARP_BLK_OK;
}

constexpr int64_t kMaxLd8 = (int64_t)1 << 22;  // a 256-row tile of 8-bit rows spans < 2^32 bytes
constexpr int kMaxK = 1 << 16;                 // 2^16 products of at most 2^14: below 2^31
constexpr int kMaxTokens = 1 << 30;            // of a product: token indexes stay in 32 bits past the last tile

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int elem_size(int dt) { return dt == HARP_BLK_F32 ? 4 : 2; }

int check_dtype(int dt, const char* name) {
  if (dt != HARP_BLK_F32 && dt != HARP_BLK_BF16) return fail(HARP_BLK_EINVAL, "%s dtype must be F32 or BF16", name);
  return HARP_BLK_OK;
}

int check_rows_cols(int rows, int cols) {
  if (rows < 0) return fail(HARP_BLK_EINVAL, "rows=%d must not be negative", rows);
  if (cols < 1) return fail(HARP_BLK_EINVAL, "cols=%d must be positive", cols);
  if (cols > kMaxCols) return fail(HARP_BLK_EUNSUPPORTED, "cols=%d > %d is not supported", cols, kMaxCols);
  return HARP_BLK_OK;
}

int check_matrix(const void* p, int64_t ld, int dt, int cols, bool output, const char* name) {
  int rc;
  if (!p) return fail(HARP_BLK_EINVAL, "%s is NULL", name);
  if ((rc = check_dtype(dt, name))) return rc;
  if (!aligned(p, (uintptr_t)elem_size(dt)))
    return fail(HARP_BLK_EINVAL, "%s must be aligned to its elements", name);
  if (output ? ld < cols : ld < 0)
    return fail(HARP_BLK_EINVAL, "%s row stride %lld must be %s", name, (long long)ld,
                output ? "at least cols (rows may not overlap)" : "non-negative");
  return HARP_BLK_OK;
}

int check_vector(const void* p, int dt, const char* name) {  // optional
  int rc;
  if (!p) return HARP_BLK_OK;
  if ((rc = check_dtype(dt, name))) return rc;
  if (!aligned(p, (uintptr_t)elem_size(dt)))
    return fail(HARP_BLK_EINVAL, "%s must be aligned to its elements", name);
  return HARP_BLK_OK;
}

int check_floats(const float* p, const char* name) {
  if (!p) return fail(HARP_BLK_EINVAL, "%s is NULL", name);
  if (!aligned(p, 4)) return fail(HARP_BLK_EINVAL, "%s must be 4-byte aligned", name);
  return HARP_BLK_OK;
}

int check_rows8(const int8_t* p, int64_t ld, int cols, int64_t max_ld, bool output, const char* name) {
  if (!p || !aligned(p, 16)) return fail(HARP_BLK_EINVAL, "%s must be a 16-byte aligned device pointer", name);
  const int64_t need = ((int64_t)cols + 15) / 16 * 16;
  if (ld % 16 || (output || ld != 0 ? ld < need : false) || ld > max_ld || ld < 0)
    return fail(HARP_BLK_EINVAL, "%s row stride %lld must be a multiple of 16 in [%lld, %lld]", name, (long long)ld,
                (long long)need, (long long)max_ld);
  return HARP_BLK_OK;
}

int check_eps(float eps) {
  if (!(eps >= 0.f)) return fail(HARP_BLK_EINVAL, "eps must be a non-negative number");
  return HARP_BLK_OK;
}

int launched(hipError_t e, const char* what) {
  if (e != hipSuccess) return fail(HARP_BLK_ELAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
  return ok();
}

// x, residual, weight, eps and h, as both forms of the norm take them
int norm_inputs(NormParams& p, const void* x, int64_t ld_x, int x_dtype, const void* residual, int64_t ld_r,
                int r_dtype, const void* weight, int w_dtype, float eps, void* h, int64_t ld_h, int rows, int cols) {
  int rc;
  if ((rc = check_rows_cols(rows, cols))) return rc;
  if (rows == 0) return HARP_BLK_OK;
  if ((rc = check_matrix(x, ld_x, x_dtype, cols, false, "x"))) return rc;
  if (residual) {
    if ((rc = check_matrix(residual, ld_r, r_dtype, cols, false, "residual"))) return rc;
    if (h && (rc = check_matrix(h, ld_h, r_dtype, cols, true, "h"))) return rc;
  } else if (h) {
    return fail(HARP_BLK_EINVAL, "h without a residual is x: pass NULL");
  }
  if ((rc = check_vector(weight, w_dtype, "weight"))) return rc;
  if ((rc = check_eps(eps))) return rc;
  p.rows = rows;
  p.cols = cols;
  p.x = x;
  p.ldx = ld_x;
  p.x_dtype = x_dtype;
  p.res = residual;
  p.ldr = ld_r;
  p.r_dtype = r_dtype;
  p.h = h;
  p.ldh = ld_h;
  p.w = weight;
  p.w_dtype = w_dtype;
  p.eps = eps;
  return HARP_BLK_OK;
}

}  // namespace

extern "C" {

const char* harp_blk_last_error(void) { return g_last_error.c_str(); }

int harp_blk_add_rms_norm_forward(const void* x, int64_t ld_x, int x_dtype, const void* residual, int64_t ld_residual,
                                  int r_dtype, const void* weight, int w_dtype, float eps, void* y, int64_t ld_y,
                                  void* h, int64_t ld_h, float* rstd, int rows, int cols, void* stream) {
  int rc;
  NormParams p{};
  if ((rc = norm_inputs(p, x, ld_x, x_dtype, residual, ld_residual, r_dtype, weight, w_dtype, eps, h, ld_h, rows,
                        cols)))
    return rc;
  if (rows == 0) return ok();
  if ((rc = check_matrix(y, ld_y, x_dtype, cols, true, "y"))) return rc;
  if (rstd && (rc = check_floats(rstd, "rstd"))) return rc;
  p.y = y;
  p.ldy = ld_y;
  p.rstd = rstd;
  return launched(launch_norm(p, (hipStream_t)stream), "RMSNorm");
}

size_t harp_blk_backward_workspace_bytes(int rows, int cols) {
  if (check_rows_cols(rows, cols)) return (size_t)-1;
  return (size_t)bwd_blocks(rows, cols) * cols * sizeof(float);
}

int harp_blk_add_rms_norm_backward(const void* dy, int64_t ld_dy, int x_dtype, const void* dh, int64_t ld_dh,
                                   const void* h, int64_t ld_h, int h_dtype, const void* weight, int w_dtype,
                                   const float* rstd, void* dx, int64_t ld_dx, void* dresidual, int64_t ld_dresidual,
                                   void* grad_weight, int gw_dtype, int rows, int cols, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_rows_cols(rows, cols))) return rc;
  if (rows == 0) return ok();
  if ((rc = check_matrix(dy, ld_dy, x_dtype, cols, false, "dy"))) return rc;
  if (dh && (rc = check_matrix(dh, ld_dh, h_dtype, cols, false, "dh"))) return rc;
  if ((rc = check_matrix(h, ld_h, h_dtype, cols, false, "h"))) return rc;
  if ((rc = check_vector(weight, w_dtype, "weight"))) return rc;
  if ((rc = check_floats(rstd, "rstd"))) return rc;
  if ((rc = check_matrix(dx, ld_dx, x_dtype, cols, true, "dx"))) return rc;
  if (dresidual && (rc = check_matrix(dresidual, ld_dresidual, h_dtype, cols, true, "dresidual"))) return rc;
  if ((rc = check_vector(grad_weight, gw_dtype, "grad_weight"))) return rc;
  const int blocks = bwd_blocks(rows, cols);
  if (grad_weight) {
    const size_t need = (size_t)blocks * cols * sizeof(float);
    if (!workspace || workspace_bytes < need)
      return fail(HARP_BLK_ENOMEM, "workspace of %zu bytes is smaller than the %zu bytes needed",
                  workspace ? workspace_bytes : (size_t)0, need);
    if (!aligned(workspace, 16)) return fail(HARP_BLK_EINVAL, "workspace must be 16-byte aligned");
  }
  NormBwdParams p{};
  p.rows = rows;
  p.cols = cols;
  p.dy = dy;
  p.ldy = ld_dy;
  p.x_dtype = x_dtype;
  p.dh = dh;
  p.lddh = ld_dh;
  p.h = h;
  p.ldh = ld_h;
  p.h_dtype = h_dtype;
  p.w = weight;
  p.w_dtype = w_dtype;
  p.rstd = rstd;
  p.dx = dx;
  p.lddx = ld_dx;
  p.dres = dresidual;
  p.lddr = ld_dresidual;
  p.wpart = grad_weight ? (float*)workspace : nullptr;
  if ((rc = launched(launch_norm_backward(p, (hipStream_t)stream), "RMSNorm backward"))) return rc;
  if (!grad_weight) return ok();
  return launched(launch_wgrad(p.wpart, blocks, cols, grad_weight, gw_dtype == HARP_BLK_F32, (hipStream_t)stream),
                  "weight-gradient reduction");
}

int harp_blk_add_rms_norm_int8(const void* x, int64_t ld_x, int x_dtype, const void* residual, int64_t ld_residual,
                               int r_dtype, const void* weight, int w_dtype, float eps, void* h, int64_t ld_h,
                               int8_t* q, int64_t ld_q, float* scales, int rows, int cols, void* stream) {
  int rc;
  NormParams p{};
  if ((rc = norm_inputs(p, x, ld_x, x_dtype, residual, ld_residual, r_dtype, weight, w_dtype, eps, h, ld_h, rows,
                        cols)))
    return rc;
  if (rows == 0) return ok();
  if ((rc = check_rows8(q, ld_q, cols, INT64_MAX, true, "q"))) return rc;
  if ((rc = check_floats(scales, "scales"))) return rc;
  p.q = q;
  p.ldq = ld_q;
  p.scale = scales;
  return launched(launch_norm_rows8(p, (hipStream_t)stream), "RMSNorm to 8 bits");
}

int harp_blk_quantize_int8(const void* x, int64_t ld_x, int x_dtype, int8_t* q, int64_t ld_q, float* scales, int rows,
                           int cols, void* stream) {
  int rc;
  if ((rc = check_rows_cols(rows, cols))) return rc;
  if (rows == 0) return ok();
  if ((rc = check_matrix(x, ld_x, x_dtype, cols, false, "x"))) return rc;
  if ((rc = check_rows8(q, ld_q, cols, INT64_MAX, true, "q"))) return rc;
  if ((rc = check_floats(scales, "scales"))) return rc;
  NormParams p{};
  p.rows = rows;
  p.cols = cols;
  p.x = x;
  p.ldx = ld_x;
  p.x_dtype = x_dtype;
  p.q = q;
  p.ldq = ld_q;
  p.scale = scales;
  return launched(launch_quantize(p, (hipStream_t)stream), "quantise");
}

int harp_blk_dequantize_int8(const int8_t* q, int64_t ld_q, const float* scales, void* out, int64_t ld_out,
                             int out_dtype, int rows, int cols, void* stream) {
  int rc;
  if (rows < 0 || cols < 1) return fail(HARP_BLK_EINVAL, "rows=%d, cols=%d: rows of at least one value", rows, cols);
  if (cols > kMaxTokens) return fail(HARP_BLK_EUNSUPPORTED, "cols=%d > 2^30", cols);  // indexes of a row stay in 32 bits
  if (rows == 0) return ok();
  if ((rc = check_rows8(q, ld_q, cols, INT64_MAX, false, "q"))) return rc;
  if ((rc = check_floats(scales, "scales"))) return rc;
  if ((rc = check_matrix(out, ld_out, out_dtype, cols, true, "out"))) return rc;
  return launched(launch_dequantize(q, ld_q, scales, out, ld_out, out_dtype, rows, cols, (hipStream_t)stream),
                  "dequantise");
}

int harp_blk_linear_int8(const int8_t* x, int64_t ld_x, const float* x_scales, const int8_t* w, int64_t ld_w,
                         const float* w_scales, const void* bias, int bias_dtype, void* y, int64_t ld_y, int y_dtype,
                         int M, int N, int K, void* stream) {
  int rc;
  if (M < 0 || N < 1 || K < 1) return fail(HARP_BLK_EINVAL, "M=%d, N=%d, K=%d: N and K must be positive", M, N, K);
  if (K > kMaxK) return fail(HARP_BLK_EUNSUPPORTED, "K=%d > %d is not supported", K, kMaxK);
  if (M > kMaxTokens || N > kMaxTokens) return fail(HARP_BLK_EUNSUPPORTED, "M=%d, N=%d: more than 2^30", M, N);
  if (M == 0) return ok();
  if ((rc = check_rows8(x, ld_x, K, kMaxLd8, false, "x"))) return rc;
  if ((rc = check_floats(x_scales, "x_scales"))) return rc;
  if ((rc = check_rows8(w, ld_w, K, kMaxLd8, false, "w"))) return rc;
  if ((rc = check_floats(w_scales, "w_scales"))) return rc;
  if ((rc = check_vector(bias, bias_dtype, "bias"))) return rc;
  if ((rc = check_matrix(y, ld_y, y_dtype, N, true, "y"))) return rc;
  Prod8Params p{};
  p.x = x;
  p.ldx = ld_x;
  p.x_scale = x_scales;
  p.M = M;
  p.N = N;
  p.K = K;
  p.S = M;
  p.n_outs = 1;
  Prod8Out& o = p.out[0];
  o.w = w;
  o.ldw = ld_w;
  o.w_scale = w_scales;
  o.bias = bias;
  o.bias_f32 = bias_dtype == HARP_BLK_F32;
  o.y = y;
  o.ldy = ld_y;
  o.y_f32 = y_dtype == HARP_BLK_F32;
  return launched(launch_prod8(p, (hipStream_t)stream), "8-bit product");
}

int harp_blk_qkv_int8(const int8_t* x, int64_t ld_x, const float* x_scales, int batch, int seq, int k_dim, int n_out,
                      const float* freqs, int64_t f_stride_b, int64_t f_stride_s, const harp_blk_qkv_out_t* outs,
                      int n_outs, void* stream) {
  int rc;
  if (batch < 0 || seq < 0) return fail(HARP_BLK_EINVAL, "batch=%d and seq=%d must not be negative", batch, seq);
  if ((int64_t)batch * seq > kMaxTokens) return fail(HARP_BLK_EUNSUPPORTED, "batch * seq > 2^30");
  if (k_dim < 1) return fail(HARP_BLK_EINVAL, "k_dim=%d must be positive", k_dim);
  if (k_dim > kMaxK) return fail(HARP_BLK_EUNSUPPORTED, "k_dim=%d > %d is not supported", k_dim, kMaxK);
  if (n_out < 128 || n_out % 128)
    return fail(HARP_BLK_EUNSUPPORTED, "n_out=%d must be a positive multiple of 128 (heads of 128)", n_out);
  if (n_out > kMaxTokens) return fail(HARP_BLK_EUNSUPPORTED, "n_out=%d > 2^30", n_out);
  if (!outs || n_outs < 1 || n_outs > kMaxOuts8)
    return fail(HARP_BLK_EINVAL, "outs must hold 1 to %d outputs (got %d)", kMaxOuts8, n_outs);
  if ((int64_t)batch * seq == 0) return ok();
  if ((rc = check_rows8(x, ld_x, k_dim, kMaxLd8, false, "x"))) return rc;
  if ((rc = check_floats(x_scales, "x_scales"))) return rc;
  if (freqs) {
    if (!aligned(freqs, 16)) return fail(HARP_BLK_EINVAL, "freqs must be 16-byte aligned");
    if (f_stride_b < 0 || f_stride_s < 0 || f_stride_b % 4 || f_stride_s % 4)
      return fail(HARP_BLK_EINVAL, "freqs strides (%lld, %lld) must be non-negative multiples of 4 floats",
                  (long long)f_stride_b, (long long)f_stride_s);
  }
  Prod8Params p{};
  p.x = x;
  p.ldx = ld_x;
  p.x_scale = x_scales;
  p.M = batch * seq;
  p.N = n_out;
  p.K = k_dim;
  p.S = seq;
  p.freqs = freqs;
  p.f_stride_b = f_stride_b;
  p.f_stride_s = f_stride_s;
  p.n_outs = n_outs;
  for (int i = 0; i < n_outs; ++i) {
    const harp_blk_qkv_out_t& s = outs[i];
    char name[32];
    snprintf(name, sizeof(name), "outs[%d].weight", i);
    if ((rc = check_rows8(s.weight, s.ld_weight, k_dim, kMaxLd8, false, name))) return rc;
    snprintf(name, sizeof(name), "outs[%d].weight_scales", i);
    if ((rc = check_floats(s.weight_scales, name))) return rc;
    snprintf(name, sizeof(name), "outs[%d].y", i);
    if ((rc = check_matrix(s.y, s.ld_y, HARP_BLK_BF16, n_out, true, name))) return rc;
    snprintf(name, sizeof(name), "outs[%d].norm_weight", i);
    if ((rc = check_vector(s.norm_weight, s.norm_weight_dtype, name))) return rc;
    if (s.norm_weight && (rc = check_eps(s.eps))) return rc;
    Prod8Out& o = p.out[i];
    o.w = s.weight;
    o.ldw = s.ld_weight;
    o.w_scale = s.weight_scales;
    o.y = s.y;
    o.ldy = s.ld_y;
    o.norm_w = s.norm_weight;
    o.norm_w_f32 = s.norm_weight && s.norm_weight_dtype == HARP_BLK_F32;
    o.eps = s.eps;
  }
  return launched(launch_prod8(p, (hipStream_t)stream), "8-bit q/k/v projection");
}

}  // extern "C"
