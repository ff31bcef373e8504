// kernels/libharp_block_ops.so — PyTorch-ROCm operators of the kernels around
// the attention block (include/harp_block_ops.h), namespace harp_block:
//   add_rms_norm                                    residual addition + RMSNorm
//   add_rms_norm_int8, quantize_int8, dequantize_int8
//   linear_int8, linear_int8_dynamic, qkv_int8      products of 8-bit rows
// The operators allocate their results from PyTorch's allocator and run on
// the current HIP stream of the input's device.  Implementations are
// registered for the CUDA dispatch key (HIP tensors carry it); the CPU key
// raises.  add_rms_norm is differentiable (once, in reverse mode); the others
// have no derivative, and where a gradient would be recorded, or an argument
// carries a forward-mode tangent, a call raises.
//
// Matrices are [.., C] tensors read as rows of C elements.  A tensor whose
// leading dimensions are no single row stride, or whose last stride is not 1,
// is copied first.  8-bit rows are never copied: they come from the operators
// here, whose storage pads each row to 16 bytes.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <string>
#include <tuple>

#include "harp_block_ops.h"
#include "torch_autograd_util.h"

namespace {

using harp_torch::given;
using harp_torch::OptTensor;

void check_status(int rc, const char* op) {
  TORCH_CHECK(rc == HARP_BLK_OK, "harp_block.", op, ": ", harp_blk_last_error(), " (status ", rc, ")");
}

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

int code(at::ScalarType t) { return t == at::kFloat ? HARP_BLK_F32 : HARP_BLK_BF16; }

void check_float(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == ref.device(), name, " must be on the HIP device ", ref.device());
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, name,
              " must be bfloat16 or float32, got ", t.scalar_type());
}

// rows of the last dimension: a tensor (kept alive), its pointer, row stride and count
struct Rows {
  at::Tensor t;
  const void* p = nullptr;
  int64_t ld = 0, rows = 0, cols = 0;
};

int checked_int(int64_t v, const char* name) {
  TORCH_CHECK(v <= 0x40000000, name, " of ", v, " is more than 2^30");
  return (int)v;
}

Rows rows_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() >= 1, name, " must have at least one dimension");
  Rows r;
  r.cols = t.size(-1);
  TORCH_CHECK(r.cols >= 1, name, " must have a last dimension of at least 1");
  r.rows = t.numel() / r.cols;
  checked_int(r.rows, "rows");
  // (the dispatcher resolves a negated view only for what is called through it)
  r.t = t.is_neg() ? t.resolve_neg() : t;
  if (r.t.stride(-1) != 1 && r.cols != 1) r.t = r.t.contiguous();
  if (r.t.dim() != 2) r.t = r.t.reshape({r.rows, r.cols});
  r.p = r.t.const_data_ptr();
  r.ld = r.rows > 1 ? r.t.stride(0) : r.cols;
  if (r.cols == 1 && r.rows > 1 && r.ld < 1) r.ld = 0;
  return r;
}

// [C] vector or none; empty optional = none
struct Vec {
  at::Tensor t;
  const void* p = nullptr;
  int dtype = HARP_BLK_BF16;
};
Vec vec_of(const OptTensor& v, const at::Tensor& ref, int64_t n, const char* name) {
  Vec r;
  if (!v.has_value() || !v->defined()) return r;
  check_float(*v, ref, name);
  TORCH_CHECK(v->dim() == 1 && v->numel() == n, name, " must be a vector of ", n, " elements, got ", v->sizes());
  r.t = (v->is_neg() ? v->resolve_neg() : *v).contiguous();
  r.p = r.t.const_data_ptr();
  r.dtype = code(r.t.scalar_type());
  return r;
}

void refuse_tangent(const at::Tensor& t, const char* op) {
  harp_torch::refuse_tangent(t, "harp_block", op);
}

void check_input(const at::Tensor& x, const char* op) {
  TORCH_CHECK(x.is_cuda(), "harp_block.", op, ": tensors must be on a HIP device");
  check_float(x, x, "x");
}

void check_residual(const at::Tensor& residual, const at::Tensor& x) {
  check_float(residual, x, "residual");
  TORCH_CHECK(residual.sizes() == x.sizes(), "residual must have x's shape ", x.sizes(), ", got ", residual.sizes());
}

// ---------------------------------------------------------------------------
// (y, h, rstd); h is undefined without a residual, rstd without keep
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_forward(const at::Tensor& x, const OptTensor& residual,
                                                                    const OptTensor& weight, double eps, bool keep) {
  check_input(x, "add_rms_norm");
  if (given(residual)) check_residual(*residual, x);
  const c10::DeviceGuard guard(x.device());
  const Rows xr = rows_of(x, "x");
  const Vec w = vec_of(weight, x, xr.cols, "weight");
  at::Tensor y = at::empty(x.sizes(), x.options());
  at::Tensor h, rstd;
  if (keep) rstd = at::empty({xr.rows}, x.options().dtype(at::kFloat));
  Rows rr;
  if (given(residual)) {
    rr = rows_of(*residual, "residual");
    h = at::empty(x.sizes(), residual->options());
  }
  if (xr.rows)
    check_status(harp_blk_add_rms_norm_forward(xr.p, xr.ld, code(x.scalar_type()), rr.p, rr.ld,
                                               rr.p ? code(rr.t.scalar_type()) : HARP_BLK_BF16, w.p, w.dtype,
                                               (float)eps, y.data_ptr(), xr.cols, h.defined() ? h.data_ptr() : nullptr,
                                               xr.cols, keep ? rstd.data_ptr<float>() : nullptr, (int)xr.rows,
                                               checked_int(xr.cols, "cols"), stream_of(x)),
                 "add_rms_norm");
  return {y, h, rstd};
}

// (dx, dresidual, grad_weight): dresidual is undefined where it equals dx
// (same type) or is not wanted, grad_weight without want_weight
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_backward(const at::Tensor& dy, const at::Tensor& dh,
                                                                     const at::Tensor& h, const at::Tensor& weight,
                                                                     const at::Tensor& rstd, bool want_residual,
                                                                     bool want_weight) {
  const c10::DeviceGuard guard(dy.device());
  const Rows dyr = rows_of(dy, "dy"), hr = rows_of(h, "h");
  Rows dhr;
  if (dh.defined()) dhr = rows_of(dh, "dh");
  const Vec w = vec_of(weight, dy, dyr.cols, "weight");
  at::Tensor dx = at::empty(dy.sizes(), dy.options()), dres, gw, ws;
  if (want_residual && h.scalar_type() != dy.scalar_type()) dres = at::empty(dy.sizes(), h.options());
  if (want_weight) gw = at::empty({dyr.cols}, w.t.options());
  const int rows = (int)dyr.rows, cols = checked_int(dyr.cols, "cols");
  if (rows == 0) {
    if (want_weight) gw.zero_();
    return {dx, dres, gw};
  }
  size_t wsb = 0;
  if (want_weight) {
    wsb = harp_blk_backward_workspace_bytes(rows, cols);
    TORCH_CHECK(wsb != (size_t)-1, "harp_block.add_rms_norm: ", harp_blk_last_error());
    ws = at::empty({(int64_t)(wsb / 4)}, dy.options().dtype(at::kFloat));
  }
  check_status(
      harp_blk_add_rms_norm_backward(dyr.p, dyr.ld, code(dy.scalar_type()), dhr.p, dhr.ld, hr.p, hr.ld,
                                     code(h.scalar_type()), w.p, w.dtype, rstd.const_data_ptr<float>(), dx.data_ptr(),
                                     cols, dres.defined() ? dres.data_ptr() : nullptr, cols,
                                     want_weight ? gw.data_ptr() : nullptr, w.dtype, rows, cols,
                                     want_weight ? ws.data_ptr() : nullptr, wsb, stream_of(dy)),
      "add_rms_norm (backward)");
  return {dx, dres, gw};
}

// (y, h) without a gradient; h is undefined (None) without a residual: no result shares memory with x
std::tuple<at::Tensor, at::Tensor> add_rms_norm(const at::Tensor& x, const OptTensor& residual,
                                                const OptTensor& weight, double eps) {
  auto [y, h, rstd] = add_rms_norm_forward(x, residual, weight, eps, false);
  return {y, h};
}

// The differentiable form: y, and h where there is a residual.
class AddRMSNorm : public torch::autograd::Function<AddRMSNorm> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                const OptTensor& residual, const OptTensor& weight, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, h, rstd] = add_rms_norm_forward(x, residual, weight, eps, true);
    ctx->set_materialize_grads(false);
    // x's type, and which of the three gradients are wanted
    ctx->saved_data["wanted"] = (int64_t)x.scalar_type() * 8 + x.requires_grad() +
                                2 * (given(residual) && residual->requires_grad()) +
                                4 * (given(weight) && weight->requires_grad());
    const at::Tensor w = given(weight) ? *weight : at::Tensor();
    if (!given(residual)) {
      ctx->save_for_backward({x, w, rstd});
      return {y};
    }
    ctx->save_for_backward({h, w, rstd});
    return {y, h};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const int64_t wanted = ctx->saved_data["wanted"].toInt();
    const bool need_x = wanted & 1, need_residual = wanted & 2, need_weight = wanted & 4;
    const at::Tensor &h = saved[0], &w = saved[1], &rstd = saved[2], &dy = grads[0];
    const at::Tensor dh = grads.size() > 1 ? grads[1] : at::Tensor();
    for (const auto& t : grads) refuse_tangent(t, "add_rms_norm (backward)");
    torch::autograd::variable_list out(4);
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      if (dy.defined()) {
        auto [dx, dres, gw] = add_rms_norm_backward(dy, dh, h, w, rstd, need_residual, need_weight);
        if (need_x) out[0] = dx;
        if (need_residual) out[1] = dres.defined() ? dres : dx;
        if (need_weight) out[2] = gw;
      } else if (dh.defined()) {  // y took no part: the addition alone
        if (need_x) out[0] = dh.to((at::ScalarType)(wanted / 8));
        if (need_residual) out[1] = dh;
      }
    }
    harp_torch::once_only(out, "add_rms_norm");
    return out;
  }
};

void check_capture(const OptTensor& t, const char* name) {
  harp_torch::check_capture(t, "add_rms_norm", name);
}

void refuse_tangents(const at::Tensor& x, const OptTensor& residual, const OptTensor& weight) {
  refuse_tangent(x, "add_rms_norm");
  if (given(residual)) refuse_tangent(*residual, "add_rms_norm");
  if (given(weight)) refuse_tangent(*weight, "add_rms_norm");
}

std::tuple<at::Tensor, at::Tensor> add_rms_norm_autograd(const at::Tensor& x, const OptTensor& residual,
                                                         const OptTensor& weight, double eps) {
  refuse_tangents(x, residual, weight);
  const bool record = at::GradMode::is_enabled() &&
                      (x.requires_grad() || (given(residual) && residual->requires_grad()) ||
                       (given(weight) && weight->requires_grad()));
  if (!record) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return add_rms_norm(x, residual, weight, eps);
  }
  const c10::DeviceGuard guard(x.device());  // the capture of x's device
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
    check_capture(x, "x");
    check_capture(residual, "residual");
    check_capture(weight, "weight");
  }
  auto out = AddRMSNorm::apply(x, residual, weight, eps);
  return {out[0], given(residual) ? out[1] : at::Tensor()};
}

// int8 values of shape `sizes` whose rows are padded to 16 bytes
at::Tensor empty_rows8(at::IntArrayRef sizes, const at::Tensor& like) {
  std::vector<int64_t> full(sizes.begin(), sizes.end());
  const int64_t cols = full.back();
  full.back() = (cols + 15) / 16 * 16;
  return at::empty(full, like.options().dtype(at::kChar)).narrow(-1, 0, cols);
}
int64_t ld8(int64_t cols) { return (cols + 15) / 16 * 16; }

at::Tensor empty_scales(const at::Tensor& x) {
  return at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
}

// (values, scales, h); h is empty without a residual
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_int8(const at::Tensor& x, const OptTensor& residual,
                                                                 const OptTensor& weight, double eps) {
  check_input(x, "add_rms_norm_int8");
  if (given(residual)) check_residual(*residual, x);
  const c10::DeviceGuard guard(x.device());
  const Rows xr = rows_of(x, "x");
  const Vec w = vec_of(weight, x, xr.cols, "weight");
  at::Tensor q = empty_rows8(x.sizes(), x), scales = empty_scales(x), h;
  Rows rr;
  if (given(residual)) {
    rr = rows_of(*residual, "residual");
    h = at::empty(x.sizes(), residual->options());
  } else {
    h = at::empty({0}, x.options());
  }
  if (xr.rows)
    check_status(harp_blk_add_rms_norm_int8(xr.p, xr.ld, code(x.scalar_type()), rr.p, rr.ld,
                                            rr.p ? code(rr.t.scalar_type()) : HARP_BLK_BF16, w.p, w.dtype, (float)eps,
                                            rr.p ? h.data_ptr() : nullptr, xr.cols, q.data_ptr<int8_t>(),
                                            ld8(xr.cols), scales.data_ptr<float>(), (int)xr.rows,
                                            checked_int(xr.cols, "cols"), stream_of(x)),
                 "add_rms_norm_int8");
  return {q, scales, h};
}

std::tuple<at::Tensor, at::Tensor> quantize_int8(const at::Tensor& x) {
  check_input(x, "quantize_int8");
  const c10::DeviceGuard guard(x.device());
  const Rows xr = rows_of(x, "x");
  at::Tensor q = empty_rows8(x.sizes(), x), scales = empty_scales(x);
  if (xr.rows)
    check_status(harp_blk_quantize_int8(xr.p, xr.ld, code(x.scalar_type()), q.data_ptr<int8_t>(), ld8(xr.cols),
                                        scales.data_ptr<float>(), (int)xr.rows, checked_int(xr.cols, "cols"),
                                        stream_of(x)),
                 "quantize_int8");
  return {q, scales};
}

// 8-bit rows given by a caller: values [.., K] with 16-byte aligned rows, scales [..]
struct Rows8 {
  at::Tensor v, s;
  const int8_t* p = nullptr;
  const float* scales = nullptr;
  int64_t ld = 0, rows = 0, cols = 0;
};
Rows8 rows8_of(const at::Tensor& values, const at::Tensor& scales, const char* name) {
  TORCH_CHECK(values.is_cuda(), name, " must be on a HIP device");
  TORCH_CHECK(values.scalar_type() == at::kChar, name, " values must be int8, got ", values.scalar_type());
  TORCH_CHECK(values.dim() >= 1 && values.size(-1) >= 1, name, " values must be rows of at least one element");
  TORCH_CHECK(scales.device() == values.device() && scales.scalar_type() == at::kFloat, name,
              " scales must be float32 on ", values.device());
  TORCH_CHECK(scales.sizes() == values.sizes().slice(0, values.dim() - 1), name, " needs one scale for each row: shape ",
              values.sizes().slice(0, values.dim() - 1), ", got ", scales.sizes());
  Rows8 r;
  r.cols = values.size(-1);
  r.rows = values.numel() / r.cols;
  checked_int(r.rows, "rows");
  checked_int(r.cols, "columns");
  r.v = values;
  if (values.dim() != 2) {
    // leading dimensions of one row stride, or this raises
    r.v = values.dim() == 1 ? values.unsqueeze(0) : values.view({r.rows, r.cols});
  }
  TORCH_CHECK(r.v.stride(1) == 1 || r.cols == 1, name, " values must have unit stride along a row");
  r.ld = r.rows > 1 ? r.v.stride(0) : ld8(r.cols);
  TORCH_CHECK(r.ld == 0 || (r.ld % 16 == 0 && r.ld >= r.cols), name, " values need rows at multiples of 16 bytes, as quantize_int8 "
              "and add_rms_norm_int8 lay them out; got a row stride of ", r.ld, " for ", r.cols, " columns");
  r.s = scales.contiguous();
  r.p = r.v.const_data_ptr<int8_t>();
  r.scales = r.s.const_data_ptr<float>();
  return r;
}

at::Tensor dequantize_int8(const at::Tensor& values, const at::Tensor& scales, at::ScalarType dtype) {
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, "dequantize_int8: bfloat16 or float32, got ", dtype);
  const Rows8 r = rows8_of(values, scales, "rows");
  const c10::DeviceGuard guard(values.device());
  at::Tensor out = at::empty(values.sizes(), values.options().dtype(dtype));
  if (r.rows)
    check_status(harp_blk_dequantize_int8(r.p, r.ld, r.scales, out.data_ptr(), r.cols, code(dtype), (int)r.rows,
                                          (int)r.cols, stream_of(values)),
                 "dequantize_int8");
  return out;
}

// 8-bit rows x times those of weight; in_features: times weight's first
// in_features columns (a module's padded storage, without a view of it)
at::Tensor linear_int8(const at::Tensor& x, const at::Tensor& x_scales, const at::Tensor& weight,
                       const at::Tensor& weight_scales, const OptTensor& bias, at::ScalarType dtype,
                       std::optional<int64_t> in_features) {
  TORCH_CHECK(dtype == at::kBFloat16 || dtype == at::kFloat, "linear_int8: bfloat16 or float32, got ", dtype);
  const Rows8 xr = rows8_of(x, x_scales, "x");
  TORCH_CHECK(!in_features || *in_features == xr.cols, "x must have ", *in_features, " columns, got ", xr.cols);
  TORCH_CHECK(weight.dim() == 2 && (in_features ? weight.size(1) >= xr.cols : weight.size(1) == xr.cols) &&
                  weight.device() == x.device(),
              "weight must be [N, ", xr.cols, "] on ", x.device(), ", got ", weight.sizes(), " on ", weight.device());
  const Rows8 wr = rows8_of(weight, weight_scales, "weight");
  const c10::DeviceGuard guard(x.device());
  const Vec b = vec_of(bias, x, wr.rows, "bias");
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = wr.rows;
  at::Tensor y = at::empty(shape, x.options().dtype(dtype));
  if (xr.rows && wr.rows)
    check_status(harp_blk_linear_int8(xr.p, xr.ld, xr.scales, wr.p, wr.ld, wr.scales, b.p, b.dtype, y.data_ptr(),
                                      wr.rows, code(dtype), (int)xr.rows, (int)wr.rows, (int)xr.cols, stream_of(x)),
                 "linear_int8");
  return y;
}

// the same of a bf16 or fp32 tensor, quantised first
at::Tensor linear_int8_dynamic(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& weight_scales,
                               const OptTensor& bias, at::ScalarType dtype, std::optional<int64_t> in_features) {
  const auto [q, scales] = quantize_int8(x);
  return linear_int8(q, scales, weight, weight_scales, bias, dtype, in_features);
}

// fp32 (cos, sin) rows of the complex [S, 64] or [B or 1, S, 64] table
struct Freqs {
  at::Tensor t;
  int64_t sb = 0, ss = 0;
};
Freqs freqs_of(const at::Tensor& f, const at::Tensor& x, int64_t B, int64_t S) {
  TORCH_CHECK(f.is_cuda() && f.device() == x.device(), "freqs_cis must be on the input's device");
  at::Tensor r = f.is_complex() ? at::view_as_real(f).flatten(-2) : f;
  TORCH_CHECK(r.scalar_type() == at::kFloat, "freqs_cis must be complex64 [.., S, 64], or float32 (cos, sin) rows [.., S, 128]");
  r = r.contiguous();
  TORCH_CHECK((r.dim() == 2 || r.dim() == 3) && r.size(-1) == 128 && r.size(-2) == S,
              "freqs_cis must be complex [S, 64] or [B, S, 64], or float32 (cos, sin) rows [.., S, 128], with S=", S,
              ", got ", f.sizes());
  TORCH_CHECK(r.dim() == 2 || r.size(0) == B || r.size(0) == 1, "freqs_cis batch must be 1 or ", B);
  Freqs q;
  q.t = r;
  q.ss = 128;
  q.sb = r.dim() == 3 && r.size(0) > 1 ? r.stride(0) : 0;
  return q;
}

// [B, H, S, 128] views of token-major storage, one for each weight
std::vector<at::Tensor> qkv_int8(const at::Tensor& x, const at::Tensor& x_scales,
                                 const std::vector<at::Tensor>& weights, const std::vector<at::Tensor>& weight_scales,
                                 const c10::List<OptTensor>& norm_weights, const std::vector<double>& eps,
                                 const OptTensor& freqs_cis) {
  TORCH_CHECK(x.dim() == 3, "x must be [B, S, dim] rows, got ", x.sizes());
  const size_t n = weights.size();
  TORCH_CHECK(n >= 1 && n <= 3 && weight_scales.size() == n && norm_weights.size() == n && eps.size() == n,
              "one to three weights with a scale vector, a norm weight (or None) and an eps each");
  const int64_t B = x.size(0), S = x.size(1), K = x.size(2), N = weights[0].size(0);
  const Rows8 xr = rows8_of(x, x_scales, "x");
  const c10::DeviceGuard guard(x.device());
  TORCH_CHECK(N >= 128 && N % 128 == 0, "weights must have heads of 128 features, got ", N, " rows");
  Freqs f;
  if (given(freqs_cis)) f = freqs_of(*freqs_cis, x, B, S);
  harp_blk_qkv_out_t outs[3] = {};
  std::vector<Rows8> wr;
  std::vector<Vec> nv;
  std::vector<at::Tensor> ys;
  for (size_t i = 0; i < n; ++i) {
    TORCH_CHECK(weights[i].dim() == 2 && weights[i].size(0) == N && weights[i].size(1) == K &&
                    weights[i].device() == x.device(),
                "every weight must be [", N, ", ", K, "] on ", x.device(), ", got ", weights[i].sizes(), " on ",
                weights[i].device());
    wr.push_back(rows8_of(weights[i], weight_scales[i], "weight"));
    const OptTensor nw = norm_weights.get(i);
    nv.push_back(vec_of(nw, x, 128, "norm weight"));
    TORCH_CHECK(nv[i].p || !f.t.defined() || i == 2, "RoPE without RMSNorm is the separate operator's");
    ys.push_back(at::empty({B, S, N}, x.options().dtype(at::kBFloat16)));
    harp_blk_qkv_out_t& o = outs[i];
    o.weight = wr[i].p;
    o.ld_weight = wr[i].ld;
    o.weight_scales = wr[i].scales;
    o.y = ys[i].data_ptr();
    o.ld_y = N;
    o.norm_weight = nv[i].p;
    o.norm_weight_dtype = nv[i].dtype;
    o.eps = (float)eps[i];
  }
  if (xr.rows)
    check_status(harp_blk_qkv_int8(xr.p, xr.ld, xr.scales, (int)B, (int)S, (int)K, (int)N,
                                   f.t.defined() ? f.t.const_data_ptr<float>() : nullptr, f.sb, f.ss, outs, (int)n,
                                   stream_of(x)),
                 "qkv_int8");
  for (auto& y : ys) y = y.unflatten(-1, {N / 128, 128}).transpose(1, 2);
  return ys;
}

[[noreturn]] void no_cpu(const char* op) {
  TORCH_CHECK(false, "harp_block.", op, ": this library runs on a HIP device only (CPU tensors given)");
}
std::tuple<at::Tensor, at::Tensor> add_rms_norm_cpu(const at::Tensor&, const OptTensor&, const OptTensor&, double) {
  no_cpu("add_rms_norm");
}
std::tuple<at::Tensor, at::Tensor> add_rms_norm_autograd_cpu(const at::Tensor& x, const OptTensor& residual,
                                                             const OptTensor& weight, double) {
  refuse_tangents(x, residual, weight);
  no_cpu("add_rms_norm");
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_rms_norm_int8_cpu(const at::Tensor&, const OptTensor&,
                                                                     const OptTensor&, double) {
  no_cpu("add_rms_norm_int8");
}
std::tuple<at::Tensor, at::Tensor> quantize_int8_cpu(const at::Tensor&) { no_cpu("quantize_int8"); }
at::Tensor dequantize_int8_cpu(const at::Tensor&, const at::Tensor&, at::ScalarType) { no_cpu("dequantize_int8"); }
at::Tensor linear_int8_cpu(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                           const OptTensor&, at::ScalarType, std::optional<int64_t>) {
  no_cpu("linear_int8");
}
at::Tensor linear_int8_dynamic_cpu(const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&,
                                   at::ScalarType, std::optional<int64_t>) {
  no_cpu("linear_int8_dynamic");
}
std::vector<at::Tensor> qkv_int8_cpu(const at::Tensor&, const at::Tensor&, const std::vector<at::Tensor>&,
                                     const std::vector<at::Tensor>&, const c10::List<OptTensor>&,
                                     const std::vector<double>&, const OptTensor&) {
  no_cpu("qkv_int8");
}

// ---------------------------------------------------------------------------
// The autograd kernels of the operators without a derivative: the checks, then
// the operator below the autograd keys.
void refuse_derivative(const char* op, const at::Tensor& t) {
  refuse_tangent(t, op);
  TORCH_CHECK(!t.defined() || !t.requires_grad() || !at::GradMode::is_enabled(), "harp_block.", op,
              " is forward only: call it under torch.no_grad(), or on tensors that need no gradient");
}
void refuse_derivative(const char* op, const OptTensor& t) {
  if (t.has_value()) refuse_derivative(op, *t);
}
void refuse_derivative(const char* op, const std::vector<at::Tensor>& ts) {
  for (const auto& t : ts) refuse_derivative(op, t);
}
void refuse_derivative(const char* op, const c10::List<OptTensor>& ts) {
  for (size_t i = 0; i < ts.size(); ++i) refuse_derivative(op, ts.get(i));
}
template <class T>
void refuse_derivative(const char*, const T&) {}  // no tensor

constexpr char kAddRmsNormInt8[] = "add_rms_norm_int8", kQuantizeInt8[] = "quantize_int8",
               kDequantizeInt8[] = "dequantize_int8", kLinearInt8[] = "linear_int8",
               kLinearInt8Dynamic[] = "linear_int8_dynamic", kQkvInt8[] = "qkv_int8";

template <const char* OP, class F>
struct ForwardOnly;
template <const char* OP, class R, class... Args>
struct ForwardOnly<OP, R(Args...)> {
  static R call(Args... args) {
    (refuse_derivative(OP, args), ...);
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow((std::string("harp_block::") + OP).c_str(), "")
                               .template typed<R(Args...)>();
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(args...);
  }
};

void forward_only_kernels(torch::Library& m) {
  m.impl(kAddRmsNormInt8, &ForwardOnly<kAddRmsNormInt8, decltype(add_rms_norm_int8)>::call);
  m.impl(kQuantizeInt8, &ForwardOnly<kQuantizeInt8, decltype(quantize_int8)>::call);
  m.impl(kDequantizeInt8, &ForwardOnly<kDequantizeInt8, decltype(dequantize_int8)>::call);
  m.impl(kLinearInt8, &ForwardOnly<kLinearInt8, decltype(linear_int8)>::call);
  m.impl(kLinearInt8Dynamic, &ForwardOnly<kLinearInt8Dynamic, decltype(linear_int8_dynamic)>::call);
  m.impl(kQkvInt8, &ForwardOnly<kQkvInt8, decltype(qkv_int8)>::call);
}

}  // namespace

TORCH_LIBRARY(harp_block, m) {
  m.def("add_rms_norm(Tensor x, Tensor? residual, Tensor? weight, float eps) -> (Tensor, Tensor)");
  m.def("add_rms_norm_int8(Tensor x, Tensor? residual, Tensor? weight, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("quantize_int8(Tensor x) -> (Tensor, Tensor)");
  m.def("dequantize_int8(Tensor values, Tensor scales, ScalarType dtype) -> Tensor");
  m.def(
      "linear_int8(Tensor x, Tensor x_scales, Tensor weight, Tensor weight_scales, Tensor? bias, ScalarType dtype, "
      "int? in_features=None) -> Tensor");
  m.def(
      "linear_int8_dynamic(Tensor x, Tensor weight, Tensor weight_scales, Tensor? bias, ScalarType dtype, int? "
      "in_features=None) -> Tensor");
  m.def(
      "qkv_int8(Tensor x, Tensor x_scales, Tensor[] weights, Tensor[] weight_scales, Tensor?[] norm_weights, float[] "
      "eps, Tensor? freqs_cis) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(harp_block, AutogradCUDA, m) {
  m.impl("add_rms_norm", &add_rms_norm_autograd);
  forward_only_kernels(m);
}

TORCH_LIBRARY_IMPL(harp_block, AutogradCPU, m) {
  m.impl("add_rms_norm", &add_rms_norm_autograd_cpu);
  forward_only_kernels(m);
}

TORCH_LIBRARY_IMPL(harp_block, CUDA, m) {
  m.impl("add_rms_norm", &add_rms_norm);
  m.impl("add_rms_norm_int8", &add_rms_norm_int8);
  m.impl("quantize_int8", &quantize_int8);
  m.impl("dequantize_int8", &dequantize_int8);
  m.impl("linear_int8", &linear_int8);
  m.impl("linear_int8_dynamic", &linear_int8_dynamic);
  m.impl("qkv_int8", &qkv_int8);
}

TORCH_LIBRARY_IMPL(harp_block, CPU, m) {
  m.impl("add_rms_norm", &add_rms_norm_cpu);
  m.impl("add_rms_norm_int8", &add_rms_norm_int8_cpu);
  m.impl("quantize_int8", &quantize_int8_cpu);
  m.impl("dequantize_int8", &dequantize_int8_cpu);
  m.impl("linear_int8", &linear_int8_cpu);
  m.impl("linear_int8_dynamic", &linear_int8_dynamic_cpu);
  m.impl("qkv_int8", &qkv_int8_cpu);
}
