// kernels/libharp_request_ops.so — PyTorch-ROCm operators of the kernels that
// give every request of a batch its own positions and its own adapter
// (include/harp_request_ops.h), namespace harp_request:
//   qk_norm_rope    RMSNorm and rotation of queries and keys by their positions
//   rope_table      the rotation's table
//   add_adapters    low-rank adapters beside a projection's result
//   qkv_adapters    the q/k/v producer with adapters beside its projections
// The operators allocate their results and workspaces from PyTorch's allocator
// and run on the current HIP stream of the input's device.  Implementations are
// registered for the CUDA dispatch key (HIP tensors carry it); the CPU key
// raises.  qk_norm_rope and add_adapters are differentiable (once, in reverse
// mode), and so is qkv_adapters where its rotation is given as positions; an argument
// with a forward-mode tangent raises.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <cstring>
#include <string>
#include <tuple>
#include <type_traits>
#include <vector>

#include "harp_request_ops.h"
#include "torch_autograd_util.h"

namespace {

using harp_torch::given;
using harp_torch::OptTensor;

void check_status(int rc, const char* op) {
  TORCH_CHECK(rc == HARP_REQ_OK, "harp_request.", op, ": ", harp_req_last_error(), " (status ", rc, ")");
}
hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
int code(at::ScalarType t) { return t == at::kFloat ? HARP_REQ_F32 : HARP_REQ_BF16; }
int int_code(at::ScalarType t) { return t == at::kLong ? HARP_REQ_I64 : HARP_REQ_I32; }

int checked_int(int64_t v, const char* name) {
  TORCH_CHECK(v <= 0x7fffffff, name, " of ", v, " is 2^31 or more");
  return (int)v;
}
void check_device(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.device() == ref.device(), name, " must be on ", ref.device(), ", got ", t.device());
}
at::Tensor plain(const at::Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
struct Axes {
  harp_req_axes_t a{};
  int64_t D = 0;
};
Axes axes_of(at::IntArrayRef widths, at::ArrayRef<double> theta, bool half) {
  Axes r;
  TORCH_CHECK(widths.size() >= 1 && widths.size() <= HARP_REQ_MAX_AXES && theta.size() == widths.size(),
              "one to four axes with a theta each, got ", widths.size(), " and ", theta.size());
  r.a.n = (int)widths.size();
  r.a.half = half;
  for (size_t i = 0; i < widths.size(); ++i) {
    TORCH_CHECK(widths[i] >= 2 && widths[i] <= 256 && widths[i] % 2 == 0, "an axis' width must be even, 2 to 256, got ",
                widths[i]);
    r.a.width[i] = (int)widths[i];
    r.a.theta[i] = theta[i];
    r.D += widths[i];
  }
  return r;
}

// positions [S, n] or [B or 1, S, n]
struct Positions {
  at::Tensor t;
  harp_req_positions_t p{};
};
Positions positions_of(const at::Tensor& pos, int64_t n, int64_t B, int64_t S) {
  Positions r;
  const auto ty = pos.scalar_type();
  TORCH_CHECK(ty == at::kInt || ty == at::kLong || ty == at::kFloat, "positions must be int32, int64 or float32, got ", ty);
  TORCH_CHECK(pos.dim() == 2 || pos.dim() == 3, "positions must be [S, axes] or [B, S, axes], got ", pos.sizes());
  TORCH_CHECK(pos.size(-1) == n && pos.size(-2) == S && (pos.dim() == 2 || pos.size(0) == B || pos.size(0) == 1),
              "positions must be [", S, ", ", n, "], or [", B, " or 1, ", S, ", ", n, "], got ", pos.sizes());
  r.t = plain(pos);
  r.p.p = r.t.const_data_ptr();
  r.p.dtype = ty == at::kFloat ? HARP_REQ_F32 : int_code(ty);
  r.p.stride_b = pos.dim() == 3 && pos.size(0) > 1 ? r.t.stride(0) : 0;
  r.p.stride_s = r.t.stride(-2);
  r.p.stride_a = r.t.stride(-1);
  return r;
}

// [B, H, S, D] views the kernels read: unit stride along D, the others multiples of 8, 16-byte aligned
bool readable(const at::Tensor& t) {
  if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) % 8 || (i && t.stride(i) > 0x7fffffff))) return false;
  return true;
}
at::Tensor heads_of(const at::Tensor& t) {
  const at::Tensor r = plain(t);
  if (r.numel() == 0 || readable(r)) return r;
  const at::Tensor c = r.contiguous();
  return readable(c) ? c : c.clone(at::MemoryFormat::Contiguous);  // (contiguous, from an odd address on)
}
// x's layout, without the holes it may have; another where the kernels cannot write that
at::Tensor like(const at::Tensor& x) {
  const at::Tensor r = at::empty_like(x);
  return r.numel() == 0 || readable(r) ? r : at::empty(x.sizes(), x.options());
}
void strides_of(const at::Tensor& t, int64_t (&st)[3]) {
  const int order[3] = {0, 1, 2};
  for (int i : order) st[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

at::Tensor weight_of(const OptTensor& w, const at::Tensor& x, const char* name) {
  if (!given(w)) return {};
  check_device(*w, x, name);
  TORCH_CHECK(w->scalar_type() == at::kBFloat16 || w->scalar_type() == at::kFloat, name,
              " must be bfloat16 or float32, got ", w->scalar_type());
  TORCH_CHECK(w->dim() == 1 && w->size(0) == x.size(3), name, " must be a vector of ", x.size(3), " elements, got ",
              w->sizes());
  return plain(*w).contiguous();
}

struct RopeCall {
  Axes axes;
  double eps[2];      // of q and k; negative: no norm
  bool want[4] = {};  // of the gradients of q, k and their weights
};
RopeCall rope_call(at::IntArrayRef widths, at::ArrayRef<double> theta, bool half, at::ArrayRef<double> eps) {
  TORCH_CHECK(eps.size() == 2, "eps must be two values, got ", eps.size());
  return RopeCall{axes_of(widths, theta, half), {eps[0], eps[1]}};
}
// as one saved value (four lists of a call would cost the host some microseconds)
std::string saved(const RopeCall& c) {
  static_assert(std::is_trivially_copyable_v<RopeCall>);
  return std::string(reinterpret_cast<const char*>(&c), sizeof(c));
}
RopeCall restored(const std::string& s) {
  RopeCall c;
  std::memcpy(&c, s.data(), sizeof(c));
  return c;
}

void check_qk(const at::Tensor& q, const OptTensor& k, const at::Tensor& positions, const RopeCall& c,
              const OptTensor& qw, const OptTensor& kw) {
  TORCH_CHECK(q.is_cuda(), "harp_request.qk_norm_rope: tensors must be on a HIP device");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kFloat, "q must be bfloat16 or float32, got ",
              q.scalar_type());
  TORCH_CHECK(q.dim() == 4, "q must be [B, heads, S, D], got ", q.sizes());
  TORCH_CHECK(q.size(3) == c.axes.D, "q has heads of ", q.size(3), " features, the axes ", c.axes.D);
  TORCH_CHECK(c.axes.D % 8 == 0 && c.axes.D <= 256, "heads must have a multiple of 8 features, at most 256, got ", c.axes.D);
  if (given(k)) {
    check_device(*k, q, "k");
    TORCH_CHECK(k->scalar_type() == q.scalar_type(), "k must be ", q.scalar_type(), " as q, got ", k->scalar_type());
    TORCH_CHECK(k->dim() == 4 && k->size(0) == q.size(0) && k->size(2) == q.size(2) && k->size(3) == q.size(3),
                "k must be [", q.size(0), ", heads, ", q.size(2), ", ", q.size(3), "], got ", k->sizes());
  }
  check_device(positions, q, "positions");
  TORCH_CHECK((!given(qw) || c.eps[0] >= 0) && (!given(kw) || c.eps[1] >= 0), "a weight needs its norm: eps is missing");
  TORCH_CHECK(!given(kw) || given(k), "k_weight without k");
  checked_int(q.size(0), "batch");
  checked_int(q.size(1), "heads");
  checked_int(q.size(2), "seq");
}

std::tuple<at::Tensor, at::Tensor> rope_forward(const at::Tensor& q, const OptTensor& k, const at::Tensor& positions,
                                                const RopeCall& c, const OptTensor& qw, const OptTensor& kw) {
  check_qk(q, k, positions, c, qw, kw);
  const c10::DeviceGuard guard(q.device());
  const Positions pos = positions_of(positions, c.axes.a.n, q.size(0), q.size(2));
  harp_req_heads_t heads[2] = {};
  at::Tensor x[2], y[2], w[2];
  for (int i = 0; i < 2; ++i) {
    if (i && !given(k)) break;
    x[i] = heads_of(i ? *k : q);
    y[i] = like(i ? *k : q);
    w[i] = weight_of(i ? kw : qw, q, i ? "k_weight" : "q_weight");
    harp_req_heads_t& h = heads[i];
    h.x = x[i].const_data_ptr();
    strides_of(x[i], h.x_stride);
    h.y = y[i].data_ptr();
    strides_of(y[i], h.y_stride);
    h.heads = checked_int(x[i].size(1), "heads");
    h.norm = c.eps[i] >= 0;
    if (w[i].defined()) {
      h.weight = w[i].const_data_ptr();
      h.weight_dtype = code(w[i].scalar_type());
    }
    h.eps = (float)c.eps[i];
  }
  check_status(harp_req_qk_norm_rope_forward(&c.axes.a, &pos.p, heads, (int)q.size(0), (int)q.size(2),
                                             code(q.scalar_type()), stream_of(q)),
               "qk_norm_rope");
  return {y[0], y[1]};
}

// the gradients of (q, k, q_weight, k_weight); undefined where dy is (its tensor took no part) or not wanted
std::vector<at::Tensor> rope_backward(const at::Tensor (&dy)[2], const at::Tensor (&x)[2], const at::Tensor (&w)[2],
                                      const at::Tensor& positions, const RopeCall& c, const bool (&want_w)[2]) {
  const at::Tensor& ref = dy[0].defined() ? dy[0] : dy[1];
  const c10::DeviceGuard guard(ref.device());
  const Positions pos = positions_of(positions, c.axes.a.n, ref.size(0), ref.size(2));
  harp_req_heads_t heads[2] = {};
  std::vector<at::Tensor> out(4);
  at::Tensor d[2], xs[2], ws[2], work;
  int normed[2] = {0, 0};
  bool any = false;
  for (int i = 0; i < 2; ++i) {
    if (!dy[i].defined()) continue;
    d[i] = heads_of(dy[i]);
    harp_req_heads_t& h = heads[i];
    h.heads = (int)d[i].size(1);
    h.norm = c.eps[i] >= 0;
    if (h.norm) {
      xs[i] = heads_of(x[i]);
      h.x = xs[i].const_data_ptr();
      strides_of(xs[i], h.x_stride);
      normed[i] = h.heads;
      if (w[i].defined()) {
        ws[i] = plain(w[i]).contiguous();
        h.weight = ws[i].const_data_ptr();
        h.weight_dtype = code(ws[i].scalar_type());
        if (want_w[i]) {
          out[2 + i] = d[i].numel() ? at::empty_like(ws[i]) : at::zeros_like(ws[i]);
          h.grad_weight = out[2 + i].data_ptr();
          any = true;
        }
      }
    }
    out[i] = like(h.norm ? xs[i] : d[i]);
    h.y = out[i].data_ptr();
    strides_of(out[i], h.y_stride);
    h.dy = d[i].const_data_ptr();
    strides_of(d[i], h.dy_stride);
    h.eps = (float)c.eps[i];
  }
  size_t bytes = 0;
  if (any && ref.size(0) * ref.size(2)) {
    bytes = harp_req_qk_backward_workspace_bytes((int)ref.size(0), (int)ref.size(2), (int)c.axes.D, normed[0], normed[1]);
    TORCH_CHECK(bytes != (size_t)-1, "harp_request.qk_norm_rope: ", harp_req_last_error());
    work = at::empty({(int64_t)(bytes / 4)}, ref.options().dtype(at::kFloat));
  }
  check_status(harp_req_qk_norm_rope_backward(&c.axes.a, &pos.p, heads, (int)ref.size(0), (int)ref.size(2),
                                              code(ref.scalar_type()), work.defined() ? work.data_ptr() : nullptr, bytes,
                                              stream_of(ref)),
               "qk_norm_rope (backward)");
  return out;
}

class QkNormRope : public torch::autograd::Function<QkNormRope> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q,
                                                const OptTensor& k, const at::Tensor& positions, const OptTensor& qw,
                                                const OptTensor& kw, RopeCall c) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [yq, yk] = rope_forward(q, k, positions, c, qw, kw);
    ctx->set_materialize_grads(false);
    const at::Tensor none;
    const OptTensor leaves[] = {q, k, qw, kw};
    for (int i = 0; i < 4; ++i) c.want[i] = given(leaves[i]) && leaves[i]->requires_grad();
    ctx->saved_data["call"] = saved(c);
    // (a rotation alone needs no input for its gradient)
    ctx->save_for_backward({c.eps[0] >= 0 ? q : none, given(k) && c.eps[1] >= 0 ? *k : none, given(qw) ? *qw : none,
                            given(kw) ? *kw : none, positions});
    if (!given(k)) return {yq};
    return {yq, yk};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const RopeCall c = restored(ctx->saved_data["call"].toStringRef());
    for (const auto& t : grads) harp_torch::refuse_tangent(t, "harp_request", "qk_norm_rope (backward)");
    torch::autograd::variable_list out(6);
    at::Tensor dy[2];
    for (size_t i = 0; i < grads.size(); ++i)
      if (c.want[i] || c.want[2 + i]) dy[i] = grads[i];
    if (dy[0].defined() || dy[1].defined()) {
      at::AutoDispatchBelowADInplaceOrView guard;
      const at::Tensor x[2] = {saved[0], saved[1]}, w[2] = {saved[2], saved[3]};
      const bool want_w[2] = {c.want[2], c.want[3]};
      auto g = rope_backward(dy, x, w, saved[4], c, want_w);
      if (c.want[0]) out[0] = g[0];
      if (c.want[1]) out[1] = g[1];
      out[3] = g[2];
      out[4] = g[3];
    }
    harp_torch::once_only(out, "qk_norm_rope");
    return out;
  }
};

void refuse_grad(const OptTensor& t, const char* op, const char* name) {
  TORCH_CHECK(!given(t) || !t->requires_grad() || !at::GradMode::is_enabled(), "harp_request.", op, ": ", name,
              " has no gradient here: pass it detached");
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope(const at::Tensor& q, const OptTensor& k, const at::Tensor& positions,
                                                at::IntArrayRef widths, at::ArrayRef<double> theta, bool half,
                                                const OptTensor& qw, const OptTensor& kw, at::ArrayRef<double> eps) {
  return rope_forward(q, k, positions, rope_call(widths, theta, half, eps), qw, kw);
}

void refuse_rope(const at::Tensor& q, const OptTensor& k, const at::Tensor& positions, const OptTensor& qw,
                 const OptTensor& kw) {
  for (const OptTensor& t : {OptTensor(q), k, OptTensor(positions), qw, kw})
    if (given(t)) harp_torch::refuse_tangent(*t, "harp_request", "qk_norm_rope");
  refuse_grad(positions, "qk_norm_rope", "positions");
}

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_autograd(const at::Tensor& q, const OptTensor& k,
                                                         const at::Tensor& positions, at::IntArrayRef widths,
                                                         at::ArrayRef<double> theta, bool half, const OptTensor& qw,
                                                         const OptTensor& kw, at::ArrayRef<double> eps) {
  refuse_rope(q, k, positions, qw, kw);
  const OptTensor leaves[] = {q, k, qw, kw};
  bool record = false;
  for (const auto& t : leaves) record |= given(t) && t->requires_grad();
  if (!record || !at::GradMode::is_enabled()) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return qk_norm_rope(q, k, positions, widths, theta, half, qw, kw, eps);
  }
  const c10::DeviceGuard guard(q.device());
  if (capturing()) {
    const char* const names[] = {"q", "k", "q_weight", "k_weight"};
    for (int i = 0; i < 4; ++i) harp_torch::check_capture(leaves[i], "qk_norm_rope", names[i]);
  }
  auto out = QkNormRope::apply(q, k, positions, qw, kw, rope_call(widths, theta, half, eps));
  return {out[0], given(k) ? out[1] : at::Tensor()};
}

at::Tensor table(const at::Tensor& positions, const Axes& ax) {
  TORCH_CHECK(positions.is_cuda(), "harp_request.rope_table: this library runs on a HIP device only");
  TORCH_CHECK(positions.dim() == 2 || positions.dim() == 3, "positions must be [S, axes] or [B, S, axes], got ",
              positions.sizes());
  const c10::DeviceGuard guard(positions.device());
  const int64_t B = positions.dim() == 3 ? positions.size(0) : 1, S = positions.size(-2);
  const Positions pos = positions_of(positions, ax.a.n, B, S);
  std::vector<int64_t> shape(positions.sizes().begin(), positions.sizes().end());
  shape.back() = ax.D / 2;
  at::Tensor out = at::empty(shape, positions.options().dtype(at::kComplexFloat));
  check_status(harp_req_rope_table(&ax.a, &pos.p, checked_int(B, "batch"), checked_int(S, "seq"),
                                   (float*)out.data_ptr(), stream_of(positions)),
               "rope_table");
  return out;
}
at::Tensor rope_table(const at::Tensor& positions, at::IntArrayRef widths, at::ArrayRef<double> theta) {
  return table(positions, axes_of(widths, theta, false));
}
at::Tensor rope_table_autograd(const at::Tensor& positions, at::IntArrayRef widths, at::ArrayRef<double> theta) {
  harp_torch::refuse_tangent(positions, "harp_request", "rope_table");
  refuse_grad(positions, "rope_table", "positions");
  at::AutoDispatchBelowADInplaceOrView guard;
  return rope_table(positions, widths, theta);
}

// ---------------------------------------------------------------------------
// adapters
// ---------------------------------------------------------------------------
// [.., C] tensors as rows; leading dimensions that are no single row stride are copied
struct Rows {
  at::Tensor t;
  const void* p = nullptr;
  int64_t ld = 0;
  int rows = 0, cols = 0;
};
Rows rows_of(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, name, " must have a last dimension of at least 1, got ", t.sizes());
  Rows r;
  r.cols = checked_int(t.size(-1), "columns");
  r.rows = checked_int(t.numel() / t.size(-1), "rows");
  r.t = plain(t);
  if (r.t.stride(-1) != 1) r.t = r.t.contiguous();
  if (r.t.dim() != 2) r.t = r.t.reshape({r.rows, r.cols});
  r.p = r.t.const_data_ptr();
  r.ld = r.rows > 1 ? r.t.stride(0) : r.cols;
  return r;
}

void check_ints(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  check_device(t, ref, name);
  TORCH_CHECK(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64, got ",
              t.scalar_type());
  TORCH_CHECK(t.dim() == 1, name, " must be a vector, got ", t.sizes());
}

struct AdapterCall {
  Rows x;
  at::Tensor a, b, scales, index, offsets;
  harp_req_adapters_t adapters{};
  harp_req_requests_t requests{};
  int N = 0;
};
AdapterCall adapter_call(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const OptTensor& scales,
                         const at::Tensor& index, const OptTensor& offsets) {
  TORCH_CHECK(x.is_cuda(), "harp_request.add_adapters: tensors must be on a HIP device");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, "x must be bfloat16, got ", x.scalar_type());
  AdapterCall c;
  c.x = rows_of(x, "x");
  for (const auto* t : {&a, &b}) {
    check_device(*t, x, t == &a ? "a" : "b");
    TORCH_CHECK(t->scalar_type() == at::kBFloat16 && t->dim() == 3, t == &a ? "a" : "b",
                " must be a bfloat16 [adapters, .., ..] tensor, got ", t->scalar_type(), " ", t->sizes());
  }
  TORCH_CHECK(a.size(2) == c.x.cols, "a must be [adapters, rank, ", c.x.cols, "], got ", a.sizes());
  TORCH_CHECK(b.size(0) == a.size(0) && b.size(2) == a.size(1), "b must be [", a.size(0), ", features, ", a.size(1),
              "], got ", b.sizes());
  TORCH_CHECK(a.size(0) >= 1 && a.size(1) >= 1 && b.size(1) >= 1, "adapters need a rank and features, got a ", a.sizes(),
              ", b ", b.sizes());
  c.a = plain(a).contiguous();
  c.b = plain(b).contiguous();
  c.N = checked_int(b.size(1), "features");
  if (given(scales)) {
    check_device(*scales, x, "scales");
    TORCH_CHECK(scales->scalar_type() == at::kFloat && scales->dim() == 1 && scales->size(0) == a.size(0),
                "scales must be float32 [", a.size(0), "], got ", scales->scalar_type(), " ", scales->sizes());
    c.scales = plain(*scales).contiguous();
  }
  check_ints(index, x, "index");
  TORCH_CHECK(index.size(0) >= 1, "index must hold an adapter for at least one request");
  c.index = index.contiguous();
  if (given(offsets)) {
    check_ints(*offsets, x, "offsets");
    TORCH_CHECK(offsets->size(0) == index.size(0) + 1, "offsets must be ", index.size(0) + 1,
                " values (one more than requests), got ", offsets->size(0));
    c.offsets = offsets->contiguous();
  } else {
    TORCH_CHECK(c.x.rows % index.size(0) == 0, c.x.rows, " tokens are not ", index.size(0),
                " requests of one length: pass their offsets");
  }
  c.adapters = harp_req_adapters_t{c.a.const_data_ptr(), c.b.const_data_ptr(),
                                   c.scales.defined() ? c.scales.const_data_ptr<float>() : nullptr,
                                   checked_int(a.size(0), "adapters"), checked_int(a.size(1), "rank")};
  c.requests = harp_req_requests_t{c.index.const_data_ptr(), int_code(index.scalar_type()),
                                   c.offsets.defined() ? c.offsets.const_data_ptr() : nullptr,
                                   c.offsets.defined() ? int_code(c.offsets.scalar_type()) : HARP_REQ_I32,
                                   checked_int(index.size(0), "requests")};
  return c;
}

// (out, t)
std::tuple<at::Tensor, at::Tensor> adapters_forward(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a,
                                                    const at::Tensor& b, const OptTensor& scales,
                                                    const at::Tensor& index, const OptTensor& offsets) {
  const AdapterCall c = adapter_call(x, a, b, scales, index, offsets);
  check_device(base, x, "base");
  TORCH_CHECK(base.scalar_type() == at::kBFloat16 || base.scalar_type() == at::kFloat,
              "base must be bfloat16 or float32, got ", base.scalar_type());
  TORCH_CHECK(base.dim() == x.dim() && base.size(-1) == c.N && base.sizes().slice(0, base.dim() - 1) ==
                                                                   x.sizes().slice(0, x.dim() - 1),
              "base must be x's shape with ", c.N, " features, got ", base.sizes(), " for x ", x.sizes());
  const c10::DeviceGuard guard(x.device());
  at::Tensor out = at::empty(base.sizes(), base.options()), t;
  const int cols = harp_req_adapter_columns(c.adapters.rank);
  TORCH_CHECK(cols > 0, "harp_request.add_adapters: ", harp_req_last_error());
  t = at::empty({c.x.rows, cols}, x.options().dtype(at::kFloat));
  if (c.x.rows) {
    const Rows br = rows_of(base, "base");
    check_status(harp_req_add_adapters_forward(c.x.p, c.x.ld, br.p, br.ld, out.data_ptr(), c.N,
                                               code(base.scalar_type()), &c.adapters, &c.requests, t.data_ptr<float>(),
                                               c.x.rows, c.x.cols, c.N, stream_of(x)),
                 "add_adapters");
  }
  return {out, t};
}

// gradients of (x, a, b), undefined where not wanted
std::tuple<at::Tensor, at::Tensor, at::Tensor> adapters_backward(const at::Tensor& dy, const at::Tensor& x,
                                                                 const at::Tensor& a, const at::Tensor& b,
                                                                 const OptTensor& scales, const at::Tensor& index,
                                                                 const OptTensor& offsets, const at::Tensor& t,
                                                                 bool want_x, bool want_a, bool want_b) {
  const AdapterCall c = adapter_call(x, a, b, scales, index, offsets);
  const c10::DeviceGuard guard(x.device());
  at::Tensor dx, da, db, work;
  const bool none = c.x.rows == 0;
  if (want_x) dx = at::empty(x.sizes(), x.options());
  if (want_a) da = none ? at::zeros(a.sizes(), a.options()) : at::empty(a.sizes(), a.options());
  if (want_b) db = none ? at::zeros(b.sizes(), b.options()) : at::empty(b.sizes(), b.options());
  if (none) return {dx, da, db};
  const Rows d = rows_of(dy, "dy");
  const size_t bytes = harp_req_adapter_backward_workspace_bytes(c.x.rows, c.x.cols, c.N, c.adapters.n, c.adapters.rank,
                                                                 c.requests.count, 1);
  TORCH_CHECK(bytes != (size_t)-1, "harp_request.add_adapters: ", harp_req_last_error());
  work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
  const harp_req_backward_set_t set{c.adapters, t.const_data_ptr<float>(), d.p, d.ld, want_a ? da.data_ptr() : nullptr,
                                    want_b ? db.data_ptr() : nullptr};
  check_status(harp_req_add_adapters_backward(&set, 1, c.x.p, c.x.ld, &c.requests, nullptr, 0,
                                              want_x ? dx.data_ptr() : nullptr, c.x.cols, c.x.rows, c.x.cols, c.N,
                                              work.data_ptr(), bytes, stream_of(x)),
               "add_adapters (backward)");
  return {dx, da, db};
}

class AddAdapters : public torch::autograd::Function<AddAdapters> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& base, const at::Tensor& x,
                            const at::Tensor& a, const at::Tensor& b, const OptTensor& scales, const at::Tensor& index,
                            const OptTensor& offsets) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [out, t] = adapters_forward(base, x, a, b, scales, index, offsets);
    ctx->saved_data["wanted"] = (int64_t)(base.requires_grad() + 2 * x.requires_grad() + 4 * a.requires_grad() +
                                          8 * b.requires_grad());
    const at::Tensor none;
    ctx->save_for_backward({x, a, b, given(scales) ? *scales : none, index, given(offsets) ? *offsets : none, t});
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t wanted = ctx->saved_data["wanted"].toInt();
    const at::Tensor& dy = grads[0];
    harp_torch::refuse_tangent(dy, "harp_request", "add_adapters (backward)");
    torch::autograd::variable_list out(7);
    if (dy.defined()) {
      at::AutoDispatchBelowADInplaceOrView guard;
      if (wanted & 1) out[0] = dy;
      if (wanted & ~1) {
        auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        auto [dx, da, db] = adapters_backward(dy, s[0], s[1], s[2], opt(s[3]), s[4], opt(s[5]), s[6], wanted & 2,
                                              wanted & 4, wanted & 8);
        out[1] = dx;
        out[2] = da;
        out[3] = db;
      }
    }
    harp_torch::once_only(out, "add_adapters");
    return out;
  }
};

at::Tensor add_adapters(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                        const OptTensor& scales, const at::Tensor& index, const OptTensor& offsets) {
  return std::get<0>(adapters_forward(base, x, a, b, scales, index, offsets));
}

void refuse_adapters(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                     const OptTensor& scales) {
  for (const OptTensor& t : {OptTensor(base), OptTensor(x), OptTensor(a), OptTensor(b), scales})
    if (given(t)) harp_torch::refuse_tangent(*t, "harp_request", "add_adapters");
  refuse_grad(scales, "add_adapters", "scales");
}

at::Tensor add_adapters_autograd(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a, const at::Tensor& b,
                                 const OptTensor& scales, const at::Tensor& index, const OptTensor& offsets) {
  refuse_adapters(base, x, a, b, scales);
  const at::Tensor* const leaves[] = {&base, &x, &a, &b};
  bool record = false;
  for (const auto* t : leaves) record |= t->requires_grad();
  if (!record || !at::GradMode::is_enabled()) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return add_adapters(base, x, a, b, scales, index, offsets);
  }
  TORCH_CHECK(base.scalar_type() == at::kBFloat16, "harp_request.add_adapters: gradients need a bfloat16 base, got ",
              base.scalar_type());
  const c10::DeviceGuard guard(x.device());
  if (capturing()) {
    const char* const names[] = {"base", "x", "a", "b"};
    for (int i = 0; i < 4; ++i) harp_torch::check_capture(*leaves[i], "add_adapters", names[i]);
  }
  return AddAdapters::apply(base, x, a, b, scales, index, offsets);
}

// ---------------------------------------------------------------------------
// the q/k/v producer with adapters
// ---------------------------------------------------------------------------
constexpr int64_t kHeadDim = 128;

using Tensors = std::vector<at::Tensor>;

// The rotation of q and k: by a table (complex64 [S, 64] or [B or 1, S, 64]), or by
// positions along axes of interleaved pairs, or none
struct QkvCall {
  AdapterCall first;           // x, requests, adapters[0]
  harp_req_adapters_t adapters[3];
  Tensors a, b, scales;        // kept alive
  at::Tensor freqs;            // fp32 (cos, sin) rows, written by the call where it has positions
  int64_t fsb = 0;
  bool axial = false;
  Axes axes;
  Positions pos;
  Tensors w, nw;               // projections, norm weights (undefined: none)
  int64_t B = 0, S = 0, K = 0, N = 0, H = 0;
};
QkvCall qkv_call(const at::Tensor& x, const Tensors& weights, const Tensors& a, const Tensors& b,
                 const c10::List<OptTensor>& scales, const at::Tensor& index, const OptTensor& offsets,
                 const c10::List<OptTensor>& norm_weights, const OptTensor& freqs) {
  TORCH_CHECK(x.dim() == 3, "x must be [B, S, dim], got ", x.sizes());
  TORCH_CHECK(weights.size() == 3 && a.size() == 3 && b.size() == 3 && scales.size() == 3 && norm_weights.size() == 2,
              "three weights with an adapter stack each, and two norm weights (or None)");
  QkvCall c;
  c.B = x.size(0);
  c.S = x.size(1);
  c.K = x.size(2);
  c.N = weights[0].size(0);
  c.H = c.N / kHeadDim;
  TORCH_CHECK(c.N >= kHeadDim && c.N % kHeadDim == 0, "weights must have heads of 128 features, got ", c.N, " rows");
  const at::Tensor xc = plain(x).contiguous();  // (its rows are read 16 bytes at a time)
  c.first = adapter_call(xc, a[0], b[0], scales.get(0), index, offsets);
  for (int i = 0; i < 3; ++i) {
    TORCH_CHECK(a[i].sizes() == a[0].sizes() && b[i].sizes() == b[0].sizes(),
                "adapters of q, k and v must have one number and one rank, got a ", a[0].sizes(), " and ", a[i].sizes());
    const AdapterCall one = i ? adapter_call(xc, a[i], b[i], scales.get(i), index, offsets) : c.first;
    TORCH_CHECK(one.N == c.N, "b must be [", a[0].size(0), ", ", c.N, ", ", a[0].size(1), "], got ", b[i].sizes());
    c.adapters[i] = one.adapters;
    c.a.push_back(one.a);
    c.b.push_back(one.b);
    c.scales.push_back(one.scales);
    check_device(weights[i], x, "weight");
    TORCH_CHECK(weights[i].scalar_type() == at::kBFloat16 && weights[i].dim() == 2 && weights[i].size(0) == c.N &&
                    weights[i].size(1) == c.K && weights[i].stride(1) == 1,
                "every weight must be a bfloat16 [", c.N, ", ", c.K, "] tensor with unit column stride, got ",
                weights[i].scalar_type(), " ", weights[i].sizes());
    c.w.push_back(plain(weights[i]));
    at::Tensor nw;
    const OptTensor n = i < 2 ? norm_weights.get(i) : OptTensor();
    if (given(n)) {
      check_device(*n, x, "norm weight");
      TORCH_CHECK((n->scalar_type() == at::kBFloat16 || n->scalar_type() == at::kFloat) && n->dim() == 1 &&
                      n->size(0) == kHeadDim,
                  "norm weights must be bfloat16 or float32 [128], got ", n->scalar_type(), " ", n->sizes());
      nw = plain(*n).contiguous();
    }
    c.nw.push_back(nw);
  }
  if (given(freqs)) {
    check_device(*freqs, x, "freqs_cis");
    TORCH_CHECK(freqs->scalar_type() == at::kComplexFloat && (freqs->dim() == 2 || freqs->dim() == 3) &&
                    freqs->size(-1) == kHeadDim / 2 && freqs->size(-2) == c.S &&
                    (freqs->dim() == 2 || freqs->size(0) == 1 || freqs->size(0) == c.B),
                "freqs_cis must be complex64 [S, 64] or [B, S, 64] with S=", c.S, ", got ", freqs->sizes());
    c.freqs = at::view_as_real(freqs->resolve_conj()).contiguous();
    c.fsb = freqs->dim() == 3 && freqs->size(0) > 1 ? c.freqs.stride(0) : 0;
  }
  return c;
}

struct QkvResult {
  Tensors y;     // q, k, v [B, H, S, 128], token-major
  Tensors lin;   // of q and k before the norm [B, S, N], with keep
  Tensors t;     // x A^T of the three, with keep
};
QkvResult qkv_forward(const QkvCall& c, const at::Tensor& x, const double (&eps)[2], bool keep) {
  const c10::DeviceGuard guard(x.device());
  QkvResult r;
  harp_qkv_out_t outs[3] = {};
  float* t[3] = {};
  for (int i = 0; i < 3; ++i) {
    r.y.push_back(at::empty({c.B, c.S, c.N}, x.options()));
    harp_qkv_out_t& o = outs[i];
    o.weight = c.w[i].const_data_ptr();
    o.ld_weight = c.w[i].stride(0);
    o.y = r.y[i].data_ptr();
    o.ld_y = c.N;
    if (c.nw[i].defined()) {
      o.norm_weight = c.nw[i].const_data_ptr();
      o.norm_weight_dtype = c.nw[i].scalar_type() == at::kFloat ? HARP_QK_F32 : HARP_QK_BF16;
      o.eps = (float)eps[i];
      if (keep) {
        r.lin.push_back(at::empty({c.B, c.S, c.N}, x.options()));
        o.y_lin = r.lin.back().data_ptr();
      }
    } else {
      TORCH_CHECK(!c.freqs.defined() || i == 2, "a rotation without its RMSNorm is the separate operator's");
    }
    if (keep) {
      r.t.push_back(at::empty({c.B * c.S, harp_req_adapter_columns(c.adapters[0].rank)}, x.options().dtype(at::kFloat)));
      t[i] = r.t[i].data_ptr<float>();
    }
  }
  if (c.B * c.S) {
    const size_t bytes = harp_req_qkv_workspace_bytes(c.first.x.rows, c.adapters[0].rank, 3);
    TORCH_CHECK(bytes != (size_t)-1, "harp_request.qkv_adapters: ", harp_req_last_error());
    const at::Tensor work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check_status(
        harp_req_qkv_project(c.first.x.p, c.first.x.ld, checked_int(c.B, "batch"), checked_int(c.S, "seq"),
                             checked_int(c.K, "dim"), checked_int(c.N, "features"),
                             c.freqs.defined() && !c.axial ? c.freqs.const_data_ptr<float>() : nullptr, c.fsb,
                             kHeadDim, c.axial ? &c.axes.a : nullptr, c.axial ? &c.pos.p : nullptr,
                             c.axial ? c.freqs.data_ptr<float>() : nullptr, outs,
                             c.adapters, 3, &c.first.requests, keep ? t : nullptr, work.data_ptr(), bytes, stream_of(x)),
        "qkv_adapters");
  }
  for (auto& y : r.y) y = y.unflatten(-1, {c.H, kHeadDim}).transpose(1, 2);
  return r;
}

// the rotation by positions, whose table the call writes
void set_positions(QkvCall& c, const at::Tensor& positions, const RopeCall& rope, const at::Tensor& x) {
  check_device(positions, x, "positions");
  TORCH_CHECK(rope.axes.D == kHeadDim, "the axes' widths must add up to 128, got ", rope.axes.D);
  c.axial = true;
  c.axes = rope.axes;
  c.pos = positions_of(positions, c.axes.a.n, c.B, c.S);
  const c10::DeviceGuard guard(x.device());
  c.freqs = at::empty({c.pos.p.stride_b ? c.B : 1, c.S, kHeadDim / 2, 2}, x.options().dtype(at::kFloat));
}

Tensors qkv_adapters(const at::Tensor& x, const Tensors& weights, const Tensors& a, const Tensors& b,
                     const c10::List<OptTensor>& scales, const at::Tensor& index, const OptTensor& offsets,
                     const c10::List<OptTensor>& norm_weights, const std::vector<double>& eps, const OptTensor& freqs,
                     const OptTensor& positions, const std::vector<int64_t>& widths, const std::vector<double>& theta) {
  TORCH_CHECK(x.is_cuda(), "harp_request.qkv_adapters: tensors must be on a HIP device");
  TORCH_CHECK(!given(freqs) || !given(positions), "one rotation: freqs_cis or positions");
  TORCH_CHECK(eps.size() == 2, "eps must be two values, got ", eps.size());
  const double both[2] = {eps[0], eps[1]};
  QkvCall c = qkv_call(x, weights, a, b, scales, index, offsets, norm_weights, freqs);
  if (given(positions)) set_positions(c, *positions, rope_call(widths, theta, false, eps), x);
  return qkv_forward(c, x, both, false).y;
}

// Differentiable arguments in this order: x, three weights, two norm weights, three a, three b
class QkvAdapters : public torch::autograd::Function<QkvAdapters> {
 public:
  static constexpr int kLeaves = 12;

  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x,
                                                const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& wv,
                                                const at::Tensor& nq, const at::Tensor& nk, const at::Tensor& aq,
                                                const at::Tensor& ak, const at::Tensor& av, const at::Tensor& bq,
                                                const at::Tensor& bk, const at::Tensor& bv,
                                                c10::List<OptTensor> scales, const at::Tensor& index,
                                                const OptTensor& offsets, const at::Tensor& positions, RopeCall call) {
    at::AutoDispatchBelowADInplaceOrView guard;
    c10::List<OptTensor> norms;
    norms.push_back(nq);
    norms.push_back(nk);
    QkvCall c = qkv_call(x, {wq, wk, wv}, {aq, ak, av}, {bq, bk, bv}, scales, index, offsets, norms, OptTensor());
    set_positions(c, positions, call, x);
    const QkvResult r = qkv_forward(c, x, call.eps, true);
    int64_t wanted = 0;
    const at::Tensor* const leaves[] = {&x, &wq, &wk, &wv, &nq, &nk, &aq, &ak, &av, &bq, &bk, &bv};
    for (int i = 0; i < kLeaves; ++i) wanted |= (int64_t)leaves[i]->requires_grad() << i;
    ctx->saved_data["wanted"] = wanted;
    ctx->saved_data["call"] = saved(call);
    auto or_none = [](const OptTensor& t) { return given(t) ? *t : at::Tensor(); };
    ctx->save_for_backward({x, wq, wk, wv, nq, nk, aq, ak, av, bq, bk, bv, or_none(scales.get(0)),
                            or_none(scales.get(1)), or_none(scales.get(2)), index, or_none(offsets), positions,
                            r.lin[0], r.lin[1], r.t[0], r.t[1], r.t[2]});
    return {r.y[0], r.y[1], r.y[2]};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const int64_t wanted = ctx->saved_data["wanted"].toInt();
    auto want = [&](int i) { return (wanted >> i & 1) != 0; };
    for (const auto& t : grads) harp_torch::refuse_tangent(t, "harp_request", "qkv_adapters (backward)");
    torch::autograd::variable_list out(17);
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      const at::Tensor &x = s[0], &index = s[15];
      const c10::DeviceGuard device(x.device());
      const int64_t B = x.size(0), S = x.size(1), K = x.size(2), N = s[1].size(0), H = N / kHeadDim, M = B * S;
      // Through the rotation and the norm: the gradients of the three products [M, N].  q and k in front of the norm
      // were kept in bf16, and these gradients are rounded to it: the library's products and the adapters' kernels read
      // bf16, as two bf16 each they would double the products' operations (3 x 37 us at 768 tokens x 30 heads), and the
      // plain producer's backward rounds there too.  What it costs: 0.0024 of the norm against 64 bits, 0.0017 of it
      // the results' own rounding.
      const RopeCall rope = restored(ctx->saved_data["call"].toStringRef());
      auto heads = [&](const at::Tensor& t) { return t.unflatten(-1, {H, kHeadDim}).transpose(1, 2); };
      const at::Tensor d[2] = {grads[0], grads[1]}, lin[2] = {heads(s[18]), heads(s[19])}, nw[2] = {s[4], s[5]};
      const bool want_nw[2] = {want(4), want(5)};
      auto g = rope_backward(d, lin, nw, s[17], rope, want_nw);
      out[4] = g[2];
      out[5] = g[3];
      auto rows = [&](const at::Tensor& t) { return t.transpose(1, 2).reshape({M, N}); };
      const at::Tensor gy[3] = {rows(g[0]), rows(g[1]), rows(plain(grads[2]))};
      const at::Tensor x2 = plain(x).reshape({M, K});
      for (int i = 0; i < 3; ++i)
        if (want(1 + i)) out[1 + i] = at::mm(gy[i].t(), x2);
      bool low = want(0);
      for (int i = 6; i < kLeaves; ++i) low |= want(i);
      if (low) {
        harp_req_backward_set_t sets[3];
        std::vector<AdapterCall> calls;
        std::vector<Rows> dys;
        for (int i = 0; i < 3; ++i) {
          const at::Tensor &a = s[6 + i], &b = s[9 + i];
          calls.push_back(adapter_call(x, a, b, s[12 + i].defined() ? OptTensor(s[12 + i]) : OptTensor(), index,
                                       s[16].defined() ? OptTensor(s[16]) : OptTensor()));
          dys.push_back(rows_of(gy[i], "dy"));
          // (without a token the sums are empty)
          if (want(6 + i)) out[6 + i] = M ? at::empty(a.sizes(), a.options()) : at::zeros(a.sizes(), a.options());
          if (want(9 + i)) out[9 + i] = M ? at::empty(b.sizes(), b.options()) : at::zeros(b.sizes(), b.options());
          sets[i] = {calls[i].adapters,
                     s[20 + i].const_data_ptr<float>(),
                     dys[i].p,
                     dys[i].ld,
                     want(6 + i) ? out[6 + i].data_ptr() : nullptr,
                     want(9 + i) ? out[9 + i].data_ptr() : nullptr};
        }
        at::Tensor dx, base;
        if (want(0)) {
          // the projections' part, added up in 32 bits; the adapters' kernel adds its own and rounds
          dx = at::empty({B, S, K}, x.options());
          if (M) {
            base = at::mm(gy[0], s[1], at::kFloat);
            for (int i = 1; i < 3; ++i) at::addmm_out(base, base, gy[i], s[1 + i], at::kFloat);
          }
        }
        if (M) {
          const size_t bytes = harp_req_adapter_backward_workspace_bytes(
              (int)M, (int)K, (int)N, calls[0].adapters.n, calls[0].adapters.rank, calls[0].requests.count, 3);
          TORCH_CHECK(bytes != (size_t)-1, "harp_request.qkv_adapters: ", harp_req_last_error());
          const at::Tensor work = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
          check_status(harp_req_add_adapters_backward(sets, 3, calls[0].x.p, calls[0].x.ld, &calls[0].requests,
                                                      base.defined() ? base.data_ptr<float>() : nullptr, K,
                                                      dx.defined() ? dx.data_ptr() : nullptr, K, (int)M, (int)K, (int)N,
                                                      work.data_ptr(), bytes, stream_of(x)),
                       "qkv_adapters (backward)");
        }
        out[0] = dx;
      }
    }
    harp_torch::once_only(out, "qkv_adapters");
    return out;
  }
};

Tensors qkv_adapters_autograd(const at::Tensor& x, const Tensors& weights, const Tensors& a, const Tensors& b,
                              const c10::List<OptTensor>& scales, const at::Tensor& index, const OptTensor& offsets,
                              const c10::List<OptTensor>& norm_weights, const std::vector<double>& eps,
                              const OptTensor& freqs, const OptTensor& positions, const std::vector<int64_t>& widths,
                              const std::vector<double>& theta) {
  Tensors leaves = {x};
  leaves.insert(leaves.end(), weights.begin(), weights.end());
  for (size_t i = 0; i < norm_weights.size(); ++i) leaves.push_back(given(norm_weights.get(i)) ? *norm_weights.get(i) : at::Tensor());
  leaves.insert(leaves.end(), a.begin(), a.end());
  leaves.insert(leaves.end(), b.begin(), b.end());
  for (const auto& t : leaves) harp_torch::refuse_tangent(t, "harp_request", "qkv_adapters");
  for (size_t i = 0; i < scales.size(); ++i) {
    if (given(scales.get(i))) harp_torch::refuse_tangent(*scales.get(i), "harp_request", "qkv_adapters");
    refuse_grad(scales.get(i), "qkv_adapters", "scales");
  }
  for (const OptTensor& t : {freqs, positions}) {
    if (given(t)) harp_torch::refuse_tangent(*t, "harp_request", "qkv_adapters");
    refuse_grad(t, "qkv_adapters", "the rotation");
  }
  bool record = false;
  for (const auto& t : leaves) record |= t.defined() && t.requires_grad();
  if (!record || !at::GradMode::is_enabled()) {
    static const auto op = c10::Dispatcher::singleton()
                               .findSchemaOrThrow("harp_request::qkv_adapters", "")
                               .typed<decltype(qkv_adapters)>();
    at::AutoDispatchBelowADInplaceOrView guard;
    return op.call(x, weights, a, b, scales, index, offsets, norm_weights, eps, freqs, positions, widths, theta);
  }
  TORCH_CHECK(x.is_cuda(), "harp_request.qkv_adapters: this library runs on a HIP device only (CPU tensors given)");
  TORCH_CHECK(leaves.size() == QkvAdapters::kLeaves && given(positions) && leaves[4].defined() && leaves[5].defined(),
              "harp_request.qkv_adapters: gradients need both norm weights, and the rotation as positions");
  const c10::DeviceGuard guard(x.device());
  if (capturing()) {
    for (const auto& t : leaves) harp_torch::check_capture(t, "qkv_adapters", "an argument");
  }
  const Tensors& l = leaves;
  return QkvAdapters::apply(l[0], l[1], l[2], l[3], l[4], l[5], l[6], l[7], l[8], l[9], l[10], l[11], scales, index,
                            offsets, *positions, rope_call(widths, theta, false, eps));
}

[[noreturn]] void no_cpu(const char* op) {
  TORCH_CHECK(false, "harp_request.", op, ": this library runs on a HIP device only (CPU tensors given)");
}
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_cpu(const at::Tensor&, const OptTensor&, const at::Tensor&,
                                                    at::IntArrayRef, at::ArrayRef<double>, bool, const OptTensor&,
                                                    const OptTensor&, at::ArrayRef<double>) {
  no_cpu("qk_norm_rope");
}
at::Tensor rope_table_cpu(const at::Tensor&, at::IntArrayRef, at::ArrayRef<double>) { no_cpu("rope_table"); }
at::Tensor add_adapters_cpu(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                            const OptTensor&, const at::Tensor&, const OptTensor&) {
  no_cpu("add_adapters");
}
Tensors qkv_adapters_cpu(const at::Tensor&, const Tensors&, const Tensors&, const Tensors&, const c10::List<OptTensor>&,
                         const at::Tensor&, const OptTensor&, const c10::List<OptTensor>&, const std::vector<double>&,
                         const OptTensor&, const OptTensor&, const std::vector<int64_t>&, const std::vector<double>&) {
  no_cpu("qkv_adapters");
}
std::tuple<at::Tensor, at::Tensor> qk_norm_rope_autograd_cpu(const at::Tensor& q, const OptTensor& k,
                                                             const at::Tensor& positions, at::IntArrayRef,
                                                             at::ArrayRef<double>, bool, const OptTensor& qw,
                                                             const OptTensor& kw, at::ArrayRef<double>) {
  refuse_rope(q, k, positions, qw, kw);
  no_cpu("qk_norm_rope");
}
at::Tensor add_adapters_autograd_cpu(const at::Tensor& base, const at::Tensor& x, const at::Tensor& a,
                                     const at::Tensor& b, const OptTensor& scales, const at::Tensor&,
                                     const OptTensor&) {
  refuse_adapters(base, x, a, b, scales);
  no_cpu("add_adapters");
}

}  // namespace

TORCH_LIBRARY(harp_request, m) {
  m.def(
      "qk_norm_rope(Tensor q, Tensor? k, Tensor positions, int[] widths, float[] theta, bool half, Tensor? q_weight, "
      "Tensor? k_weight, float[] eps) -> (Tensor, Tensor)");
  m.def("rope_table(Tensor positions, int[] widths, float[] theta) -> Tensor");
  m.def(
      "add_adapters(Tensor base, Tensor x, Tensor a, Tensor b, Tensor? scales, Tensor index, Tensor? offsets) -> "
      "Tensor");
  m.def(
      "qkv_adapters(Tensor x, Tensor[] weights, Tensor[] a, Tensor[] b, Tensor?[] scales, Tensor index, Tensor? "
      "offsets, Tensor?[] norm_weights, float[] eps, Tensor? freqs_cis, Tensor? positions, int[] widths, float[] "
      "theta) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(harp_request, AutogradCUDA, m) {
  m.impl("qk_norm_rope", &qk_norm_rope_autograd);
  m.impl("rope_table", &rope_table_autograd);
  m.impl("add_adapters", &add_adapters_autograd);
  m.impl("qkv_adapters", &qkv_adapters_autograd);
}

TORCH_LIBRARY_IMPL(harp_request, AutogradCPU, m) {
  m.impl("qk_norm_rope", &qk_norm_rope_autograd_cpu);
  m.impl("rope_table", &rope_table_autograd);
  m.impl("add_adapters", &add_adapters_autograd_cpu);
  m.impl("qkv_adapters", &qkv_adapters_autograd);
}

TORCH_LIBRARY_IMPL(harp_request, CUDA, m) {
  m.impl("qk_norm_rope", &qk_norm_rope);
  m.impl("rope_table", &rope_table);
  m.impl("add_adapters", &add_adapters);
  m.impl("qkv_adapters", &qkv_adapters);
}

TORCH_LIBRARY_IMPL(harp_request, CPU, m) {
  m.impl("qk_norm_rope", &qk_norm_rope_cpu);
  m.impl("rope_table", &rope_table_cpu);
  m.impl("add_adapters", &add_adapters_cpu);
  m.impl("qkv_adapters", &qkv_adapters_cpu);
}
