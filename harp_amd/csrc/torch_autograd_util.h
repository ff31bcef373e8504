// What the operator libraries' autograd kernels share: refusals of derivatives
// that do not exist, and of captured backward passes that would end the process.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include <memory>
#include <string>
#include <utility>

namespace harp_torch {

using OptTensor = std::optional<at::Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

// A forward-mode tangent would be lost below the autograd keys.
inline void refuse_tangent(const at::Tensor& t, const char* library, const char* op) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), library, ".", op,
              " has no forward-mode derivative: an argument carries a tangent");
}

// While a graph of an earlier call is alive, a leaf keeps the accumulator node
// of that graph, with the stream it was made on.  A backward captured on
// another stream would have the engine wait across the two streams inside the
// capture, which ends the process: such a call is refused while it can be.  (The
// current stream is asked for as the node did when it was made.)
inline void check_capture(const OptTensor& t, const char* op, const char* name) {
  if (!given(t) || !t->requires_grad() || t->grad_fn()) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
  if (!node) return;
  const auto made_on = node->stream();
  const c10::Stream current = c10::impl::VirtualGuardImpl(t->device().type()).getStream(t->device());
  TORCH_CHECK(!made_on || *made_on == current, op, ": ", name,
              " belongs to a live autograd graph of another stream, so its gradient cannot be captured: delete that "
              "graph's tensors (an earlier step's outputs or loss) before the capture");
}

// Gradients under create_graph: a gradient of these raises.
inline void once_only(torch::autograd::variable_list& out, const char* op) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::variable_list given_out;
  for (auto& t : out)
    if (t.defined()) given_out.push_back(t.detach().requires_grad_());
  if (given_out.empty()) return;
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(op) + " is differentiable once only",
                                                              given_out.size());
  given_out = (*error)(std::move(given_out));
  size_t i = 0;
  for (auto& t : out)
    if (t.defined()) t = given_out[i++];
}

}  // namespace harp_torch
