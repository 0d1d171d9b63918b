// For operators that are autograd nodes in C++.
#pragma once
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace dca {

// The persistent gradient a kernel may add to for parameter `p` (ops/_grad.py target()), or nothing.
// Asked at backward time, since engines install gradients shortly before; a parameter without a
// gradient has none, which spares the call.
inline c10::optional<torch::Tensor> grad_target(const torch::Tensor& p) {
  if (!p.is_leaf() || !p.grad().defined()) return c10::nullopt;
  pybind11::gil_scoped_acquire gil;
  pybind11::object t = pybind11::module_::import("determined_clone_amd.ops._grad").attr("target")(p);
  if (t.is_none()) return c10::nullopt;
  return t.cast<torch::Tensor>();
}

// `out`, gradients that cannot be differentiated again: under create_graph doing so raises. `depends`:
// whether they depend on anything that could ask for it (an incoming gradient, saved inputs).
inline torch::autograd::variable_list once(torch::autograd::variable_list&& out, bool depends) {
  if (!at::GradMode::is_enabled() || !depends) return std::move(out);
  for (auto& g : out)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function whose backward is a kernel", static_cast<int64_t>(out.size()));
  return (*node)(std::move(out));
}
}  // namespace dca
