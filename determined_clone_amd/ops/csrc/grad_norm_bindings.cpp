// Bindings for the multi-tensor gradient norm / clipping kernels (grad_norm.hip).
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>

#include "grad_norm_api.h"

namespace {
using torch::Tensor;

hipStream_t stream() { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }

// Tensor subclasses, which may have no memory of their own.
bool wrapped(const Tensor& g) { return g.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python); }

// Whether two of the tensors share memory (each taken from its first to its last element).
bool overlaps(const std::vector<Tensor>& grads) {
  std::vector<std::pair<const char*, const char*>> spans;
  spans.reserve(grads.size());
  for (const Tensor& g : grads) {
    if (!g.defined() || g.is_nested() || g.layout() != at::kStrided || wrapped(g) || !g.numel()) continue;
    int64_t last = 0;
    for (int64_t d = 0; d < g.dim(); ++d) last += (g.size(d) - 1) * g.stride(d);
    const char* p = static_cast<const char*>(g.data_ptr());
    spans.emplace_back(p, p + (last + 1) * static_cast<int64_t>(g.element_size()));
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return true;
  return false;
}

// The list as the kernels take it; false where they do not apply: another device or dtype among
// them, tensors that are not dense or (to be written) that share memory.
bool describe(const std::vector<Tensor>& grads, bool write, std::vector<dca::GradTensor>& out) {
  out.reserve(grads.size());
  for (const Tensor& g : grads) {
    if (!g.defined() || g.is_nested() || g.layout() != at::kStrided || !g.is_cuda() || g.device() != grads[0].device() ||
        g.is_conj() || g.is_neg() || wrapped(g))
      return false;
    dca::TDtype dt;
    switch (g.scalar_type()) {
      case at::kBFloat16: dt = dca::TDtype::kBF16; break;
      case at::kHalf: dt = dca::TDtype::kF16; break;
      case at::kFloat: dt = dca::TDtype::kF32; break;
      default: return false;
    }
    if (!g.is_non_overlapping_and_dense()) return false;
    out.push_back({g.data_ptr(), g.numel(), dt});
  }
  return !write || !overlaps(grads);
}

// Scales the tensors; autograd hears of it, as of any change in place.
void clip(const std::vector<Tensor>& grads, const std::vector<dca::GradTensor>& t, const Tensor& norm, double max_norm) {
  dca::grad_clip(t, norm.data_ptr<float>(), static_cast<float>(max_norm), stream());
  for (const Tensor& g : grads)
    if (!g.is_inference()) g.unsafeGetTensorImpl()->bump_version();
}

// kind: 0 L2, 1 L1, 2 max. -> the fp32 norm, or None where the kernels do not apply. With max_norm
// the tensors are also scaled by min(1, max_norm / (norm + 1e-6)).
c10::optional<Tensor> grad_list_norm(const std::vector<Tensor>& grads, int64_t kind, c10::optional<double> max_norm) {
  TORCH_CHECK(!grads.empty() && kind >= 0 && kind <= 2, "grad_list_norm: a list and a known norm are required");
  std::vector<dca::GradTensor> t;
  if (!describe(grads, max_norm.has_value(), t)) return c10::nullopt;
  const c10::DeviceGuard g(grads[0].device());
  Tensor ws = torch::empty({dca::grad_norm_workspace(t)}, grads[0].options().dtype(at::kDouble));
  Tensor norm = torch::empty({}, grads[0].options().dtype(at::kFloat));
  dca::grad_norm(t, static_cast<dca::NormKind>(kind), ws.data_ptr<double>(), norm.data_ptr<float>(), stream());
  if (max_norm.has_value()) clip(grads, t, norm, *max_norm);
  return norm;
}

// Scales the tensors by a norm that is there; None (nothing done) where the kernels do not apply.
c10::optional<Tensor> grad_list_clip(const std::vector<Tensor>& grads, const Tensor& norm, double max_norm) {
  std::vector<dca::GradTensor> t;
  if (grads.empty() || !describe(grads, true, t)) return c10::nullopt;
  TORCH_CHECK(norm.scalar_type() == at::kFloat && norm.numel() == 1 && norm.device() == grads[0].device(),
              "grad_list_clip: the norm must be one fp32 value on the gradients' device");
  const c10::DeviceGuard g(grads[0].device());
  clip(grads, t, norm, max_norm);
  return norm;
}
}  // namespace

void register_grad_norm_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("grad_list_norm", &grad_list_norm, py::arg("grads"), py::arg("kind"), py::arg("max_norm") = py::none());
  m.def("grad_list_overlaps", &overlaps, py::arg("grads"));
  m.def("grad_list_clip", &grad_list_clip, py::arg("grads"), py::arg("norm"), py::arg("max_norm"));
}
