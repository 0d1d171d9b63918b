// Bindings for the query / key norm + rotary kernels (qk_norm.hip).
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include "autograd_util.h"
#include "qk_norm_api.h"

namespace {
using torch::Tensor;
using OptT = c10::optional<Tensor>;

hipStream_t stream() { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
bool given(const OptT& t) { return t.has_value() && t->defined(); }

dca::TDtype tdt(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return dca::TDtype::kBF16;
    case at::kHalf: return dca::TDtype::kF16;
    case at::kFloat: return dca::TDtype::kF32;
    default: TORCH_CHECK(false, "qk_norm_rope: unsupported dtype ", t.scalar_type());
  }
}

// The arguments that forward and backward share, checked.
struct Call {
  dca::QkShape s;
  const float* w[2] = {nullptr, nullptr};
  const float* cosT = nullptr;
  const float* sinT = nullptr;
  dca::WidestVec vec{1};
  Tensor like;

  dca::HeadView view(const Tensor& t, int which) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device() && t.scalar_type() == like.scalar_type() &&
                    t.dim() == 4 && t.size(0) == s.B && t.size(1) == s.S && t.size(2) == s.heads[which] &&
                    t.size(3) == s.D && (s.D <= 1 || t.stride(3) == 1 || t.numel() == 0),
                "qk_norm_rope: [B, S, heads, D] tensors of one dtype and device with contiguous rows are required");
    vec.elems(t.stride(0));
    vec.elems(t.stride(1));
    vec.elems(t.stride(2));
    vec.ptr(t.data_ptr());
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
  }

  Call(const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk, const OptT& cos, const OptT& sin,
       int64_t rot, const OptT& positions, double eps)
      : vec(static_cast<int>(q.element_size())), like(q) {
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "qk_norm_rope: q and k must be [B, S, heads, D]");
    s.B = q.size(0);
    s.S = q.size(1);
    TORCH_CHECK(q.size(3) >= 1 && q.size(3) <= 1024, "qk_norm_rope: head dim must be 1 .. 1024");
    TORCH_CHECK(q.size(2) < (1 << 24) && k.size(2) < (1 << 24), "qk_norm_rope: too many heads");
    s.heads[0] = static_cast<int>(q.size(2));
    s.heads[1] = static_cast<int>(k.size(2));
    s.D = static_cast<int>(q.size(3));
    s.eps = static_cast<float>(eps);
    const OptT* ws[2] = {&wq, &wk};
    for (int i = 0; i < 2; ++i) {
      if (!given(*ws[i])) continue;
      const Tensor& t = **ws[i];
      TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == s.D && t.device() == q.device(),
                  "qk_norm_rope: weights must be contiguous fp32 of D values");
      w[i] = t.data_ptr<float>();
    }
    TORCH_CHECK(rot >= 0 && rot % 2 == 0 && rot <= s.D, "qk_norm_rope: rot_dim must be even and <= head dim");
    s.rot = static_cast<int>(rot);
    vec.elems(s.D);
    vec.elems(s.rot / 2);
    if (!s.rot) return;
    TORCH_CHECK(given(cos) && given(sin), "qk_norm_rope: rotation needs cos and sin");
    for (const Tensor* t : {&*cos, &*sin})
      TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->dim() == 2 &&
                      t->size(1) == s.rot / 2 && t->size(0) == cos->size(0) && t->device() == q.device(),
                  "qk_norm_rope: cos and sin must be contiguous fp32 [P, rot_dim / 2]");
    cosT = cos->data_ptr<float>();
    sinT = sin->data_ptr<float>();
    s.table_rows = cos->size(0);
    if (given(positions)) {
      const Tensor& p = *positions;
      TORCH_CHECK((p.scalar_type() == at::kLong || p.scalar_type() == at::kInt) && p.is_contiguous() &&
                      p.device() == q.device() && (p.numel() == s.S || p.numel() == s.B * s.S),
                  "qk_norm_rope: positions must be contiguous int32 / int64 [S] or [B, S]");
      s.pos = {p.data_ptr(), p.scalar_type() == at::kInt};
      s.pos_sb = p.numel() == s.S ? 0 : s.S;
    } else {
      TORCH_CHECK(s.S <= s.table_rows, "qk_norm_rope: ", s.S, " tokens, ", s.table_rows, " table rows");
    }
  }
};

std::vector<Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk, const OptT& cos,
                                 const OptT& sin, int64_t rot, const OptT& positions, double eps) {
  const c10::DeviceGuard g(q.device());
  Call c(q, k, wq, wk, cos, sin, rot, positions, eps);
  const Tensor yq = torch::empty(q.sizes(), q.options()), yk = torch::empty(k.sizes(), k.options());
  const dca::HeadView x[2] = {c.view(q, 0), c.view(k, 1)}, y[2] = {c.view(yq, 0), c.view(yk, 1)};
  dca::qk_norm_rope_fwd(tdt(q), c.vec.bytes(), c.s, x, y, c.w, c.cosT, c.sinT, stream());
  return {yq, yk};
}

// dq_out / dk_out: where the gradients go (may be dyq / dyk themselves); absent: new tensors.
// need_dw: which weight gradients are wanted; acc_*: added to these instead of returned (fp32).
std::vector<Tensor> qk_norm_rope_bwd(const Tensor& dyq, const Tensor& dyk, const Tensor& q, const Tensor& k,
                                     const OptT& wq, const OptT& wk, const OptT& cos, const OptT& sin, int64_t rot,
                                     const OptT& positions, double eps, bool need_dwq, bool need_dwk,
                                     const OptT& acc_q, const OptT& acc_k, const OptT& dq_out, const OptT& dk_out) {
  const c10::DeviceGuard g(q.device());
  Call c(q, k, wq, wk, cos, sin, rot, positions, eps);
  const Tensor dq = given(dq_out) ? *dq_out : torch::empty(q.sizes(), q.options());
  const Tensor dk = given(dk_out) ? *dk_out : torch::empty(k.sizes(), k.options());
  const dca::HeadView dy[2] = {c.view(dyq, 0), c.view(dyk, 1)}, x[2] = {c.view(q, 0), c.view(k, 1)},
                      dx[2] = {c.view(dq, 0), c.view(dk, 1)};
  const bool need[2] = {need_dwq && c.w[0], need_dwk && c.w[1]};
  const OptT* acc[2] = {&acc_q, &acc_k};
  Tensor dw[2], partial;
  dca::ColumnOut out[2];
  const dca::ColumnOut* to[2] = {nullptr, nullptr};
  auto fo = q.options().dtype(at::kFloat);
  for (int i = 0; i < 2; ++i) {
    if (!need[i]) continue;
    Tensor t;
    if (given(*acc[i])) {
      t = **acc[i];
      TORCH_CHECK(t.is_contiguous() && t.numel() == c.s.D && t.device() == q.device() &&
                      (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16),
                  "qk_norm_rope: accumulation target must be contiguous fp32 / bf16 of D values");
    } else {
      t = dw[i] = torch::empty({c.s.D}, fo);
    }
    out[i] = {t.data_ptr(), nullptr, c.s.D, t.scalar_type() == at::kBFloat16, given(*acc[i])};
    to[i] = &out[i];
  }
  if (to[0] || to[1]) partial = torch::empty({dca::qk_norm_rope_partial_floats(c.s)}, fo);
  dca::qk_norm_rope_bwd(tdt(q), c.vec.bytes(), c.s, dy, x, dx, c.w, c.cosT, c.sinT,
                        partial.defined() ? partial.data_ptr<float>() : nullptr, to, stream());
  return {dq, dk, dw[0], dw[1]};
}

Tensor f32(const Tensor& w) { return w.defined() ? w.to(at::kFloat).contiguous() : w; }
OptT opt(const Tensor& t) { return t.defined() ? OptT(t) : OptT(); }
Tensor viewable(const Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }

// The operator with its gradient (an autograd node here: see EmbeddingNode).
struct QkNormRopeNode : torch::autograd::Function<QkNormRopeNode> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q_in,
                                                const Tensor& k_in, const OptT& wq, const OptT& wk, const OptT& cos,
                                                const OptT& sin, int64_t rot, const OptT& positions, double eps) {
    const Tensor q = viewable(q_in), k = viewable(k_in);
    const Tensor none, w[2] = {given(wq) ? *wq : none, given(wk) ? *wk : none};
    ctx->save_for_backward({q, k, w[0], w[1], given(cos) ? *cos : none, given(sin) ? *sin : none,
                            given(positions) ? *positions : none});
    // the parameters themselves, for their persistent gradients
    ctx->saved_data["wq"] = w[0];
    ctx->saved_data["wk"] = w[1];
    ctx->saved_data["rot"] = rot;
    ctx->saved_data["eps"] = eps;
    return qk_norm_rope(q, k, opt(f32(w[0])), opt(f32(w[1])), cos, sin, rot, positions, eps);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor params[2] = {ctx->saved_data["wq"].toTensor(), ctx->saved_data["wk"].toTensor()};
    bool need[2];
    OptT acc[2];
    size_t edge = 2;  // needs_input_grad counts the graph's edges: q, k and the weights that are there
    for (int i = 0; i < 2; ++i) {
      need[i] = params[i].defined() && ctx->needs_input_grad(edge++);
      if (need[i]) acc[i] = dca::grad_target(params[i]);
    }
    auto d = qk_norm_rope_bwd(viewable(grads[0]), viewable(grads[1]), s[0], s[1], opt(f32(s[2])), opt(f32(s[3])),
                              opt(s[4]), opt(s[5]), ctx->saved_data["rot"].toInt(), opt(s[6]),
                              ctx->saved_data["eps"].toDouble(), need[0], need[1], acc[0], acc[1], OptT(), OptT());
    torch::autograd::variable_list out(9);
    for (int i = 0; i < 2; ++i) {
      out[i] = d[i];
      if (d[2 + i].defined()) out[2 + i] = d[2 + i].to(params[i].scalar_type());
    }
    return dca::once(std::move(out), true);  // they depend on q, k and the weights
  }
};

std::vector<Tensor> qk_norm_rope_autograd(const Tensor& q, const Tensor& k, const OptT& wq, const OptT& wk,
                                          const OptT& cos, const OptT& sin, int64_t rot, const OptT& positions,
                                          double eps) {
  return QkNormRopeNode::apply(q, k, wq, wk, cos, sin, rot, positions, eps);
}
}  // namespace

void register_qk_norm_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("qk_norm_rope_autograd", &qk_norm_rope_autograd);
  m.def("qk_norm_rope", &qk_norm_rope, py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"),
        py::arg("cos"), py::arg("sin"), py::arg("rot"), py::arg("positions"), py::arg("eps"));
  m.def("qk_norm_rope_bwd", &qk_norm_rope_bwd, py::arg("dyq"), py::arg("dyk"), py::arg("q"), py::arg("k"),
        py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"), py::arg("sin"), py::arg("rot"),
        py::arg("positions"), py::arg("eps"), py::arg("need_dwq"), py::arg("need_dwk"),
        py::arg("acc_q") = py::none(), py::arg("acc_k") = py::none(), py::arg("dq_out") = py::none(),
        py::arg("dk_out") = py::none());
}
