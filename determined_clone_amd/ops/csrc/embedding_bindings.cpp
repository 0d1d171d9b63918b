// Bindings for the embedding kernels (embedding.hip).
#include <torch/extension.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>

#include <limits>

#include "autograd_util.h"
#include "embedding_api.h"

namespace {
using torch::Tensor;
using OptT = c10::optional<Tensor>;

hipStream_t stream() { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
constexpr int64_t kMaxWidth = 1 << 20;  // the kernels' grids take a row's columns in their second dimension
bool given(const OptT& t) { return t.has_value() && t->defined(); }

dca::TDtype tdt(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return dca::TDtype::kBF16;
    case at::kHalf: return dca::TDtype::kF16;
    case at::kFloat: return dca::TDtype::kF32;
    default: TORCH_CHECK(false, "embedding: unsupported dtype ", t.scalar_type());
  }
}

dca::Index index(const Tensor& t, const Tensor& like, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, what, " must be int32 or int64");
  TORCH_CHECK(t.is_contiguous() && t.device() == like.device(), what, " must be contiguous and on the table's device");
  return {t.data_ptr(), t.scalar_type() == at::kInt};
}

dca::EmbedIds ids_of(const Tensor& idx, const Tensor& like, int64_t rows, int64_t start, bool shard) {
  constexpr int64_t most = std::numeric_limits<int32_t>::max();
  TORCH_CHECK(idx.numel() < most && rows < most, "embedding: more than 2^31 - 2 ids or table rows");
  return {index(idx, like, "embedding: ids"), idx.numel(), start, rows, shard};
}

void check_table(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), what,
              ": a GPU table [rows, E] with contiguous rows is required");
  TORCH_CHECK(t.size(1) <= kMaxWidth, what, ": rows of more than ", kMaxWidth, " elements");
}

// idx [...], weight [V, E], pos_weight [P, E], positions like idx (absent: t % seq) -> [..., E]
Tensor embed_fwd(const Tensor& idx, const Tensor& weight, const OptT& pos_weight, const OptT& positions,
                 double scale, int64_t start, bool shard) {
  check_table(weight, "embed_fwd");
  const c10::DeviceGuard g(weight.device());
  const int64_t E = weight.size(1);
  const dca::EmbedIds ids = ids_of(idx, weight, weight.size(0), start, shard);
  auto sizes = idx.sizes().vec();
  sizes.push_back(E);
  Tensor out = torch::empty(sizes, weight.options());
  dca::WidestVec vec(static_cast<int>(weight.element_size()));
  vec.elems(E);
  vec.elems(weight.stride(0));
  vec.ptr(weight.data_ptr());
  dca::EmbedPos pos;
  if (given(pos_weight)) {
    check_table(*pos_weight, "embed_fwd positions");
    TORCH_CHECK(pos_weight->size(1) == E && pos_weight->scalar_type() == weight.scalar_type() &&
                    pos_weight->device() == weight.device(),
                "embed_fwd: the position table must match the token table's width, dtype and device");
    pos.table = pos_weight->data_ptr();
    pos.stride = pos_weight->stride(0);
    pos.rows = pos_weight->size(0);
    vec.elems(pos.stride);
    vec.ptr(pos.table);
    if (given(positions)) {
      TORCH_CHECK(positions->numel() == idx.numel(), "embed_fwd: one position per id is required");
      pos.ids = index(*positions, weight, "embed_fwd: positions");
    } else {
      TORCH_CHECK(idx.dim() > 0 && idx.size(-1) <= pos.rows, "embed_fwd: more tokens than positions");
      pos.S = idx.size(-1);
    }
  }
  TORCH_CHECK(idx.numel() == 0 || (weight.size(0) > 0 && (!given(pos_weight) || pos.rows > 0)),
              "embed_fwd: ids for an empty table");
  dca::embed_fwd(tdt(weight), vec.bytes() == 16, ids, weight.data_ptr(), weight.stride(0), pos,
                 static_cast<float>(scale), out.data_ptr(), static_cast<int>(E), stream());
  return out;
}

// The gradient's destination: `acc` (added to) or a new table.
Tensor destination(const OptT& acc, int64_t rows, int64_t E, const Tensor& dy) {
  if (!given(acc)) return torch::empty({rows, E}, dy.options());
  TORCH_CHECK(acc->is_contiguous() && acc->dim() == 2 && acc->size(0) == rows && acc->size(1) == E &&
                  acc->scalar_type() == dy.scalar_type() && acc->device() == dy.device(),
              "embedding: the accumulation target must be contiguous and like the table");
  return *acc;
}

// dW[v] (+)= scale * sum of dy's rows with id v; rows without an id keep what `acc` holds (or zero).
Tensor embed_grad(const Tensor& dy_in, const Tensor& idx, int64_t rows, double scale, int64_t start,
                  const OptT& acc) {
  TORCH_CHECK(dy_in.is_cuda() && dy_in.dim() == idx.dim() + 1 &&
                  dy_in.numel() == idx.numel() * dy_in.size(-1), "embed_grad: dy must be [*ids.shape, E]");
  const c10::DeviceGuard g(dy_in.device());
  Tensor dy = dy_in.contiguous();
  const int64_t E = dy.size(-1);
  TORCH_CHECK(E <= kMaxWidth, "embed_grad: rows of more than ", kMaxWidth, " elements");
  const dca::EmbedIds ids = ids_of(idx, dy, rows, start, true);
  Tensor out = destination(acc, rows, E, dy);
  if (E == 0) return out;
  Tensor ws = torch::empty({dca::embed_grad_workspace(ids.n, ids.rows, static_cast<int>(E))}, dy.options().dtype(at::kByte));
  dca::WidestVec vec(static_cast<int>(dy.element_size()));
  vec.elems(E);
  vec.ptr(dy.data_ptr());
  vec.ptr(out.data_ptr());
  dca::embed_grad(tdt(dy), vec.bytes() == 16, ids, dy.data_ptr(), out.data_ptr(), static_cast<int>(E),
                  static_cast<float>(scale), given(acc), ws.data_ptr(), stream());
  return out;
}

// dP[s] (+)= sum over the batch of dy [..., S, E]; rows S and up keep what `acc` holds (or zero).
Tensor embed_pos_grad(const Tensor& dy_in, int64_t rows, const OptT& acc) {
  TORCH_CHECK(dy_in.is_cuda() && dy_in.dim() >= 2 && dy_in.size(-2) <= rows,
              "embed_pos_grad: dy must be [..., S, E] with S <= rows");
  const c10::DeviceGuard g(dy_in.device());
  Tensor dy = dy_in.contiguous();
  const int64_t S = dy.size(-2), E = dy.size(-1), N = S * E;
  const int64_t filled = dy.numel() ? S : 0;
  Tensor out = destination(acc, rows, E, dy);
  if (!given(acc) && filled < rows) out.narrow(0, filled, rows - filled).zero_();
  if (dy.numel() == 0) return out;
  dca::WidestVec vec(static_cast<int>(dy.element_size()));
  vec.elems(N);
  vec.ptr(dy.data_ptr());
  vec.ptr(out.data_ptr());
  dca::batch_sum(tdt(dy), vec.bytes() == 16, dy.data_ptr(), out.data_ptr(), dy.numel() / N, N, given(acc), stream());
  return out;
}

// The operator with its gradient, as an autograd node here rather than in Python: a training step's
// lookup is a few microseconds of GPU time, less than a Python node costs on the host.
struct EmbeddingNode : torch::autograd::Function<EmbeddingNode> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& idx_in, const Tensor& weight,
                        const OptT& pos_weight, const OptT& positions_in, double scale, int64_t start, bool shard) {
    const Tensor idx = idx_in.contiguous();
    OptT positions, pos_rows;
    if (given(positions_in)) positions = positions_in->expand(idx.sizes()).contiguous();
    if (given(pos_weight)) pos_rows = rows_of(*pos_weight);
    // the tables as they are now are not needed again (and may be updated or moved before the backward)
    ctx->save_for_backward({idx, positions.has_value() ? *positions : Tensor()});
    ctx->saved_data["weight"] = weight;
    ctx->saved_data["pos_weight"] = given(pos_weight) ? *pos_weight : Tensor();
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["start"] = start;
    return embed_fwd(idx, rows_of(weight), pos_rows, positions, scale, start, shard);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &idx = saved[0], &positions = saved[1];
    const Tensor weight = ctx->saved_data["weight"].toTensor(), pos_weight = ctx->saved_data["pos_weight"].toTensor();
    const Tensor dy = grads[0].contiguous();
    torch::autograd::variable_list out(7);
    if (ctx->needs_input_grad(1)) {
      const OptT acc = dca::grad_target(weight);
      const Tensor dw = embed_grad(dy, idx, weight.size(0), ctx->saved_data["scale"].toDouble(),
                                   ctx->saved_data["start"].toInt(), acc);
      if (!given(acc)) out[1] = dw;
    }
    if (pos_weight.defined() && ctx->needs_input_grad(2)) {
      const OptT acc = dca::grad_target(pos_weight);
      const Tensor dp = positions.defined() ? embed_grad(dy, positions, pos_weight.size(0), 1.0, 0, acc)
                                            : embed_pos_grad(dy, pos_weight.size(0), acc);
      if (!given(acc)) out[2] = dp;
    }
    return dca::once(std::move(out), grads[0].requires_grad());  // linear: the tables do not enter
  }

 private:
  static Tensor rows_of(const Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.contiguous(); }
};

Tensor embedding(const Tensor& idx, const Tensor& weight, const OptT& pos_weight, const OptT& positions, double scale,
                 int64_t start, bool shard) {
  return EmbeddingNode::apply(idx, weight, pos_weight, positions, scale, start, shard);
}
}  // namespace

void register_embedding_ops(pybind11::module& m) {
  namespace py = pybind11;
  m.def("embedding", &embedding);
  m.def("embed_fwd", &embed_fwd, py::arg("idx"), py::arg("weight"), py::arg("pos_weight") = py::none(),
        py::arg("positions") = py::none(), py::arg("scale") = 1.0, py::arg("start") = 0, py::arg("shard") = false);
  m.def("embed_grad", &embed_grad, py::arg("dy"), py::arg("idx"), py::arg("rows"), py::arg("scale") = 1.0,
        py::arg("start") = 0, py::arg("acc") = py::none());
  m.def("embed_pos_grad", &embed_pos_grad, py::arg("dy"), py::arg("rows"), py::arg("acc") = py::none());
}
