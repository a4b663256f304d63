#include "row_ops.h"

#include <ATen/TensorSubclassLikeUtils.h>
#include <torch/csrc/autograd/custom_function.h>

#include "hip_ops.h"

namespace gs {
namespace {
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A tensor that a gradient may flow back to, and a call recorded into a graph: the backward pass makes the
// stream of the node that made t (the accumulator of a leaf) wait for the recording one, which ends the process
// when that stream is outside the recording.
void CheckRecording(const torch::Tensor& t) {
  if (!t.is_cuda() || !hip::Capturing(t)) return;
  const auto node = t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn();
  if (!node) return;
  const auto stream = node->stream();
  TORCH_CHECK(stream.has_value() && hip::RecordedWith(t, stream->id()),
              "a graph is being recorded, and an eager graph of the same leaf lives, or the tensor was made, on a "
              "stream outside the recording: its gradient cannot be recorded (drop the eager outputs first, or "
              "make them on the recording stream)");
}

// whether somebody follows what becomes of t: only then is a node made
bool Followed(const torch::Tensor& t) {
  if (!t.defined()) return false;
  TORCH_CHECK(!at::isTensorSubclassLike(t), "tensors under a transform, and tensor subclasses, are not taken");
  if (t._fw_grad(0).defined()) return true;
  if (!at::GradMode::is_enabled() || !t.requires_grad()) return false;
  CheckRecording(t);
  return true;
}

void NoSecond(bool needed, const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled() || !needed, "the gradient of ", what, " cannot be differentiated once more");
}

torch::Tensor Rows2d(const torch::Tensor& t, int64_t rows) {
  if (t.dim() == 2 && t.size(0) == rows) return t;
  const int64_t dim = t.dim() > 0 ? t.size(-1) : 1;
  return t.reshape({rows, dim});
}

struct EmbeddingFunction : public torch::autograd::Function<EmbeddingFunction> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& table, const torch::Tensor& ids, double scale,
                               bool sparse_grad) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = table.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["sparse"] = sparse_grad;
    return hip::EmbeddingLookup(table, ids, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto ids = ctx->get_saved_variables()[0];
    if (!grads[0].defined()) return {{}, {}, {}, {}};
    NoSecond(grads[0].requires_grad(), "an embedding");
    at::NoGradGuard off;
    const int64_t rows = ctx->saved_data["rows"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    const auto g = Rows2d(grads[0], ids.numel());
    if (!ctx->saved_data["sparse"].toBool()) return {hip::EmbeddingGrad(g, ids, rows, scale), {}, {}, {}};
    const auto [met, values] = hip::EmbeddingSparseGrad(g, ids, rows, scale);
    const auto sparse = at::_sparse_coo_tensor_unsafe(met.unsqueeze(0), values, {rows, g.size(1)});
    sparse._coalesced_(true);
    return {sparse, {}, {}, {}};
  }
};

struct GatherFunction : public torch::autograd::Function<GatherFunction> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& place,
                               const torch::Tensor& offsets) {
    ctx->save_for_backward({place});
    return hip::ExpertGather(x, place, offsets);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto place = ctx->get_saved_variables()[0];
    if (!grads[0].defined()) return {{}, {}, {}};
    NoSecond(grads[0].requires_grad(), "rows sent to experts");
    at::NoGradGuard off;
    return {hip::ExpertCombine(grads[0], place, torch::nullopt), {}, {}};
  }
};

struct DispatchFunction : public torch::autograd::Function<DispatchFunction> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& experts,
                               int64_t num_experts) {
    const auto [rows, order, place, offsets] = hip::ExpertDispatch(x, experts, num_experts);
    ctx->save_for_backward({place});
    ctx->mark_non_differentiable({order, place, offsets});
    ctx->set_materialize_grads(false);  // (zeros for the three that have none)
    return {rows, order, place, offsets};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return GatherFunction::backward(ctx, {grads[0]});
  }
};

struct CombineFunction : public torch::autograd::Function<CombineFunction> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& y, const torch::Tensor& place,
                               const torch::Tensor& offsets, const torch::optional<torch::Tensor>& weights) {
    const bool of_rows = y.requires_grad(), of_weights = weights.has_value() && weights.value().requires_grad();
    // (y, the larger, is kept for the weights' gradient only)
    ctx->save_for_backward({of_weights ? y : torch::Tensor(), place, offsets,
                            weights.has_value() ? weights.value() : torch::Tensor()});
    ctx->saved_data["weights"] = of_weights;
    ctx->saved_data["rows"] = of_rows;
    return hip::ExpertCombine(y, place, weights);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {{}, {}, {}, {}};
    const torch::Tensor &y = saved[0], &weights = saved[3];
    const bool of_rows = ctx->saved_data["rows"].toBool(), of_weights = ctx->saved_data["weights"].toBool();
    NoSecond(grads[0].requires_grad() || (of_rows && weights.defined() && weights.requires_grad()) ||
                 (of_weights && y.requires_grad()),
             "experts' rows added up");
    at::NoGradGuard off;
    auto [dy, dw] = hip::ExpertCombineGrad(grads[0], y, saved[1], saved[2], weights, of_rows, of_weights);
    return {dy, {}, {}, dw};
  }
};

// order is the caller's: the kernels go by place, but the three belong together
void CheckOrder(const torch::Tensor& order, const torch::Tensor& place) {
  TORCH_CHECK(order.defined() && place.defined(), "order or place is undefined");
  TORCH_CHECK(order.dim() == 1 && order.numel() == place.numel() && order.scalar_type() == torch::kInt32,
              "order must be int32 [", place.numel(), "], got ", order.scalar_type(), " ", order.sizes());
}
}  // namespace

torch::Tensor Embedding(torch::Tensor table, torch::Tensor ids, double scale, bool sparse_grad) {
  return Followed(table) ? EmbeddingFunction::apply(table, ids, scale, sparse_grad)
                         : hip::EmbeddingLookup(table, ids, scale);
}

torch::Tensor EmbeddingGrad(torch::Tensor grad, torch::Tensor ids, int64_t num_rows, double scale) {
  TORCH_CHECK(!Followed(grad), "the gradient of an embedding cannot be differentiated once more");
  return hip::EmbeddingGrad(Rows2d(grad, ids.numel()), ids, num_rows, scale);
}

std::tuple<torch::Tensor, torch::Tensor> EmbeddingSparseGrad(torch::Tensor grad, torch::Tensor ids, int64_t num_rows,
                                                             double scale) {
  TORCH_CHECK(!Followed(grad), "the gradient of an embedding cannot be differentiated once more");
  return hip::EmbeddingSparseGrad(Rows2d(grad, ids.numel()), ids, num_rows, scale);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> ExpertSort(torch::Tensor experts, int64_t num_experts) {
  return hip::ExpertSort(experts, num_experts);
}

torch::Tensor ExpertGather(torch::Tensor x, torch::Tensor order, torch::Tensor place, torch::Tensor offsets) {
  CheckOrder(order, place);
  return Followed(x) ? GatherFunction::apply(x, place, offsets) : hip::ExpertGather(x, place, offsets);
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> ExpertDispatch(torch::Tensor x,
                                                                                      torch::Tensor experts,
                                                                                      int64_t num_experts) {
  if (!Followed(x)) return hip::ExpertDispatch(x, experts, num_experts);
  const auto out = DispatchFunction::apply(x, experts, num_experts);
  return {out[0], out[1], out[2], out[3]};
}

torch::Tensor ExpertCombine(torch::Tensor y, torch::Tensor order, torch::Tensor place, torch::Tensor offsets,
                            torch::optional<torch::Tensor> weights) {
  CheckOrder(order, place);
  const torch::Tensor w = weights.has_value() ? weights.value() : torch::Tensor();
  const bool followed = Followed(y), weighed = Followed(w);
  if (!w.defined()) weights = torch::nullopt;
  return followed || weighed ? CombineFunction::apply(y, place, offsets, weights) : hip::ExpertCombine(y, place, weights);
}

std::tuple<torch::Tensor, torch::Tensor> ExpertCombineGrad(torch::Tensor grad, torch::Tensor y, torch::Tensor order,
                                                           torch::Tensor place, torch::Tensor offsets,
                                                           torch::optional<torch::Tensor> weights) {
  CheckOrder(order, place);
  const torch::Tensor w = weights.has_value() ? weights.value() : torch::Tensor();
  TORCH_CHECK(!Followed(grad) && !Followed(y) && !Followed(w),
              "the gradient of experts' rows added up cannot be differentiated once more");
  auto [dy, dw] = hip::ExpertCombineGrad(grad, y, place, offsets, weights, true, w.defined());
  if (!dw.defined()) dw = torch::empty({0}, grad.options());
  return {dy, dw};
}

}  // namespace gs
