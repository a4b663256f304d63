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

struct ChooseFunction : public torch::autograd::Function<ChooseFunction> {
  static variable_list forward(AutogradContext* ctx, const torch::Tensor& logits, int64_t choices, bool normalize) {
    const auto [experts, weights] = hip::ExpertChoose(logits, choices, normalize);
    // (with normalize the logits are not looked at again: nothing of them is kept)
    ctx->save_for_backward({normalize ? torch::Tensor() : logits, experts, weights});
    ctx->saved_data["normalize"] = normalize;
    ctx->saved_data["num"] = logits.size(1);
    ctx->saved_data["type"] = static_cast<int64_t>(logits.scalar_type());
    ctx->mark_non_differentiable({experts});
    ctx->set_materialize_grads(false);
    return {experts, weights};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[1].defined()) return {{}, {}, {}};
    NoSecond(true, "experts' weights");  // (they depend on the logits, which are followed)
    at::NoGradGuard off;
    if (ctx->saved_data["normalize"].toBool())
      return {hip::ExpertChooseGradOfChosen(grads[1], saved[1], saved[2], ctx->saved_data["num"].toInt(),
                                            static_cast<torch::ScalarType>(ctx->saved_data["type"].toInt())),
              {},
              {}};
    return {hip::ExpertChooseGrad(grads[1], saved[0], saved[1], saved[2], false), {}, {}};
  }
};

struct MatmulFunction : public torch::autograd::Function<MatmulFunction> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& rows, const torch::Tensor& offsets,
                               const torch::Tensor& weight) {
    const auto out = hip::ExpertMatmul(rows, offsets, weight);  // (refuses what else would be asked for its sizes here)
    const bool of_rows = rows.requires_grad(), of_weight = weight.requires_grad();
    // (each is kept for the other's gradient)
    ctx->save_for_backward({of_weight ? rows : torch::Tensor(), offsets, of_rows ? weight : torch::Tensor()});
    ctx->saved_data["rows"] = of_rows;
    ctx->saved_data["weight"] = of_weight;
    ctx->saved_data["transposed"] = hip::ColumnsContiguous(weight);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {{}, {}, {}};
    const torch::Tensor &rows = saved[0], &weight = saved[2];
    const bool of_rows = ctx->saved_data["rows"].toBool(), of_weight = ctx->saved_data["weight"].toBool();
    NoSecond(grads[0].requires_grad() || (of_rows && weight.requires_grad()) || (of_weight && rows.requires_grad()),
             "experts' products");
    at::NoGradGuard off;
    torch::Tensor d_rows, d_weight;
    if (of_rows) d_rows = hip::ExpertMatmul(grads[0], saved[1], weight.transpose(1, 2));
    if (of_weight) d_weight = hip::ExpertMatmulGrad(grads[0], rows, saved[1], ctx->saved_data["transposed"].toBool());
    return {d_rows, {}, d_weight};
  }
};

struct DropoutFunction : public torch::autograd::Function<DropoutFunction> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::optional<torch::Tensor>& added,
                               double p, int64_t seed, const torch::optional<torch::Tensor>& seed_tensor) {
    const auto residual = added.value_or(torch::Tensor()), seed_at = seed_tensor.value_or(torch::Tensor());
    ctx->save_for_backward({seed_at});  // (a seed that changes between the passes is refused by its version)
    ctx->saved_data["p"] = p;
    ctx->saved_data["seed"] = seed;
    ctx->saved_data["x"] = x.requires_grad();
    ctx->saved_data["residual"] = residual.defined() && residual.requires_grad();
    return hip::Dropout(x, p, seed, seed_at, residual);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto seed_at = ctx->get_saved_variables()[0];
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}};
    torch::Tensor dx, d_residual;
    if (ctx->saved_data["residual"].toBool()) d_residual = grads[0];
    if (ctx->saved_data["x"].toBool()) {
      NoSecond(grads[0].requires_grad(), "a dropout");
      at::NoGradGuard off;
      dx = hip::Dropout(grads[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt(), seed_at,
                        torch::Tensor());
    }
    return {dx, d_residual, {}, {}, {}};
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

std::tuple<torch::Tensor, torch::Tensor> ExpertChoose(torch::Tensor logits, int64_t choices, bool normalize) {
  if (!Followed(logits)) return hip::ExpertChoose(logits, choices, normalize);
  const auto out = ChooseFunction::apply(logits, choices, normalize);
  return {out[0], out[1]};
}

torch::Tensor ExpertChooseGrad(torch::Tensor grad, torch::Tensor logits, torch::Tensor experts, torch::Tensor weights,
                               bool normalize) {
  TORCH_CHECK(!Followed(grad) && !Followed(logits) && !Followed(weights),
              "the gradient of experts' weights cannot be differentiated once more");
  return hip::ExpertChooseGrad(grad, logits, experts, weights, normalize);
}

torch::Tensor ExpertMatmul(torch::Tensor rows, torch::Tensor order, torch::Tensor place, torch::Tensor offsets,
                           torch::Tensor weight) {
  CheckOrder(order, place);
  const bool followed = Followed(rows), weighed = Followed(weight);
  TORCH_CHECK(rows.dim() != 2 || rows.size(0) == place.numel(), "rows of ", rows.size(0), " items, places of ", place.numel());
  return followed || weighed ? MatmulFunction::apply(rows, offsets, weight) : hip::ExpertMatmul(rows, offsets, weight);
}

torch::Tensor ExpertMatmulGrad(torch::Tensor grad, torch::Tensor rows, torch::Tensor offsets) {
  TORCH_CHECK(!Followed(grad) && !Followed(rows), "the gradient of experts' products cannot be differentiated once more");
  return hip::ExpertMatmulGrad(grad, rows, offsets, false);
}

torch::Tensor Dropout(torch::Tensor x, double p, torch::optional<int64_t> seed, torch::optional<torch::Tensor> seed_at,
                      torch::optional<torch::Tensor> residual) {
  const torch::Tensor at = seed_at.has_value() ? seed_at.value() : torch::Tensor();
  const torch::Tensor r = residual.has_value() ? residual.value() : torch::Tensor();
  TORCH_CHECK(!seed.has_value() || !at.defined(), "one seed, a number or a tensor, not both");
  const bool followed = Followed(x), added = Followed(r);
  // (a number would be recorded, and every replay draw the same)
  TORCH_CHECK(seed.has_value() || at.defined() || !x.is_cuda() || !hip::Capturing(x),
              "a graph is being recorded: dropout needs a seed, a tensor that changes between replays");
  const int64_t number = seed.has_value() ? seed.value() : at.defined() ? 0 : static_cast<int64_t>(hip::NextSeed());
  if (!at.defined()) seed_at = torch::nullopt;
  if (!r.defined()) residual = torch::nullopt;
  return followed || added ? DropoutFunction::apply(x, residual, p, number, seed_at) : hip::Dropout(x, p, number, at, r);
}

}  // namespace gs
