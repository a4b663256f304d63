// Rows of values moved by ids, with gradients: embedding lookup, rows sorted by expert (or node
// type) and back.  No counterpart in the reference, whose examples index feature matrices with
// torch.  Values are float32, float16 or bfloat16, sums are float32, rounded once.
//
// Gradients are first ones: where a second one would be needed the backward pass raises.  The backward
// pass of a leaf whose gradient is accumulated on another stream (an eager graph of it lives) cannot be
// recorded into a HIP graph; that is refused in the forward call.
#pragma once

#include <torch/torch.h>

#include <tuple>

namespace gs {

// [*ids.shape, dim]: scale * table[ids], zeros for an id outside the table.  sparse_grad: the table's
// gradient is a coalesced sparse tensor of the rows that were met.
torch::Tensor Embedding(torch::Tensor table, torch::Tensor ids, double scale, bool sparse_grad);
// the gradients by themselves, from the gradient of what was looked up, [*ids.shape, dim]
torch::Tensor EmbeddingGrad(torch::Tensor grad, torch::Tensor ids, int64_t num_rows, double scale);
std::tuple<torch::Tensor, torch::Tensor> EmbeddingSparseGrad(torch::Tensor grad, torch::Tensor ids,
                                                             int64_t num_rows, double scale);

// (order, place, offsets) of experts [tokens] or [tokens, choices]; see gs_expert_sort in gs_hip.h
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> ExpertSort(torch::Tensor experts, int64_t num_experts);
// [tokens * choices, dim]: a copy of each token's row at each of its places, zeros behind offsets[-1]
torch::Tensor ExpertGather(torch::Tensor x, torch::Tensor order, torch::Tensor place, torch::Tensor offsets);
// both: (rows, order, place, offsets)
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> ExpertDispatch(torch::Tensor x,
                                                                                      torch::Tensor experts,
                                                                                      int64_t num_experts);
// [tokens, dim]: the sum of each token's rows, times weights (like place; none: ones)
torch::Tensor ExpertCombine(torch::Tensor y, torch::Tensor order, torch::Tensor place, torch::Tensor offsets,
                            torch::optional<torch::Tensor> weights);
// (gradient of y, gradient of the weights or an empty tensor without any)
std::tuple<torch::Tensor, torch::Tensor> ExpertCombineGrad(torch::Tensor grad, torch::Tensor y, torch::Tensor order,
                                                           torch::Tensor place, torch::Tensor offsets,
                                                           torch::optional<torch::Tensor> weights);

}  // namespace gs
