// Gradients of the experts' matrices (gs_expert_products.hip), on gfx950.
//
//   dweight[e] = sum over the rows p of expert e of rows[p, :]^T * grad[p, :],   zeros for an expert without rows
//
// Products whose depth is an expert's number of rows.  No counterpart in the reference.
#include "gs_products.hpp"

namespace gs {
namespace {

using products::Acc;
using products::Group;
using products::Operand;

template <typename T>
struct WeightGradArgs {
  const T* rows;
  int64_t row_stride;
  const T* grad;
  int64_t grad_stride, n, inner, outer;
  const int64_t* offsets;
  int64_t experts;
  T* out;
  int64_t row_tiles, col_tiles;
};

template <typename T, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * kWave)
weight_grad_kernel(WeightGradArgs<T> p) {
  using Tile = products::Tile<T, true, true, BM, BN, WM, WN>;
  __shared__ __attribute__((aligned(16))) char s_steps[Tile::kBytes];
  const int64_t in_expert = p.row_tiles * p.col_tiles, expert = blockIdx.x / in_expert, at = blockIdx.x % in_expert;
  const int64_t row = at / p.col_tiles * BM, col = at % p.col_tiles * BN;
  const Group g = products::group_of(p.offsets, p.experts, p.n, expert);
  Tile tile;
  tile.run(Operand<T>{p.rows + g.begin * p.row_stride + row, p.row_stride, g.rows(), p.inner - row},
           Operand<T>{p.grad + g.begin * p.grad_stride + col, p.grad_stride, g.rows(), p.outer - col}, g.rows(), s_steps);
  T* const out = p.out + (expert * p.inner + row) * p.outer + col;
  tile.each([&](int m, int n, Acc v) {
    if (row + m < p.inner) products::store_four(out + m * p.outer + n, v, p.outer - col - n);
  });
}

template <typename T, int BM, int BN, int WM, int WN>
int launch_weight_grad(WeightGradArgs<T> p, hipStream_t st) {
  constexpr int threads = WM * WN * kWave;
  p.row_tiles = (p.inner + BM - 1) / BM;
  p.col_tiles = (p.outer + BN - 1) / BN;
  const int64_t tiles = p.row_tiles * p.col_tiles;
  if (p.experts > most_blocks(threads) / tiles) return check_grid("gs_expert_matmul_grad", most_blocks(threads) + 1, threads);
  hipLaunchKernelGGL((weight_grad_kernel<T, BM, BN, WM, WN>), dim3(static_cast<unsigned>(p.experts * tiles)), dim3(threads), 0,
                     st, p);
  return check_launch("expert_matmul_grad");
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_expert_matmul_grad(const void* rows, int64_t row_stride, int64_t inner, const void* grad,
                                     int64_t grad_stride, int64_t outer, int type, int64_t n, const int64_t* offsets,
                                     int64_t num_experts, void* dweight, void* stream) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16,
             "gs_expert_matmul_grad: value type %d is none of GS_F32, GS_F16, GS_BF16", type);
  GS_REQUIRE(n >= 0 && inner >= 0 && outer >= 0 && num_experts >= 0, "gs_expert_matmul_grad: negative size");
  GS_REQUIRE(n < (int64_t(1) << 31), "gs_expert_matmul_grad: %lld rows, at most 2^31 - 1 are taken",
             static_cast<long long>(n));
  GS_REQUIRE(inner < (int64_t(1) << 24) && outer < (int64_t(1) << 24),
             "gs_expert_matmul_grad: rows of %lld and %lld values, at most 2^24 - 1 are taken",
             static_cast<long long>(inner), static_cast<long long>(outer));
  GS_REQUIRE(num_experts < (int64_t(1) << 31), "gs_expert_matmul_grad: %lld experts, at most 2^31 - 1 are taken",
             static_cast<long long>(num_experts));
  GS_REQUIRE(row_stride >= 0 && grad_stride >= 0, "gs_expert_matmul_grad: negative stride");
  if (num_experts == 0 || inner == 0 || outer == 0) return GS_OK;
  GS_REQUIRE(offsets && dweight && (n == 0 || (rows && grad)), "gs_expert_matmul_grad: null array");
  GS_REQUIRE(aligned_to(rows, value_bytes(type)) && aligned_to(grad, value_bytes(type)) &&
                 aligned_to(dweight, value_bytes(type)),
             "gs_expert_matmul_grad: rows or matrices not aligned to their type");
  return with_value_type(type, "gs_expert_matmul_grad", [&](auto zero) {
    using T = decltype(zero);
    return launch_weight_grad<T, 128, 128, 2, 2>(
        WeightGradArgs<T>{static_cast<const T*>(rows), row_stride, static_cast<const T*>(grad), grad_stride, n, inner, outer,
                          offsets, num_experts, static_cast<T*>(dweight), 0, 0},
        static_cast<hipStream_t>(stream));
  });
}
