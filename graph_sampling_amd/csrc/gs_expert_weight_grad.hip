// Gradients of the experts' matrices (gs_expert_products.hip), on gfx950.
//
//   dweight[e] = sum over the rows p of expert e of rows[p, :]^T * grad[p, :],   zeros for an expert without rows
//
// Products whose depth is an expert's number of rows.  No counterpart in the reference.
#include "gs_products.hpp"

namespace gs {
namespace {

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
  // where the rows are cut into pieces of `piece` for the sake of more workgroups: the sums of each, and how many there are
  float* sums;
  int64_t piece, pieces;
};

// Pieces are cut at multiples of `piece`, and where an expert ends.  Of expert e, piece c (from piece * c on) is the
// (c + e)-th of all: the next expert begins in the same piece or behind it.
struct Pieces {
  int64_t first, last;  // of an expert; last < first: it has no rows
};
__device__ __forceinline__ Pieces pieces_of(const Group& g, int64_t expert, int64_t piece) {
  return {g.begin / piece + expert, g.rows() > 0 ? (g.end - 1) / piece + expert : -1};
}

// The expert whose piece `at` is, or -1.
template <int THREADS>
__device__ __forceinline__ int64_t find_expert(const int64_t* __restrict__ offsets, int64_t experts, int64_t n, int64_t piece,
                                               int64_t at) {
  __shared__ int64_t s_found;
  if (threadIdx.x == 0) s_found = -1;
  __syncthreads();
  for (int64_t e = threadIdx.x; e < experts; e += THREADS) {
    const Pieces p = pieces_of(products::group_of(offsets, experts, n, e), e, piece);
    if (at >= p.first && at <= p.last) s_found = e;  // (one, if the offsets ascend)
  }
  __syncthreads();
  return products::uniform(s_found);
}

template <typename T, int BM, int BN, int WM, int WN, int RING, bool DIRECT, bool PIECES>
__global__ void __launch_bounds__(WM * WN * kWave)
weight_grad_kernel(WeightGradArgs<T> p) {
  using Tile = products::Tile<T, true, true, BM, BN, WM, WN, RING, DIRECT>;
  __shared__ __attribute__((aligned(1024))) char s_steps[Tile::kBytes];
  // (workgroups of one die make tiles of the same expert, or piece, which share its rows)
  const int64_t in_expert = p.row_tiles * p.col_tiles, all = in_expert * (PIECES ? p.pieces : p.experts);
  const int64_t per_die = (all + kXcds - 1) / kXcds, slot = blockIdx.x / kXcds, which = blockIdx.x % kXcds * per_die + slot;
  if (slot >= per_die || which >= all) return;
  const int64_t at = which % in_expert, row = at / p.col_tiles * BM, col = at % p.col_tiles * BN;
  int64_t expert = which / in_expert;
  if (PIECES) expert = find_expert<Tile::kThreads>(p.offsets, p.experts, p.n, p.piece, which / in_expert);
  if (expert < 0) return;
  Group g = products::group_of(p.offsets, p.experts, p.n, expert);
  if (PIECES) {
    const int64_t first = (which / in_expert - expert) * p.piece;
    g = {g.begin > first ? g.begin : first, g.end < first + p.piece ? g.end : first + p.piece};
  }
  g = {products::uniform(g.begin), products::uniform(g.end)};
  Tile tile;
  tile.run(Operand<T>{p.rows + g.begin * p.row_stride + row, p.row_stride, g.rows(), p.inner - row},
           Operand<T>{p.grad + g.begin * p.grad_stride + col, p.grad_stride, g.rows(), p.outer - col}, g.rows(), s_steps);
  if (PIECES)
    tile.write(p.sums + (which / in_expert * p.inner + row) * p.outer + col, p.outer, p.inner - row, p.outer - col);
  else
    tile.write(p.out + (expert * p.inner + row) * p.outer + col, p.outer, p.inner - row, p.outer - col);
}

// dweight[e] = the sums of its pieces, one after the other.
constexpr int kThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kThreads)
join_pieces_kernel(WeightGradArgs<T> p) {
  const int64_t size = p.inner * p.outer, total = p.experts * size;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t e = i / size, at = i - e * size;
    const Pieces of = pieces_of(products::group_of(p.offsets, p.experts, p.n, e), e, p.piece);
    float sum = 0.0f;
    for (int64_t q = of.first; q <= of.last; ++q) sum += p.sums[q * size + at];
    p.out[i] = static_cast<T>(sum);
  }
}

// How the rows are cut: not at all (0) where there are tiles enough.
int64_t piece_rows(int64_t n, int64_t experts, int64_t tiles) {
  constexpr int64_t kTiles = 1024, kRows = 512;
  if (tiles * experts >= kTiles / 2 || n < 2 * kRows * experts) return 0;
  const int64_t pieces = kTiles / tiles, rows = (n + pieces - 1) / pieces;
  return rows < kRows ? kRows : (rows + 31) / 32 * 32;
}
int64_t pieces_there(int64_t n, int64_t experts, int64_t piece) { return (n + piece - 1) / piece + experts; }

template <typename T, int BM, int BN, int WM, int WN, int RING, bool DIRECT>
int launch_weight_grad(WeightGradArgs<T> p, void* workspace, size_t workspace_bytes, hipStream_t st) {
  constexpr int threads = WM * WN * kWave;
  p.row_tiles = (p.inner + BM - 1) / BM;
  p.col_tiles = (p.outer + BN - 1) / BN;
  const int64_t tiles = p.row_tiles * p.col_tiles;
  p.piece = piece_rows(p.n, p.experts, (p.inner + 127) / 128 * ((p.outer + 127) / 128));
  const int64_t items = p.piece ? pieces_there(p.n, p.experts, p.piece) : p.experts;
  if (items > most_blocks(threads) / tiles - kXcds) return check_grid("gs_expert_matmul_grad", most_blocks(threads) + 1, threads);
  const dim3 grid(static_cast<unsigned>((items * tiles + kXcds - 1) / kXcds * kXcds));
  if (!p.piece) {
    hipLaunchKernelGGL((weight_grad_kernel<T, BM, BN, WM, WN, RING, DIRECT, false>), grid, dim3(threads), 0, st, p);
    return check_launch("expert_matmul_grad");
  }
  p.pieces = items;
  Carver ws(workspace, workspace_bytes);
  p.sums = ws.take<float>(static_cast<size_t>(items * p.inner * p.outer));
  if (!ws.ok) {
    set_error_text("gs_expert_matmul_grad: workspace needs %zu bytes, 256-byte aligned",
                   gs_expert_matmul_grad_workspace_bytes(p.n, p.inner, p.outer, p.experts));
    return GS_ERR_WORKSPACE;
  }
  hipLaunchKernelGGL((weight_grad_kernel<T, BM, BN, WM, WN, RING, DIRECT, true>), grid, dim3(threads), 0, st, p);
  GS_RETURN_IF_ERROR(check_launch("expert_matmul_grad"));
  const int64_t blocks = (p.experts * p.inner * p.outer + kThreads - 1) / kThreads;
  hipLaunchKernelGGL((join_pieces_kernel<T>), dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096)), dim3(kThreads), 0, st, p);
  return check_launch("expert_matmul_grad");
}

template <typename T>
int choose_weight_grad(const WeightGradArgs<T>& p, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const bool direct = products::direct_rows(p.rows, p.row_stride, p.inner, 32) &&
                      products::direct_rows(p.grad, p.grad_stride, p.outer, 32);
  if (!direct) return launch_weight_grad<T, 128, 128, 2, 2, 3, false>(p, workspace, workspace_bytes, st);
  if constexpr (sizeof(T) == 2) {
    if (p.inner > 128 && p.outer > 128)
      return launch_weight_grad<T, 256, 256, 2, 4, 4, true>(p, workspace, workspace_bytes, st);
  }
  return launch_weight_grad<T, 128, 128, 2, 2, 3, true>(p, workspace, workspace_bytes, st);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

size_t gs_expert_matmul_grad_workspace_bytes(int64_t n, int64_t inner, int64_t outer, int64_t num_experts) {
  constexpr int64_t kMost = int64_t(1) << 24;
  if (n <= 0 || n >= (int64_t(1) << 31) || inner <= 0 || inner >= kMost || outer <= 0 || outer >= kMost || num_experts <= 0 ||
      num_experts >= (int64_t(1) << 31))
    return 256;
  const int64_t piece = piece_rows(n, num_experts, (inner + 127) / 128 * ((outer + 127) / 128));
  return piece ? padded(static_cast<size_t>(pieces_there(n, num_experts, piece) * inner * outer) * sizeof(float)) : 256;
}

int gs_expert_matmul_grad(const void* rows, int64_t row_stride, int64_t inner, const void* grad,
                                     int64_t grad_stride, int64_t outer, int type, int64_t n, const int64_t* offsets,
                                     int64_t num_experts, void* dweight, void* workspace, size_t workspace_bytes,
                          void* stream) {
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
    const WeightGradArgs<T> p{static_cast<const T*>(rows), row_stride, static_cast<const T*>(grad), grad_stride, n, inner, outer,
                              offsets, num_experts, static_cast<T*>(dweight), 0, 0, nullptr, 0, 0};
    return choose_weight_grad<T>(p, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
