// Products of rows sorted by expert (or node type) with each expert's matrix, on gfx950.
//
//   out[p, :] = rows[p, :] * weight[e]   for the rows p of expert e, offsets[e] <= p < offsets[e + 1]
//   out[p, :] = 0                        for the rows behind the last expert's
//
// The gradient of the rows is the same product with the matrices transposed.  No counterpart in the reference.
#include "gs_products.hpp"

namespace gs {
namespace {

using products::Acc;
using products::Group;
using products::Operand;

// Which tile of rows a workgroup makes: the tiles of all experts side by side, then those of the rows behind the last.
struct RowTile {
  int64_t expert, begin;  // of the tile's rows
  int64_t rows;           // up to the expert's last; none: no tile
  int64_t tiles;          // of all experts
};

// Every thread counts the tiles of its share of the experts; the one in whose share tile `at` lies finds it.
template <int THREADS>
__device__ __forceinline__ RowTile find_tile(const int64_t* __restrict__ offsets, int64_t experts, int64_t n, int tile_rows,
                                             int64_t at) {
  __shared__ int64_t s_wave[THREADS / kWave];
  __shared__ RowTile s_found;
  const int64_t each = (experts + 1 + THREADS - 1) / THREADS, first = each * threadIdx.x;
  const int64_t last = first + each < experts + 1 ? first + each : experts + 1;
  int64_t mine = 0;
  for (int64_t e = first; e < last; ++e)
    mine += (products::group_of(offsets, experts, n, e).rows() + tile_rows - 1) / tile_rows;
  int64_t upto = mine;
  const int lane = threadIdx.x % kWave;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t other = __shfl_up(upto, d, kWave);
    if (lane >= d) upto += other;
  }
  if (lane == kWave - 1) s_wave[threadIdx.x / kWave] = upto;
  if (threadIdx.x == 0) s_found.rows = 0;
  __syncthreads();
  int64_t total = 0;
  for (int w = 0; w < THREADS / kWave; ++w) {
    if (w < static_cast<int>(threadIdx.x) / kWave) upto += s_wave[w];
    total += s_wave[w];
  }
  int64_t from = upto - mine;
  if (at >= from && at < upto) {
    for (int64_t e = first; e < last; ++e) {
      const Group g = products::group_of(offsets, experts, n, e);
      const int64_t here = (g.rows() + tile_rows - 1) / tile_rows;
      if (at < from + here) {
        s_found.expert = e;
        s_found.begin = g.begin + (at - from) * tile_rows;
        s_found.rows = g.end - s_found.begin;
        break;
      }
      from += here;
    }
  }
  __syncthreads();
  RowTile t = s_found;
  t.tiles = total;
  return t;
}

template <typename T>
struct ProductArgs {
  const T* rows;
  int64_t row_stride, n, inner;
  const T* weight;
  int64_t expert_stride, weight_stride, experts, outer;
  const int64_t* offsets;
  T* out;
  int64_t col_tiles;
};

template <typename T, bool ACROSS, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(WM * WN * kWave)
product_kernel(ProductArgs<T> p) {
  using Tile = products::Tile<T, false, ACROSS, BM, BN, WM, WN>;
  __shared__ __attribute__((aligned(16))) char s_steps[Tile::kBytes];
  const int64_t at = blockIdx.x;
  const RowTile t = find_tile<Tile::kThreads>(p.offsets, p.experts, p.n, BM, at / p.col_tiles);
  if (t.rows <= 0) return;
  const int64_t col = at % p.col_tiles * BN, rows = t.rows < BM ? t.rows : BM;
  Tile tile;
  const bool live = t.expert < p.experts;
  const T* w = p.weight + (live ? t.expert * p.expert_stride : 0) + (ACROSS ? col : col * p.weight_stride);
  const Operand<T> a{p.rows + t.begin * p.row_stride, p.row_stride, rows, p.inner};
  const Operand<T> b = ACROSS ? Operand<T>{w, p.weight_stride, p.inner, p.outer - col}
                              : Operand<T>{w, p.weight_stride, p.outer - col, p.inner};
  tile.run(a, b, live ? p.inner : 0, s_steps);
  T* const out = p.out + t.begin * p.outer + col;
  tile.each([&](int m, int n, Acc v) {
    if (m < rows) products::store_four(out + m * p.outer + n, v, p.outer - col - n);
  });
}

// Tiles of rows that there can be: a part of one for every expert that has rows, and for the rows behind.
int64_t most_row_tiles(int64_t n, int64_t experts, int64_t tile_rows) {
  return n / tile_rows + (experts + 1 < n ? experts + 1 : n);
}

template <typename T, bool ACROSS, int BM, int BN, int WM, int WN>
int launch_product(ProductArgs<T> p, hipStream_t st) {
  constexpr int threads = WM * WN * kWave;
  p.col_tiles = (p.outer + BN - 1) / BN;
  const int64_t blocks = most_row_tiles(p.n, p.experts, BM) * p.col_tiles;
  GS_RETURN_IF_ERROR(check_grid("gs_expert_matmul", blocks, threads));
  hipLaunchKernelGGL((product_kernel<T, ACROSS, BM, BN, WM, WN>), dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, st, p);
  return check_launch("expert_matmul");
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_expert_matmul(const void* rows, int64_t row_stride, int64_t n, int64_t inner, int type, const void* weight,
                                int64_t expert_stride, int64_t weight_stride, int transposed, int64_t num_experts,
                                int64_t outer, const int64_t* offsets, void* out, void* stream) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16,
             "gs_expert_matmul: value type %d is none of GS_F32, GS_F16, GS_BF16", type);
  GS_REQUIRE(n >= 0 && inner >= 0 && outer >= 0 && num_experts >= 0, "gs_expert_matmul: negative size");
  GS_REQUIRE(n < (int64_t(1) << 31), "gs_expert_matmul: %lld rows, at most 2^31 - 1 are taken", static_cast<long long>(n));
  GS_REQUIRE(inner < (int64_t(1) << 24) && outer < (int64_t(1) << 24),
             "gs_expert_matmul: rows of %lld and %lld values, at most 2^24 - 1 are taken", static_cast<long long>(inner),
             static_cast<long long>(outer));
  GS_REQUIRE(num_experts < (int64_t(1) << 31), "gs_expert_matmul: %lld experts, at most 2^31 - 1 are taken",
             static_cast<long long>(num_experts));
  GS_REQUIRE(row_stride >= 0 && expert_stride >= 0 && weight_stride >= 0, "gs_expert_matmul: negative stride");
  if (n == 0 || outer == 0) return GS_OK;
  GS_REQUIRE(offsets && out && (inner == 0 || (rows && (num_experts == 0 || weight))), "gs_expert_matmul: null array");
  GS_REQUIRE(aligned_to(rows, value_bytes(type)) && aligned_to(weight, value_bytes(type)) && aligned_to(out, value_bytes(type)),
             "gs_expert_matmul: rows or matrices not aligned to their type");
  return with_value_type(type, "gs_expert_matmul", [&](auto zero) {
    using T = decltype(zero);
    const ProductArgs<T> p{static_cast<const T*>(rows), row_stride, n, inner, static_cast<const T*>(weight), expert_stride,
                           weight_stride, num_experts, outer, offsets, static_cast<T*>(out), 0};
    const auto st = static_cast<hipStream_t>(stream);
    return transposed ? launch_product<T, false, 128, 128, 2, 2>(p, st) : launch_product<T, true, 128, 128, 2, 2>(p, st);
  });
}
