// Products of rows sorted by expert (or node type) with each expert's matrix, on gfx950.
//
//   out[p, :] = rows[p, :] * weight[e]   for the rows p of expert e, offsets[e] <= p < offsets[e + 1]
//   out[p, :] = 0                        for the rows behind the last expert's
//
// The gradient of the rows is the same product with the matrices transposed.  No counterpart in the reference.
#include "gs_products.hpp"

namespace gs {
namespace {

using products::Group;
using products::Operand;

// Which tile of rows a workgroup makes: the tiles of all experts side by side, then those of the rows behind the last.
struct RowTile {
  int64_t expert, begin;  // of the tile's rows
  int64_t rows;           // up to the expert's last; none: no tile
  int64_t col;            // which tile of columns
};

// Every thread counts the tiles of rows of its share of the experts; the one in whose share the workgroup's lies finds it.
// Workgroups of one die take tiles that lie side by side, so that its cache holds what they share.
template <int THREADS>
__device__ __forceinline__ RowTile find_tile(const int64_t* __restrict__ offsets, int64_t experts, int64_t n, int tile_rows,
                                             int64_t col_tiles) {
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
  const int64_t tiles = total * col_tiles, per_die = (tiles + kXcds - 1) / kXcds, slot = blockIdx.x / kXcds;
  const int64_t which = blockIdx.x % kXcds * per_die + slot, at = slot < per_die ? which / col_tiles : total;
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
  t.col = which % col_tiles;
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

template <typename T, bool ACROSS, int BM, int BN, int WM, int WN, int RING, bool DIRECT>
__global__ void __launch_bounds__(WM * WN * kWave)
product_kernel(ProductArgs<T> p) {
  using Tile = products::Tile<T, false, ACROSS, BM, BN, WM, WN, RING, DIRECT>;
  __shared__ __attribute__((aligned(1024))) char s_steps[Tile::kBytes];
  RowTile t = find_tile<Tile::kThreads>(p.offsets, p.experts, p.n, BM, p.col_tiles);
  if (t.rows <= 0) return;
  t = {products::uniform(t.expert), products::uniform(t.begin), products::uniform(t.rows), products::uniform(t.col)};
  const int64_t col = t.col * BN, rows = t.rows < BM ? t.rows : BM;
  Tile tile;
  const bool live = t.expert < p.experts;
  const T* w = p.weight + (live ? t.expert * p.expert_stride : 0) + (ACROSS ? col : col * p.weight_stride);
  const Operand<T> a{p.rows + t.begin * p.row_stride, p.row_stride, rows, p.inner};
  const Operand<T> b = ACROSS ? Operand<T>{w, p.weight_stride, p.inner, p.outer - col}
                              : Operand<T>{w, p.weight_stride, p.outer - col, p.inner};
  tile.run(a, b, live ? p.inner : 0, s_steps);
  tile.write(p.out + t.begin * p.outer + col, p.outer, rows, p.outer - col);
}

// Tiles of rows that there can be: a part of one for every expert that has rows, and for the rows behind.
int64_t most_row_tiles(int64_t n, int64_t experts, int64_t tile_rows) {
  return n / tile_rows + (experts + 1 < n ? experts + 1 : n);
}

template <typename T, bool ACROSS, int BM, int BN, int WM, int WN, int RING, bool DIRECT>
int launch_product(ProductArgs<T> p, hipStream_t st) {
  constexpr int threads = WM * WN * kWave;
  p.col_tiles = (p.outer + BN - 1) / BN;
  const int64_t blocks = (most_row_tiles(p.n, p.experts, BM) * p.col_tiles + kXcds - 1) / kXcds * kXcds;
  GS_RETURN_IF_ERROR(check_grid("gs_expert_matmul", blocks, threads));
  hipLaunchKernelGGL((product_kernel<T, ACROSS, BM, BN, WM, WN, RING, DIRECT>), dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, st, p);
  return check_launch("expert_matmul");
}

template <typename T, bool ACROSS>
int choose_product(const ProductArgs<T>& p, hipStream_t st) {
  const bool direct = products::direct_rows(p.rows, p.row_stride, p.inner, 256) &&
                      products::direct_rows(p.weight, p.weight_stride, ACROSS ? p.outer : p.inner, 256) &&
                      p.expert_stride % Chunk<T>::kVec == 0;
  if (!direct) return launch_product<T, ACROSS, 128, 128, 2, 2, 3, false>(p, st);
  if constexpr (sizeof(T) == 2)
    return launch_product<T, ACROSS, 256, 256, 2, 4, 4, true>(p, st);
  return launch_product<T, ACROSS, 128, 128, 2, 2, 3, true>(p, st);
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
    return transposed ? choose_product<T, false>(p, st) : choose_product<T, true>(p, st);
  });
}
