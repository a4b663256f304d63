// Products of rows sorted by expert (or node type) with each expert's matrix, on gfx950.
//
//   out[p, :] = rows[p, :] * weight[e]   for the rows p of expert e, offsets[e] <= p < offsets[e + 1]
//   out[p, :] = 0                        for the rows behind the last expert's
//
// The gradient of the rows is the same product with the matrices transposed.  No counterpart in the reference.
#include "gs_expert_products.hpp"

namespace gs {
namespace {

using products::Operand;
using products::ProductArgs;
using products::RowTile;
using products::Way;

// rows, col: of the tile's first value
template <typename Tile, typename T, bool ACROSS>
__device__ __forceinline__ void make_tile(const ProductArgs<T>& p, const RowTile& t, int64_t first, int64_t rows, int64_t col,
                                          char* steps) {
  Tile tile;
  const bool live = t.expert < p.experts;
  const T* w = p.weight + (live ? t.expert * p.expert_stride : 0) + (ACROSS ? col : col * p.weight_stride);
  const Operand<T> a{p.rows + first * p.row_stride, p.row_stride, rows, p.inner};
  const Operand<T> b = ACROSS ? Operand<T>{w, p.weight_stride, p.inner, p.outer - col}
                              : Operand<T>{w, p.weight_stride, p.outer - col, p.inner};
  tile.run(a, b, live ? p.inner : 0, steps);
  tile.write(p.out + first * p.outer + col, p.outer, rows, p.outer - col);
}

// Large products: 131 072 rows x 2048 x 1024 by 64 experts, bf16, 519 us, 1.06 PFLOP/s (a batched library product of as many even
// groups 1.13), with the matrix cores busy 59 % of the cycles and the clock near 1.5 GHz in both.  What the others go to is not
// known: of matrices along the depth, where these take 577 us, a library product reaches 1.44 PFLOP/s.
// Large tiles, one a compute unit, leave much of the card idle behind the last full round; where they would fill less than
// half of it, their quarters are spread over it, which take a little over a third of the time: 16384 rows x 4096 x 2048 by
// 8 experts, bf16, 544 tiles, 253 us, 283 in whole tiles.
template <typename T, bool ACROSS, int BM, int BN, int WM, int WN, int RING, Way WAY>
__global__ void __launch_bounds__(WM * WN * kWave)
product_kernel(ProductArgs<T> p) {
  using Tile = products::Tile<T, false, ACROSS, BM, BN, WM, WN, RING, WAY>;
  constexpr bool kQuarters = BM == 256 && BN == 256;
  __shared__ __attribute__((aligned(1024))) char s_steps[Tile::kBytes];
  RowTile t = products::find_tile<Tile::kThreads, kQuarters>(p.offsets, p.experts, p.n, BM, p.col_tiles, p.first_block);
  if (t.rows <= 0) return;
  t = {products::uniform(t.expert), products::uniform(t.begin), products::uniform(t.rows), products::uniform(t.col),
       products::uniform(t.quarter)};
  if constexpr (kQuarters) {
    if (t.quarter >= 0) {
      using Quarter = products::Tile<T, false, ACROSS, BM / 2, BN / 2, WM, WN, RING, WAY>;
      const int64_t row = t.quarter / 2 * (BM / 2), col = t.col * BN + t.quarter % 2 * (BN / 2);
      if (row >= t.rows || col >= p.outer) return;
      make_tile<Quarter, T, ACROSS>(p, t, t.begin + row, t.rows - row < BM / 2 ? t.rows - row : BM / 2, col, s_steps);
      return;
    }
  }
  make_tile<Tile, T, ACROSS>(p, t, t.begin, t.rows < BM ? t.rows : BM, t.col * BN, s_steps);
}

template <typename T, bool ACROSS, int BM, int BN, int WM, int WN, int RING, Way WAY>
int launch_product(ProductArgs<T> p, hipStream_t st) {
  constexpr int threads = WM * WN * kWave;
  p.col_tiles = (p.outer + BN - 1) / BN;
  const int64_t more = BM == 256 && BN == 256 ? products::kCus / 2 * 3 : 0;  // (where some are made in quarters)
  const int64_t blocks = products::blocks_of(products::most_row_tiles(p.n, p.experts, BM), p.col_tiles, more);
  return products::launch_blocks(product_kernel<T, ACROSS, BM, BN, WM, WN, RING, WAY>, p, blocks, threads, "expert_matmul", st);
}

// Large tiles read less, small ones fill the card with less work and waste less of it; chunks that are not aligned come more
// slowly, and make large tiles worth while sooner.  bf16, kernel times of tiles of 256 x 256, 128 x 128, 64 x 128 and 64 x 64, us
// (aligned: 1152 x 896, 336 x 1008 and 152 x 256; not: 1150 x 890 and 333 x 1001):
//   32 experts of 1152 x 896, 1000 rows each 63, 74, 88, 115; 200 rows 31, 26, 29, 44; 40 rows (tiles of 64 x 64 fill the card
//   but twice) 32, 28, 26, 25; of 336 x 1008, 500 rows 29, 28, 33, 44; 5000 rows 204, 236, 287, 348
//   32 of 1150 x 890, 1000 rows 85, 105, 121, 178; 200 rows 33, 31, 35, 51; of 333 x 1001, 1000 rows 53, 60, 70, 84
//   160 of 152 x 256, 100 rows 14, 10, 10, 9
// Where one round of workgroups is all there is, nobody works while one waits, and more steps on their way (a ring of four for 128 x
// 128, five for 64 x 128, six for 64 x 64) hide the rest; otherwise three, which leave room for more workgroups, are better:
//   16 of 1150 x 890, 200 rows, 128 x 128, 18 with four, 27 with three; 64 x 128, 21 with five, 23 with three
//   3 of 1152 x 896, 1000 rows, 64 x 64, 16 with six, 19 with three; 16 of 64 x 128, 5000 rows, 16 and 10
// fp32, which is bound by its products, is within 5 % of its best with the smallest.
template <typename T, bool ACROSS>
int choose_product(const ProductArgs<T>& p, hipStream_t st) {
  if (products::narrow(p, ACROSS)) return products::launch_narrow(p, ACROSS, st);
  if (products::few_rows(p, ACROSS)) return products::launch_few_rows(p, ACROSS, st);
  const Way way = products::slower(products::way_of<T>(p.row_stride, p.inner, 256),
                                   products::way_of<T>(p.weight_stride, ACROSS ? p.outer : p.inner, 256));
  if (way == Way::kValues) return launch_product<T, ACROSS, 64, 64, 2, 2, 3, Way::kValues>(p, st);
  const bool deep = p.inner >= 8 * products::kStep<T>;
  if constexpr (sizeof(T) == 2) {
    const bool aligned = products::aligned_rows(p.rows, p.row_stride, 0) &&
                         products::aligned_rows(p.weight, p.weight_stride, p.expert_stride);
    const int64_t enough = !aligned ? 160 : p.inner >= 512 ? 224 : 600, tiles128 = products::likely_tiles(p, 128, 128);
    if (p.outer > 128 && p.inner >= 256 && p.n >= 128 * p.experts && products::likely_tiles(p, 256, 256) >= enough)
      return launch_product<T, ACROSS, 256, 256, 2, 4, 4, Way::kDirect>(p, st);
    if (p.outer > 64 && deep && tiles128 >= 160 && tiles128 <= products::kCus)
      return launch_product<T, ACROSS, 128, 128, 2, 2, 4, Way::kDirect>(p, st);
    if (p.outer > 64 && p.n >= 64 * p.experts && tiles128 >= 350)
      return launch_product<T, ACROSS, 128, 128, 2, 2, 3, Way::kDirect>(p, st);
    const int64_t tiles = products::likely_tiles(p, 64, 128);
    if (p.outer > 64 && tiles >= 150) {
      return deep && tiles < 2 * products::kCus ? launch_product<T, ACROSS, 64, 128, 2, 2, 5, Way::kDirect>(p, st)
                                                : launch_product<T, ACROSS, 64, 128, 2, 2, 3, Way::kDirect>(p, st);
    }
  }
  return deep && products::likely_tiles(p, 64, 64) <= 4 * products::kCus
             ? launch_product<T, ACROSS, 64, 64, 2, 2, 6, Way::kDirect>(p, st)
             : launch_product<T, ACROSS, 64, 64, 2, 2, 3, Way::kDirect>(p, st);
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
  GS_REQUIRE(num_experts <= products::kMostExperts, "gs_expert_matmul: %lld experts, at most %lld are taken",
             static_cast<long long>(num_experts), static_cast<long long>(products::kMostExperts));
  GS_REQUIRE(row_stride >= 0 && expert_stride >= 0 && weight_stride >= 0, "gs_expert_matmul: negative stride");
  if (n == 0 || outer == 0) return GS_OK;
  GS_REQUIRE(offsets && out && (inner == 0 || (rows && (num_experts == 0 || weight))), "gs_expert_matmul: null array");
  GS_REQUIRE(aligned_to(rows, value_bytes(type)) && aligned_to(weight, value_bytes(type)) && aligned_to(out, value_bytes(type)),
             "gs_expert_matmul: rows or matrices not aligned to their type");
  return with_value_type(type, "gs_expert_matmul", [&](auto zero) {
    using T = decltype(zero);
    const ProductArgs<T> p{static_cast<const T*>(rows), row_stride, n, inner, static_cast<const T*>(weight), expert_stride,
                           weight_stride, num_experts, outer, offsets, static_cast<T*>(out), 0, 0};
    const auto st = static_cast<hipStream_t>(stream);
    return transposed ? choose_product<T, false>(p, st) : choose_product<T, true>(p, st);
  });
}
