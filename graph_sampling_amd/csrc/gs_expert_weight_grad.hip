// Gradients of the experts' matrices (gs_expert_products.hip), on gfx950.
//
//   dweight[e] = sum over the rows p of expert e of rows[p, :]^T * grad[p, :],   zeros for an expert without rows
//
// Products whose depth is an expert's number of rows.  8 experts of 4096 x 2048, 2000 rows each, bf16: 264 us, 1.02 PFLOP/s, bound
// as large products of rows are; 5 types of 64 x 128, 120 000 rows each, fp32: 120 us in 610 pieces and 7 to join them, 3.8 TB/s
// with the matrix cores half busy.  No counterpart in the reference.
#include <cmath>

#include "gs_products.hpp"

namespace gs {
namespace {

using products::Group;
using products::Operand;
using products::Way;

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
  // where the rows are cut into pieces of `piece` for the sake of more workgroups: the sums of each
  float* sums;
  int64_t piece;
  int64_t first_block;  // of the launch
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

// Whether every die has its share of each expert's tiles.  Experts by the die have their rows read by one of them, and leave
// dies idle whose experts have few; of few experts, or many tiles, that is worse.  bf16, shares and whole experts, us: 8 experts of
// 4096 x 2048, 2000 rows each 254 and 290; 32 of 250 x 1150, 500 rows 29 and 22; of 2048 x 1024, 200 rows 52 and 58; 160 of
// 336 x 1008, 200 rows 70 and 48.
__host__ __device__ __forceinline__ bool shares(int64_t in_expert, int64_t experts) {
  return in_expert >= (experts < 24 ? 2 * kXcds : 100);
}

template <typename T, int BM, int BN, int WM, int WN, int RING, Way WAY, bool PIECES>
__global__ void __launch_bounds__(WM * WN * kWave)
weight_grad_kernel(WeightGradArgs<T> p) {
  using Tile = products::Tile<T, true, true, BM, BN, WM, WN, RING, WAY>;
  __shared__ __attribute__((aligned(1024))) char s_steps[Tile::kBytes];
  // Workgroups of one die make tiles that share rows: neighbours of one expert, or piece.  Which die has an expert, or a part
  // of each, is `shares`.
  // (behind the last expert's rows there are no pieces)
  const int64_t live = PIECES ? products::inside(p.offsets[p.experts], p.n) : 0;
  const int64_t pieces = live > 0 ? (live - 1) / p.piece + p.experts : 0;
  const int64_t in_expert = p.row_tiles * p.col_tiles, all = in_expert * (PIECES ? pieces : p.experts);
  const int64_t die = blockIdx.x % kXcds, slot = (p.first_block + blockIdx.x) / kXcds;
  int64_t which;
  if (shares(in_expert, p.experts)) {
    const int64_t share = (in_expert + kXcds - 1) / kXcds, nth = die * share + slot % share;
    which = nth < in_expert ? slot / share * in_expert + nth : all;
  } else {
    const int64_t per_die = (all + kXcds - 1) / kXcds;
    which = slot < per_die ? die * per_die + slot : all;
  }
  if (which >= all) return;
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

// dweight[e] = the sums of its pieces: 16 lanes a run of 64 values, SLICES of them an expert's pieces, slice by slice, the
// slices one after the other.
constexpr int kThreads = 256;
template <typename T, int SLICES>
__global__ void __launch_bounds__(kThreads)
join_pieces_kernel(WeightGradArgs<T> p, int64_t runs) {
  constexpr int kRuns = kThreads / 16 / SLICES;  // of a workgroup
  typedef float Four __attribute__((ext_vector_type(4)));
  typedef T Narrow __attribute__((ext_vector_type(4)));
  __shared__ Four s_sums[SLICES][kRuns * 16];
  const int in_run = threadIdx.x % (kRuns * 16), slice = threadIdx.x / (kRuns * 16);
  const int64_t size = p.inner * p.outer, chunk = static_cast<int64_t>(blockIdx.x) * (kRuns * 16) + in_run;
  const int64_t e = chunk / (runs * 16), at = (chunk - e * (runs * 16)) * 4, there = e < p.experts ? size - at : 0;
  Four sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (there > 0) {
    const Pieces of = pieces_of(products::group_of(p.offsets, p.experts, p.n, e), e, p.piece);
    const int64_t many = of.last < of.first ? 0 : of.last - of.first + 1, each = (many + SLICES - 1) / SLICES;
    const int64_t first = of.first + slice * each, end = first + each <= of.last ? first + each : of.last + 1;
    const float* from = p.sums + at;
#pragma unroll 4
    for (int64_t q = first; q < end; ++q) {
      Four v;
      if (there >= 4) {
        __builtin_memcpy(&v, from + q * size, 16);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < there ? from[q * size + i] : 0.0f;
      }
      sum += v;
    }
  }
  s_sums[slice][in_run] = sum;
  __syncthreads();
  if (slice != 0 || there <= 0) return;
#pragma unroll
  for (int k = 1; k < SLICES; ++k) sum += s_sums[k][in_run];
  products::store_part(p.out + e * size + at, __builtin_convertvector(sum, Narrow), there);
}

// How the rows are cut: not at all (0) where there are tiles enough, or where pieces would not be much shorter.  A piece of R rows
// keeps a workgroup busy for R / 100 us or so, and its sums are written and read, 8 bytes each at 4 TB/s: the two together are
// least at R^2 = n * inner * outer / 5000.  No more pieces than give 2048 small tiles: by then the card is full.  With three experts or
// less an uncut one takes its rows' time, with more the largest one's, which has twice the others' or so.  bf16, us: 2 experts of 512 x 512,
// 1000 rows each, uncut 11, pieces of 256 17, of 128 20; 2000 rows 33, 17 (of 512), 30 (of 128); 32 of 256 x 256, 300 rows 8 uncut,
// 27 in pieces of 128, 2000 rows 62 and 36 (of 512); 5 of 64 x 128, 120 000 rows, pieces of 608 56, of 1184 43.
constexpr int64_t tiles_of(int64_t inner, int64_t outer) { return (inner + 63) / 64 * ((outer + 63) / 64); }
int64_t piece_rows(int64_t n, int64_t experts, int64_t inner, int64_t outer) {
  constexpr int64_t kTiles = 2048, kRows = 128;
  const int64_t tiles = tiles_of(inner, outer);
  if (tiles * experts >= kTiles / 2 || n < 2 * kRows * experts) return 0;
  const int64_t full = (n * tiles + kTiles - 1) / kTiles;
  const int64_t least = static_cast<int64_t>(std::sqrt(static_cast<double>(n) * static_cast<double>(inner * outer) / 5000.0));
  const int64_t rows = least > full ? least : full;
  if (10 * n < (experts < 4 ? 32 : 19) * rows * experts) return 0;
  return rows < kRows ? kRows : (rows + 31) / 32 * 32;
}
int64_t pieces_there(int64_t n, int64_t experts, int64_t piece) { return (n + piece - 1) / piece + experts; }

template <typename T, int SLICES>
int launch_join(const WeightGradArgs<T>& p, hipStream_t st) {
  const int64_t runs = (p.inner * p.outer + 63) / 64, a_block = kThreads / 16 / SLICES;
  const int64_t blocks = (p.experts * runs + a_block - 1) / a_block;
  GS_RETURN_IF_ERROR(check_grid("gs_expert_matmul_grad", blocks, kThreads));
  hipLaunchKernelGGL((join_pieces_kernel<T, SLICES>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, p, runs);
  return check_launch("expert_matmul_grad");
}

// CUT: whether the rows can be in pieces (which have 128 rows at least, as the experts have then: a tile for fewer makes whole ones).
template <typename T, int BM, int BN, int WM, int WN, int RING, Way WAY, bool CUT = true>
int launch_weight_grad(WeightGradArgs<T> p, void* workspace, size_t workspace_bytes, hipStream_t st) {
  constexpr int threads = WM * WN * kWave;
  p.row_tiles = (p.inner + BM - 1) / BM;
  p.col_tiles = (p.outer + BN - 1) / BN;
  const int64_t tiles = p.row_tiles * p.col_tiles;
  p.piece = piece_rows(p.n, p.experts, p.inner, p.outer);
  const int64_t items = p.piece ? pieces_there(p.n, p.experts, p.piece) : p.experts;
  const int64_t padded_tiles = shares(tiles, p.experts) ? (tiles + kXcds - 1) / kXcds * kXcds : tiles;
  const int64_t blocks = (items * padded_tiles + kXcds - 1) / kXcds * kXcds;
  if (!CUT || !p.piece)
    return products::launch_blocks(weight_grad_kernel<T, BM, BN, WM, WN, RING, WAY, false>, p, blocks, threads, "expert_matmul_grad", st);
  if constexpr (CUT) {
    Carver ws(workspace, workspace_bytes);
    p.sums = ws.take<float>(static_cast<size_t>(items * p.inner * p.outer));
    if (!ws.ok) {
      set_error_text("gs_expert_matmul_grad: workspace needs %zu bytes, 256-byte aligned",
                     gs_expert_matmul_grad_workspace_bytes(p.n, p.inner, p.outer, p.experts));
      return GS_ERR_WORKSPACE;
    }
    GS_RETURN_IF_ERROR(
        products::launch_blocks(weight_grad_kernel<T, BM, BN, WM, WN, RING, WAY, true>, p, blocks, threads, "expert_matmul_grad", st));
    return items > 16 * p.experts ? launch_join<T, 16>(p, st) : launch_join<T, 4>(p, st);
  }
}

// As for the products of rows; here a matrix, or what a piece adds to it, is a product of its own, and one of few rows is not
// worth a large tile's start and end, nor a deep ring's.  bf16, tiles of 256 x 256, 128 x 128 (ring of four, and of three), 64 x 128
// (five) and 64 x 64 (six), us: 32 experts of 1024 x 1024, 2000 rows each 164, -, 217, -, 371; 60 of 1152 x 896, 300 rows 72, 64, 61,
// 84, 93; 16 of 1150 x 890, 1000 rows 63, 50, 50, 64, 84; 60 of 336 x 1008, 500 rows 50, 42, 45, 55, 71; 3 of 1152 x 896, 1000 rows
// 31, 15, 23, 13, 14, 2000 rows 57, 26, 44, 20, 22; 4 of 333 x 1001 (not aligned), 40 000 rows 209, -, 307, -, 545.  fp32 is within 12 %
// of its best with the smallest; 64 of 256 x 256, 2000 rows 184 with a ring of six, 271 with three.
template <typename T>
int choose_weight_grad(const WeightGradArgs<T>& p, void* workspace, size_t workspace_bytes, hipStream_t st) {
  const Way way = products::slower(products::way_of<T>(p.row_stride, p.inner, 256), products::way_of<T>(p.grad_stride, p.outer, 256));
  if (way == Way::kValues) return launch_weight_grad<T, 64, 64, 2, 2, 3, Way::kValues>(p, workspace, workspace_bytes, st);
  const int64_t piece = piece_rows(p.n, p.experts, p.inner, p.outer), each = p.n / p.experts;
  const int64_t items = piece ? pieces_there(p.n, p.experts, piece) : p.experts, rows = piece && piece < each ? piece : each;
  const auto tiles = [&](int64_t rows_of, int64_t cols_of) {
    return (p.inner + rows_of - 1) / rows_of * ((p.outer + cols_of - 1) / cols_of) * items;
  };
  if constexpr (sizeof(T) == 2) {
    if (p.inner > 128 && p.outer > 128 && rows >= 300 && tiles(256, 256) >= (piece ? 128 : 600))
      return launch_weight_grad<T, 256, 256, 2, 4, 4, Way::kDirect>(p, workspace, workspace_bytes, st);
    if (p.inner > 64 && p.outer > 64 && tiles(128, 128) >= 250)
      return rows >= 128 ? launch_weight_grad<T, 128, 128, 2, 2, 4, Way::kDirect>(p, workspace, workspace_bytes, st)
                         : launch_weight_grad<T, 128, 128, 2, 2, 3, Way::kDirect, false>(p, workspace, workspace_bytes, st);
    if (p.outer > 64 && rows >= 128 && tiles(64, 128) >= 140 && tiles(64, 128) <= 512)
      return launch_weight_grad<T, 64, 128, 2, 2, 5, Way::kDirect>(p, workspace, workspace_bytes, st);
  }
  return rows >= (sizeof(T) == 2 ? 200 : 128) && tiles(64, 64) <= 1024
             ? launch_weight_grad<T, 64, 64, 2, 2, 6, Way::kDirect>(p, workspace, workspace_bytes, st)
             : launch_weight_grad<T, 64, 64, 2, 2, 3, Way::kDirect>(p, workspace, workspace_bytes, st);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

size_t gs_expert_matmul_grad_workspace_bytes(int64_t n, int64_t inner, int64_t outer, int64_t num_experts) {
  constexpr int64_t kMost = int64_t(1) << 24;
  if (n <= 0 || n >= (int64_t(1) << 31) || inner <= 0 || inner >= kMost || outer <= 0 || outer >= kMost || num_experts <= 0 ||
      num_experts > products::kMostExperts)
    return 256;
  const int64_t piece = piece_rows(n, num_experts, inner, outer);
  return piece ? padded(static_cast<size_t>(pieces_there(n, num_experts, piece) * inner * outer) * sizeof(float)) : 256;
}

int gs_expert_matmul_grad(const void* rows, int64_t row_stride, int64_t inner, const void* grad, int64_t grad_stride,
                          int64_t outer, int type, int64_t n, const int64_t* offsets, int64_t num_experts, void* dweight,
                          void* workspace, size_t workspace_bytes, void* stream) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16,
             "gs_expert_matmul_grad: value type %d is none of GS_F32, GS_F16, GS_BF16", type);
  GS_REQUIRE(n >= 0 && inner >= 0 && outer >= 0 && num_experts >= 0, "gs_expert_matmul_grad: negative size");
  GS_REQUIRE(n < (int64_t(1) << 31), "gs_expert_matmul_grad: %lld rows, at most 2^31 - 1 are taken",
             static_cast<long long>(n));
  GS_REQUIRE(inner < (int64_t(1) << 24) && outer < (int64_t(1) << 24),
             "gs_expert_matmul_grad: rows of %lld and %lld values, at most 2^24 - 1 are taken",
             static_cast<long long>(inner), static_cast<long long>(outer));
  GS_REQUIRE(num_experts <= products::kMostExperts, "gs_expert_matmul_grad: %lld experts, at most %lld are taken",
             static_cast<long long>(num_experts), static_cast<long long>(products::kMostExperts));
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
