// Products of rows sorted by expert with each expert's matrix (gs_expert_products.hip) where experts have few rows, whose tiles would
// not fill the card, or deep matrices, on gfx950: tokens that are being generated.
//
// Every matrix that is met is read once, which bounds them: 30 experts of 4096 x 256, 8 rows each, bf16, 16 us, 3.9
// TB/s, start and end included.  A workgroup takes up to 16 * MI rows of an expert and 16 *
// COLS columns; its waves share out the depth, step by step, each with several steps of the matrix
// on their way to registers, and their sums meet in LDS.  No value goes through LDS on its way in: a lane's chunks
// are what the matrix cores take (along the depth), or become that by exchanging halves of registers (across it).
// No counterpart in the reference.
#include "gs_expert_products.hpp"

namespace gs {
namespace products {
namespace {

constexpr int kWaves = 8, kThreads = kWaves * kWave;

template <typename T, bool ACROSS, int MI, int COLS>
__global__ void __launch_bounds__(kThreads)
few_rows_kernel(ProductArgs<T> p) {
  using S = Slab<T, ACROSS, COLS>;
  constexpr int kVec = S::kVec, kRows = 16 * MI, kDepth = 4;  // steps on their way
  constexpr int kPad = S::kWide + 4;
  __shared__ __attribute__((aligned(16))) float s_sums[kWaves][kRows][kPad];
  RowTile t = find_tile<kThreads>(p.offsets, p.experts, p.n, kRows, p.col_tiles, p.first_block);
  if (t.rows <= 0) return;
  t = {uniform(t.expert), uniform(t.begin), uniform(t.rows), uniform(t.col), -1};
  const int lane = threadIdx.x % kWave, row16 = lane % 16, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t rows = t.rows < kRows ? t.rows : kRows;
  const bool live = t.expert < p.experts;
  const int64_t inner = live ? p.inner : 0, whole = inner / kStep<T>;
  // The last tile of columns ends where the matrix does, and so do a narrow matrix's last lanes: columns that they share with
  // others come out the same.
  const int64_t col = t.col * S::kWide + S::kWide <= p.outer ? t.col * S::kWide : (p.outer > S::kWide ? p.outer - S::kWide : 0);

  // where the lane's chunks of step 0 begin
  const T* const w = p.weight + (live ? t.expert * p.expert_stride : 0);
  const T* from[ACROSS ? 1 : COLS];
  const int64_t most = p.outer - COLS - col;
  const int first = ACROSS && row16 * COLS > most ? static_cast<int>(most) : row16 * COLS;  // the lane's columns, across
  if (ACROSS) {
    from[0] = w + quarter * kVec * p.weight_stride + col + first;
  } else {
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const int64_t n = col + c * 16 + row16;
      from[ACROSS ? 0 : c] = w + (n < p.outer ? n : p.outer - 1) * p.weight_stride + quarter * kVec;
    }
  }
  const T* x[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int64_t m = i * 16 + row16;
    x[i] = p.rows + (t.begin + (m < rows ? m : rows - 1)) * p.row_stride + quarter * kVec;
  }

  S slab[kDepth];
  Values<T> a[kDepth][MI];
  auto load = [&](S& to, Values<T>* rows_to, int64_t step) {
    const int64_t k = step * kStep<T>;
    if constexpr (ACROSS) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) __builtin_memcpy(&to.held[j], from[0] + (k + j) * p.weight_stride, sizeof(typename S::Piece));
    } else {
#pragma unroll
      for (int c = 0; c < COLS; ++c) __builtin_memcpy(&to.held[c], from[c] + k, 16);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) __builtin_memcpy(&rows_to[i], x[i] + k, 16);
  };
  Acc acc[MI][COLS];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int c = 0; c < COLS; ++c) acc[i][c] = Acc{};
  auto work = [&](const S& s, const Values<T>* r) {
#pragma unroll
    for (int c = 0; c < COLS; ++c) {
      const Values<T> b = s.fragment(c);
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[i][c] = multiply(r[i], b, acc[i][c]);
    }
  };

  // the wave's steps: wave, wave + kWaves, ..
  const int64_t count = whole > wave ? (whole - wave + kWaves - 1) / kWaves : 0;
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (d < count) load(slab[d], a[d], wave + d * kWaves);
  int64_t i = 0;
  for (; i + 2 * kDepth <= count; i += kDepth) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      work(slab[d], a[d]);
      load(slab[d], a[d], wave + (i + kDepth + d) * kWaves);
    }
  }
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    if (i + d < count) work(slab[d], a[d]);
    if (i + kDepth + d < count) load(slab[d], a[d], wave + (i + kDepth + d) * kWaves);
  }
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (i + kDepth + d < count) work(slab[d], a[d]);
  // what is left of the depth, value by value, by the wave whose turn it is
  const int64_t k = whole * kStep<T>;
  if (k < inner && wave == static_cast<int>(whole % kWaves)) {
    S s;
    Values<T> r[MI];
    const int64_t left = inner - k - quarter * kVec;
    if constexpr (ACROSS) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        s.held[j] = typename S::Piece{};
        if (j < left) __builtin_memcpy(&s.held[j], from[0] + (k + j) * p.weight_stride, sizeof(typename S::Piece));
      }
    } else {
#pragma unroll
      for (int c = 0; c < COLS; ++c) s.held[c] = load_part(from[c] + k, left);
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) r[m] = load_part(x[m] + k, left);
    work(s, r);
  }

  // lane l has rows (l / 16) * 4 .. + 3 of each 16, and the columns of its fragments
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int c = 0; c < COLS; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        s_sums[wave][m * 16 + quarter * 4 + j][ACROSS ? first + c : c * 16 + row16] = acc[m][c][j];
  __syncthreads();
  typedef T Four __attribute__((ext_vector_type(4)));
  for (int q = threadIdx.x; q < kRows * (S::kWide / 4); q += kThreads) {
    const int m = q / (S::kWide / 4), n = q % (S::kWide / 4) * 4;
    if (m >= rows) continue;
    Acc sum = *reinterpret_cast<const Acc*>(&s_sums[0][m][n]);
#pragma unroll
    for (int v = 1; v < kWaves; ++v) sum += *reinterpret_cast<const Acc*>(&s_sums[v][m][n]);
    store_part(p.out + (t.begin + m) * p.outer + col + n, __builtin_convertvector(sum, Four), p.outer - col - n);
  }
}

template <typename T, bool ACROSS, int MI, int COLS>
int launch(ProductArgs<T> p, hipStream_t st) {
  p.col_tiles = (p.outer + 16 * COLS - 1) / (16 * COLS);
  const int64_t blocks = blocks_of(most_row_tiles(p.n, p.experts, 16 * MI), p.col_tiles);
  return launch_blocks(few_rows_kernel<T, ACROSS, MI, COLS>, p, blocks, kThreads, "expert_matmul", st);
}

}  // namespace

// Twice the rows where experts have more than 16, and twice the columns with 16-bit values, whose loads are wider then, where there
// are workgroups enough; half the columns where they would fill the card but once, since a workgroup's own loads bound it then,
// and its products in fp32, most of whose rows are missing where experts have one or two.  Kernel times, us: 32 experts of 1024 x 1024,
// bf16, a row each, 128 columns 11, 64 15; of 4096 x 512 26 and 22; 8 of 4096 x 1024, 2 rows, 64 columns 16 to 20, 32 15; 4 of
// 3496 x 72, 40 rows (32 at once) 16 to 18, 64 columns of 16 rows 13 to 16, 32 9 to 11; fp32 39 to 50, 25 to 33, 17 to 20; 160 of 1001 x 333,
// a row each, fp32 35 to 44 and 31 to 35.
template <typename T>
int launch_few_rows(const ProductArgs<T>& p, bool across, hipStream_t st) {
  auto go = [&](auto mi, auto cols) {
    constexpr int MI = decltype(mi)::value, COLS = decltype(cols)::value;
    return across ? launch<T, true, MI, COLS>(p, st) : launch<T, false, MI, COLS>(p, st);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  if (likely_tiles(p, 16, 32) <= kCus || (sizeof(T) == 4 && p.n <= 2 * p.experts)) return go(One(), Two());
  if (likely_tiles(p, 16, 64) <= kCus) return go(One(), Four());
  auto with_rows = [&](auto mi) {
    constexpr int MI = decltype(mi)::value;
    if constexpr (sizeof(T) == 2) {  // (twice of both along the depth is more than the registers hold)
      const bool many = likely_tiles(p, 16 * MI, 64) >= 320;
      if (many && across) return launch<T, true, MI, 8>(p, st);
      if constexpr (MI == 1) {
        if (many) return launch<T, false, MI, 8>(p, st);
      }
    }
    return go(mi, Four());
  };
  if (p.n > 16 * p.experts) return with_rows(Two());
  return with_rows(One());
}
template int launch_few_rows<float>(const ProductArgs<float>&, bool, hipStream_t);
template int launch_few_rows<_Float16>(const ProductArgs<_Float16>&, bool, hipStream_t);
template int launch_few_rows<__bf16>(const ProductArgs<__bf16>&, bool, hipStream_t);

}  // namespace products
}  // namespace gs
