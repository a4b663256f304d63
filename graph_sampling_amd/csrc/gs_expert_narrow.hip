// Products of rows sorted by expert with each expert's matrix (gs_expert_products.hip) where matrices are small, or low, and
// rows many, on gfx950: the types of the nodes of a frontier.
//
// Rows bound them, in and out.  A wave holds an expert's matrix (up to 128 columns of it) in registers, as what
// the matrix cores take, and streams rows past it, 16 at a time, several of those on their way; nothing goes through LDS.  One
// round of workgroups: each has its share of all rows.  600 000 rows x 64 x 128 of 5 types, fp32: 123 us (64 x 64 tiles 178; 461 MB
// at 3.7 TB/s), the products with the matrices transposed 141; the fp32 products alone, at the rate of a large library
// product, are 64 us of either, and do not hide all of the reads.  No counterpart in the reference.
#include "gs_expert_products.hpp"

namespace gs {
namespace products {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;

// Workgroups a compute unit: what the matrix leaves of the registers.
constexpr int resident(int steps, int fragments) { return steps * fragments >= 32 ? 1 : 2; }
constexpr int kAhead = 4;  // strips on their way

// Every workgroup writes its share of `many` zeros.
template <typename T>
__device__ __forceinline__ void zero(T* out, int64_t many) {
  constexpr int kVec = Chunk<T>::kVec;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kVec; at < many; at += threads * kVec)
    store_part(out + at, Values<T>{}, many - at);
}

// STEPS: of the depth, at least as many as there are; SLABS slabs of COLS * 16 columns
template <typename T, bool ACROSS, int STEPS, int COLS, int SLABS>
__global__ void __launch_bounds__(kThreads, resident(STEPS, COLS* SLABS))
narrow_kernel(ProductArgs<T> p, int shares) {
  constexpr int kVec = Chunk<T>::kVec, kWide = 16 * COLS, kFrags = COLS * SLABS;
  const int64_t live = inside(p.offsets[p.experts], p.n);
  zero(p.out + live * p.outer, (p.n - live) * p.outer);
  const int64_t each = (live + shares - 1) / shares;
  const int tile_rows = each > 0 ? static_cast<int>((each + 16 * kWaves - 1) / (16 * kWaves) * (16 * kWaves)) : 16 * kWaves;
  RowTile t = find_tile<kThreads>(p.offsets, p.experts, live, tile_rows, p.col_tiles);
  if (t.rows <= 0) return;
  t = {uniform(t.expert), uniform(t.begin), uniform(t.rows), uniform(t.col), -1};
  const int lane = threadIdx.x % kWave, row16 = lane % 16, quarter = lane / 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int rows = static_cast<int>(t.rows < tile_rows ? t.rows : tile_rows);
  const int inner = static_cast<int>(p.inner), steps = (inner + kStep<T> - 1) / kStep<T>;
  const int64_t col = t.col * (kWide * SLABS);

  // the matrix
  Values<T> b[STEPS][kFrags];
  int first[SLABS];  // the lane's columns of a slab, across the depth
  const T* const w = p.weight + t.expert * p.expert_stride;
#pragma unroll
  for (int s = 0; s < SLABS; ++s) {
    const int64_t most = p.outer - COLS - col - s * kWide;  // (a slab's last lanes end where the matrix does; behind it, none)
    first[s] = row16 * COLS > most ? static_cast<int>(most) : row16 * COLS;
  }
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    const int left = inner - k * kStep<T> - quarter * kVec;
#pragma unroll
    for (int s = 0; s < SLABS; ++s) {
      if constexpr (ACROSS) {
        Slab<T, true, COLS> slab;
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          slab.held[j] = typename Slab<T, true, COLS>::Piece{};
          const T* const from = w + (k * kStep<T> + quarter * kVec + j) * p.weight_stride + col + s * kWide + first[s];
          if (j < left && col + s * kWide + first[s] >= 0) __builtin_memcpy(&slab.held[j], from, sizeof(slab.held[j]));
        }
#pragma unroll
        for (int c = 0; c < COLS; ++c) b[k][s * COLS + c] = slab.fragment(c);
      } else {
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
          const int64_t n = col + (s * COLS + c) * 16 + row16;
          b[k][s * COLS + c] = load_part(w + (n < p.outer ? n : p.outer - 1) * p.weight_stride + k * kStep<T> + quarter * kVec, left);
        }
      }
    }
  }

  // the wave's strips: wave, wave + kWaves, ..
  const int strips = (rows + 15) / 16, count = strips > wave ? (strips - wave + kWaves - 1) / kWaves : 0;
  // (chunks that end behind the depth are read from as far in front of it as they lack, and shifted when they are used)
  const bool ragged = inner % kStep<T> != 0;
  int at[STEPS], lack = 0;
#pragma unroll
  for (int k = 0; k < STEPS; ++k) {
    at[k] = k * kStep<T> + quarter * kVec;
    const int over = at[k] + kVec - inner;
    if (over > 0) at[k] -= over < at[k] ? over : at[k];
    if (k == steps - 1) lack = over > 0 ? over : 0;
  }
  const T* const x = p.rows + t.begin * p.row_stride;
  Values<T> a[kAhead][STEPS];
  auto load = [&](Values<T>* to, int i) {
    const int m = (wave + i * kWaves) * 16 + row16;
    const T* const from = x + static_cast<int64_t>(m < rows ? m : rows - 1) * p.row_stride;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) __builtin_memcpy(&to[k], from + at[k], 16);
  };
  T* const out = p.out + t.begin * p.outer + col;
  auto work = [&](const Values<T>* from, int i) {
    Acc acc[kFrags];
#pragma unroll
    for (int c = 0; c < kFrags; ++c) acc[c] = Acc{};
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (k < steps) {
        Values<T> v = from[k];
        if (ragged && k == steps - 1) v = lack < kVec ? shifted<T>(v, lack) : Values<T>{};
#pragma unroll
        for (int c = 0; c < kFrags; ++c) acc[c] = ACROSS ? multiply(v, b[k][c], acc[c]) : multiply(b[k][c], v, acc[c]);
      }
    }
    const int strip = (wave + i * kWaves) * 16;
    if constexpr (ACROSS) {  // rows quarter * 4 + j, the lane's columns
      typedef T Out __attribute__((ext_vector_type(COLS)));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int m = strip + quarter * 4 + j;
        if (m >= rows) continue;
#pragma unroll
        for (int s = 0; s < SLABS; ++s) {
          Out v;
#pragma unroll
          for (int c = 0; c < COLS; ++c) v[c] = static_cast<T>(acc[s * COLS + c][j]);
          if (col + s * kWide + first[s] >= 0 && s * kWide < p.outer - col)
            __builtin_memcpy(out + static_cast<int64_t>(m) * p.outer + s * kWide + first[s], &v, sizeof(v));
        }
      }
    } else {  // row row16, columns c * 16 + quarter * 4 ..
      write_row<kFrags>(acc, out + static_cast<int64_t>(strip + row16) * p.outer, strip + row16 < rows ? p.outer - col : 0);
    }
  };
#pragma unroll
  for (int d = 0; d < kAhead; ++d)
    if (d < count) load(a[d], d);
  int i = 0;
  for (; i + 2 * kAhead <= count; i += kAhead) {
#pragma unroll
    for (int d = 0; d < kAhead; ++d) {
      work(a[d], i + d);
      load(a[d], i + kAhead + d);
    }
  }
#pragma unroll
  for (int d = 0; d < kAhead; ++d) {
    if (i + d < count) work(a[d], i + d);
    if (i + kAhead + d < count) load(a[d], i + kAhead + d);
  }
#pragma unroll
  for (int d = 0; d < kAhead; ++d)
    if (i + kAhead + d < count) work(a[d], i + kAhead + d);
}

template <typename T, bool ACROSS, int STEPS, int COLS, int SLABS>
int launch(ProductArgs<T> p, hipStream_t st) {
  p.col_tiles = (p.outer + 16 * COLS * SLABS - 1) / (16 * COLS * SLABS);
  const int64_t shares = kCus * resident(STEPS, COLS * SLABS) / p.col_tiles - p.experts - 1;
  const int64_t blocks = blocks_of(shares + p.experts, p.col_tiles);  // (a part of a share for every expert)
  GS_RETURN_IF_ERROR(check_grid("gs_expert_matmul", blocks, kThreads));
  hipLaunchKernelGGL((narrow_kernel<T, ACROSS, STEPS, COLS, SLABS>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, p,
                     static_cast<int>(shares));
  return check_launch("expert_matmul");
}

}  // namespace

// What a matrix takes of the registers decides on columns: 128 of them a wave are 128 registers at 256 bytes of depth, 64 at
// 512.
template <typename T>
int launch_narrow(const ProductArgs<T>& p, bool across, hipStream_t st) {
  const int64_t steps = (p.inner + kStep<T> - 1) / kStep<T>;
  auto go = [&](auto of_depth, auto cols, auto slabs) {
    constexpr int STEPS = decltype(of_depth)::value, COLS = decltype(cols)::value, SLABS = decltype(slabs)::value;
    return across ? launch<T, true, STEPS, COLS, SLABS>(p, st) : launch<T, false, STEPS, COLS, SLABS>(p, st);
  };
  using One = std::integral_constant<int, 1>;
  using Two = std::integral_constant<int, 2>;
  using Four = std::integral_constant<int, 4>;
  using Eight = std::integral_constant<int, 8>;
  constexpr bool kHalf = sizeof(T) == 2;
  if (p.outer > 64 && steps <= 4) {
    using Cols = std::conditional_t<kHalf, Eight, Four>;
    using Slabs = std::conditional_t<kHalf, One, Two>;
    return steps <= 2 ? go(Two(), Cols(), Slabs()) : go(Four(), Cols(), Slabs());
  }
  return steps <= 2 ? go(Two(), Four(), One()) : steps <= 4 ? go(Four(), Four(), One()) : go(Eight(), Four(), One());
}
template int launch_narrow<float>(const ProductArgs<float>&, bool, hipStream_t);
template int launch_narrow<_Float16>(const ProductArgs<_Float16>&, bool, hipStream_t);
template int launch_narrow<__bf16>(const ProductArgs<__bf16>&, bool, hipStream_t);

}  // namespace products
}  // namespace gs
