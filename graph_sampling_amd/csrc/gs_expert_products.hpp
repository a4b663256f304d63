// Products of rows sorted by expert: what the kernels for many rows and those for few share.
#pragma once

#include "gs_products.hpp"

namespace gs {
namespace products {

// Which tile of rows a workgroup makes: the tiles of all experts side by side, then those of the rows behind the last.
struct RowTile {
  int64_t expert, begin;  // of the tile's rows
  int64_t rows;           // up to the expert's last; none: no tile
  int64_t col;            // which tile of columns
  int64_t quarter;        // of the tile, or -1: the whole of it
};

constexpr int64_t kCus = 256;  // workgroups of large tiles that run at once

// Every thread counts the tiles of rows of its share of the experts; the one in whose share the workgroup's lies finds it.
// Workgroups of one die take tiles that lie side by side, so that its cache holds what they share.  QUARTERS: tiles that
// would fill less than half of the card, after all others have filled it, are made in quarters.  The rows behind the last come
// after all of these, so that every die has its share of the work.
template <int THREADS, bool QUARTERS = false>
__device__ __forceinline__ RowTile find_tile(const int64_t* __restrict__ offsets, int64_t experts, int64_t n, int tile_rows,
                                             int64_t col_tiles, int64_t first_block = 0) {
  __shared__ int64_t s_wave[THREADS / kWave];
  __shared__ RowTile s_found;
  const int64_t each = (experts + THREADS - 1) / THREADS, first = each * threadIdx.x;
  const int64_t last = first + each < experts ? first + each : experts;
  int64_t mine = 0;
  for (int64_t e = first; e < last; ++e)
    mine += (group_of(offsets, experts, n, e).rows() + tile_rows - 1) / tile_rows;
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
  // blocks of whole tiles, of quarters, of the rows behind
  const Group behind = group_of(offsets, experts, n, experts);
  const int64_t tiles = total * col_tiles, rest = QUARTERS && tiles % kCus <= kCus / 2 ? tiles % kCus : 0, whole = tiles - rest;
  const int64_t whole_blocks = (whole + kXcds - 1) / kXcds * kXcds, part_blocks = (rest * 4 + kXcds - 1) / kXcds * kXcds;
  int64_t block = first_block + blockIdx.x, many = whole;
  bool part = false, dead = false;
  if (block >= whole_blocks) {
    block -= whole_blocks;
    part = block < part_blocks;
    dead = !part;
    if (dead) block -= part_blocks;
    many = part ? rest * 4 : (behind.rows() + tile_rows - 1) / tile_rows * col_tiles;
  }
  const int64_t per_die = (many + kXcds - 1) / kXcds, slot = block / kXcds, nth = block % kXcds * per_die + slot;
  const int64_t which = part ? whole + nth / 4 : nth, at = which / col_tiles;
  if (slot < per_die && nth < many) {
    int64_t from = upto - mine;
    if (dead) {
      if (threadIdx.x == 0) s_found = {experts, behind.begin + at * tile_rows, behind.rows() - at * tile_rows, 0, 0};
    } else if (at >= from && at < upto) {
      for (int64_t e = first; e < last; ++e) {
        const Group g = group_of(offsets, experts, n, e);
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
  }
  __syncthreads();
  RowTile t = s_found;
  t.col = which % col_tiles;
  t.quarter = part ? nth % 4 : -1;
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
  int64_t first_block;  // of the launch
};

// Tiles of rows that there can be: a part of one for every expert that has rows, and for the rows behind.
inline int64_t most_row_tiles(int64_t n, int64_t experts, int64_t tile_rows) {
  return n / tile_rows + (experts + 1 < n ? experts + 1 : n);
}
// Workgroups for them; more: where some are made in quarters.
inline int64_t blocks_of(int64_t row_tiles, int64_t col_tiles, int64_t more = 0) {
  return (row_tiles * col_tiles + more + kXcds - 1) / kXcds * kXcds + 2 * kXcds;
}
// Tiles that there will be, more or less: half a tile of rows for every expert is not full.
template <typename T>
int64_t likely_tiles(const ProductArgs<T>& p, int64_t tile_rows, int64_t tile_cols) {
  const int64_t some = p.n < p.experts ? p.n : p.experts, full = p.n / tile_rows + some / 2;
  return (full > some ? full : some) * ((p.outer + tile_cols - 1) / tile_cols);
}

// A step of 16 * COLS columns of a matrix: what a lane holds of it.
//   across the depth: column group l % 16, kVec rows of k from (l / 16) * kVec on, COLS values of each
//   along the depth: columns l % 16 of kFrags groups of 16, kVec values of k from (l / 16) * kVec on
template <typename T, bool ACROSS, int COLS>
struct Slab {
  static constexpr int kVec = Chunk<T>::kVec;
  static constexpr int kLoads = ACROSS ? kVec : COLS;  // (COLS fragments)
  static constexpr int kWide = 16 * COLS;              // columns
  typedef T Piece __attribute__((ext_vector_type(ACROSS ? COLS : kVec)));
  Piece held[kLoads];

  // The fragment of columns (l % 16) * COLS + c, or c * 16 + l % 16.
  __device__ __forceinline__ Values<T> fragment(int c) const {
    if constexpr (!ACROSS) {
      return held[c];
    } else if constexpr (sizeof(T) == 4) {
      return Values<T>{held[0][c], held[1][c], held[2][c], held[3][c]};
    } else {
      typedef uint32_t Words __attribute__((ext_vector_type(COLS / 2)));
      union {
        uint32_t word[4];
        Values<T> v;
      } u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t low = __builtin_bit_cast(Words, held[2 * i])[c / 2], high = __builtin_bit_cast(Words, held[2 * i + 1])[c / 2];
        u.word[i] = __builtin_amdgcn_perm(high, low, c % 2 ? 0x07060302u : 0x05040100u);
      }
      return u.v;
    }
  }
};

// The products of experts with few rows each (gs_expert_few_rows.hip), and whether they are such.
template <typename T>
int launch_few_rows(const ProductArgs<T>& p, bool across, hipStream_t st);

// The products with small matrices (gs_expert_narrow.hip), and whether they are such: a wave's registers hold one, and each
// workgroup of one round has rows enough to make up for fetching it.  Kernel times of this and of tiles, us: bf16, 5 experts
// of 100 x 128, 150 000 rows 18 and 27, 700 000 rows 64 and 123; 64 x 128, 150 000 rows 17 and 17, transposed, 300 000 rows 25
// and 28; 256 x 64, 150 000 rows 25 and 22, 300 000 rows 39 and 39; 64 experts of 128 x 64, 150 000 rows 17 and 16, 300 000 rows
// 23 and 28; fp32, 5 experts of 64 x 128, 150 000 rows 37 and 37, 700 000 rows 126 and 174; 60 x 40, 300 000 rows 36 and 35; 64
// experts of 128 x 64, 700 000 rows 149 and 136.
// More than 128 columns take a wave for each 128, which all fetch the rows: 3 experts of 64 x 1024, 42 838 rows, bf16, 21 and 28,
// transposed 26 and 28, fp32 72 and 84; 8 of 42 x 477, 81 744 rows, bf16, 19 and 34; 5 of 144 x 352, 390 000 rows, bf16, 176 and 143;
// 3 of 64 x 512, 20 000 rows, bf16, 10 and 10, transposed 14 and 10, fp32 25 and 23.
template <typename T>
int launch_narrow(const ProductArgs<T>& p, bool across, hipStream_t st);
template <typename T>
bool narrow(const ProductArgs<T>& p, bool across) {
  constexpr bool kHalf = sizeof(T) == 2;
  const int64_t steps = (p.inner + kStep<T> - 1) / kStep<T>;
  if (p.inner < 8 || p.outer < 8 || p.experts > (kHalf ? 64 : 16)) return false;
  if (p.outer <= 128) return steps <= (p.outer <= 64 ? 8 : 4) && p.n >= (kHalf ? 1 << 18 : 1 << 19);
  const int64_t shares = kCus / ((p.outer + 127) / 128) - p.experts - 1;
  return across && steps <= 4 && shares >= 4 && shares >= 2 * p.experts && p.n >= (kHalf ? 1 << 23 : 1 << 24) / p.outer;
}

// Where 64 x 64 tiles do not fill the card, the depth of a tile has to be shared out, too, if it is long: the more tiles
// there are, the longer it has to be, and much longer where the matrix's values lie along the depth, which is read in pieces of
// 64 bytes, at odd places above all.  With eight rows an expert or less a tile's products are mostly of no row: then fp32, whose
// products take sixteen times as long, gains whatever their number, 16-bit values if the depth is very long.  Kernel times of both, us,
// few rows first: bf16, 3 experts of 520 x 512, 60 rows each 6 and 6; 9 of 2048 x 1024, 2 rows 9 and 12; 30 of 4096 x 256, 8 rows 16
// and 19; of 2048 x 1024, 16 rows 32 and 21; of 2053 x 1030, transposed, 8 rows 89 and 39; 100 of 3504 x 1760, 2 rows 185 and 229;
// of 1001 x 333, 8 rows 22 and 18; fp32, 100 of 2048 x 1024, 8 rows 172 and 264, 16 rows 212 and 269, transposed 258 and 246; 3 of
// 250 x 700, 60 rows 6 and 10; 9 of 2048 x 1024, 60 rows 55 and 47.
template <typename T>
bool few_rows(const ProductArgs<T>& p, bool across) {
  constexpr bool kHalf = sizeof(T) == 2;
  const int64_t tiles = likely_tiles(p, 64, 64);
  if (p.outer < 8) return false;
  const bool odd = kHalf && !across && !(aligned_to(p.weight, 4) && p.weight_stride % 2 == 0 && p.expert_stride % 2 == 0);
  if (odd) return tiles * 80 <= p.inner;
  if (p.n <= 8 * p.experts && p.inner >= (kHalf ? 3000 : 128)) return true;
  if (p.n <= 16 * p.experts && (tiles < 160 || (!kHalf && across && p.inner >= 512))) return true;
  return p.inner >= 128 && tiles < 200 && tiles * (kHalf ? (across ? 24 : 100) : across ? 2 : 5) <= p.inner;
}

}  // namespace products
}  // namespace gs
