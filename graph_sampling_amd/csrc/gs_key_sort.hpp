// Stable sort of the positions 0..n-1 by a key, for keys of a few bits: what the gradient of an
// embedding and the sending of rows to experts start from.  One 64-bit word per item, the key
// above its position, eight bits of the key a pass; nothing here keeps a state between calls or
// waits for another workgroup, so that a call can be captured into a graph.
#pragma once

#include "gs_common.hpp"

namespace gs {
namespace key_sort {

constexpr int kBits = 8;
constexpr int kDigits = 1 << kBits;
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kItems = 4;
constexpr int kTile = kThreads * kItems;
// tiles whose counts every workgroup of a pass adds up by itself
constexpr int64_t kSelfTiles = 256;

using Word = unsigned long long;

// An id as a key: what lies outside [0, num) comes behind all others, under the key num.
template <typename IdT>
struct IdWords {
  const IdT* ids;
  uint32_t num;
  __device__ __forceinline__ Word operator()(int64_t i) const {
    const int64_t id = static_cast<int64_t>(ids[i]);
    const uint32_t key = id >= 0 && id < static_cast<int64_t>(num) ? static_cast<uint32_t>(id) : num;
    return (static_cast<Word>(key) << 32) | static_cast<uint32_t>(i);
  }
};
struct StoredWords {
  const Word* word;
  __device__ __forceinline__ Word operator()(int64_t i) const { return word[i]; }
};

__device__ __forceinline__ uint32_t key_of(Word w) { return static_cast<uint32_t>(w >> 32); }
__device__ __forceinline__ uint32_t position_of(Word w) { return static_cast<uint32_t>(w); }
__device__ __forceinline__ uint32_t digit_of(Word w, int pass) {
  return (key_of(w) >> (kBits * pass)) & (kDigits - 1);
}

// passes for the keys 0..num
inline int passes_for(uint32_t num) {
  int passes = 1;
  while (passes < 4 && (static_cast<uint64_t>(num) >> (kBits * passes)) != 0) ++passes;
  return passes;
}

struct TileTables {
  uint32_t count[kWaves][kDigits];  // of a wave's items, then of the waves before it
  uint32_t scan[kDigits / kWave];
};

// item r of this thread: a wave owns 64 * kItems consecutive items, 64 of them a round
__device__ __forceinline__ uint32_t item_of(int r) {
  return (threadIdx.x / kWave) * (kWave * kItems) + r * kWave + (threadIdx.x & (kWave - 1));
}

// Rank of each item among the earlier items of the tile with its digit, and in `total` (threads
// below 256) how many items the tile holds of digit threadIdx.x.  A round's 64 items are compared by
// eight ballots; only the wave itself touches its counts until the barrier.  Items from `live`
// on are not counted.  Every thread of the workgroup calls this.
__device__ __forceinline__ void rank_tile(const uint32_t (&digit)[kItems], uint32_t live, TileTables& t,
                                          uint32_t (&rank)[kItems], uint32_t* total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  for (int j = threadIdx.x; j < kWaves * kDigits; j += kThreads) (&t.count[0][0])[j] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const bool in = item_of(r) < live;
    unsigned long long same = __ballot(in);
#pragma unroll
    for (int b = 0; b < kBits; ++b) {
      const unsigned long long set = __ballot((digit[r] >> b) & 1u);
      same &= (digit[r] >> b) & 1u ? set : ~set;
    }
    uint32_t earlier = 0;
    if (in) earlier = t.count[wave][digit[r]];
    const uint32_t in_round = __popcll(same & ((1ull << lane) - 1));
    rank[r] = earlier + in_round;
    __builtin_amdgcn_wave_barrier();  // (all have read before the last of the equal ones adds them)
    if (in && (same >> lane) == 1ull) t.count[wave][digit[r]] = rank[r] + 1;
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  uint32_t sum = 0;
  if (threadIdx.x < kDigits) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = t.count[w][threadIdx.x];
      t.count[w][threadIdx.x] = sum;
      sum += c;
    }
  }
  *total = sum;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r)
    if (item_of(r) < live) rank[r] += t.count[wave][digit[r]];
}

// Exclusive prefix over the digits, one a thread (threads below 256 hold a value); ends with a barrier
// for all.
__device__ __forceinline__ uint32_t scan_digits(uint32_t v, TileTables& t) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  uint32_t incl = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = __shfl_up(incl, d, kWave);
    if (lane >= d) incl += o;
  }
  if (threadIdx.x < kDigits && lane == kWave - 1) t.scan[wave] = incl;
  __syncthreads();
  uint32_t before = 0;
  if (threadIdx.x < kDigits)
    for (int w = 0; w < wave; ++w) before += t.scan[w];
  __syncthreads();
  return before + incl - v;
}

// counts[tile * 256 + d] = items of the tile with digit d
template <typename Src>
__global__ void __launch_bounds__(kThreads)
count_kernel(Src src, int64_t n, int pass, uint32_t* __restrict__ counts) {
  __shared__ uint32_t s_hist[4][kDigits];
  for (int j = threadIdx.x; j < 4 * kDigits; j += kThreads) (&s_hist[0][0])[j] = 0;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  Word w[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int64_t i = base + r * kThreads + threadIdx.x;
    w[r] = src(i < n ? i : n - 1);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r)
    if (base + r * kThreads + threadIdx.x < n) atomicAdd(&s_hist[threadIdx.x & 3][digit_of(w[r], pass)], 1u);
  __syncthreads();
  if (threadIdx.x < kDigits) {
    uint32_t all = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) all += s_hist[c][threadIdx.x];
    counts[static_cast<int64_t>(blockIdx.x) * kDigits + threadIdx.x] = all;
  }
}

// For sorts of more than kSelfTiles tiles: in place of every count, how many items of its digit the
// tiles before hold, and in totals[d] how many all hold.  A workgroup a digit.
static __global__ void __launch_bounds__(kThreads)
prefix_kernel(uint32_t* __restrict__ counts, int64_t tiles, uint32_t* __restrict__ totals) {
  __shared__ int64_t s_scan[kWaves + 1];
  const int digit = blockIdx.x;
  int64_t run = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += kThreads) {
    const int64_t t = t0 + threadIdx.x;
    const int64_t c = t < tiles ? counts[t * kDigits + digit] : 0;
    int64_t all;
    const int64_t at = block_exclusive_scan<kThreads>(c, &all, s_scan);
    if (t < tiles) counts[t * kDigits + digit] = static_cast<uint32_t>(run + at);
    run += all;
  }
  if (threadIdx.x == 0) totals[digit] = static_cast<uint32_t>(run);
}

// One pass over one tile.  Out: what becomes of an item at its place (and, of the first tile, of the
// places where the digits start).
template <typename Src, bool SELF, typename Out>
__global__ void __launch_bounds__(kThreads)
pass_kernel(Src src, int64_t n, int pass, int64_t tiles, const uint32_t* __restrict__ counts,
            const uint32_t* __restrict__ totals, Out out) {
  __shared__ TileTables s_tables;
  __shared__ uint32_t s_all[4][kDigits], s_before[4][kDigits], s_base[kDigits];
  const int64_t tile = blockIdx.x, base = tile * kTile;
  const uint32_t live = n - base < kTile ? static_cast<uint32_t>(n - base) : kTile;
  Word w[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const uint32_t j = item_of(r);
    w[r] = src(base + (j < live ? j : live - 1));
  }
  const int digit = threadIdx.x & (kDigits - 1);
  if (SELF) {  // four threads a digit, a quarter of the tiles each
    const int part = threadIdx.x / kDigits;
    uint32_t all = 0, before = 0;
    for (int64_t b0 = part; b0 < tiles; b0 += 8 * (kThreads / kDigits)) {
      uint32_t c[8];  // (asked for together)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t b = b0 + k * (kThreads / kDigits);
        c[k] = counts[(b < tiles ? b : tiles - 1) * kDigits + digit];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int64_t b = b0 + k * (kThreads / kDigits);
        all += b < tiles ? c[k] : 0;
        before += b < tile ? c[k] : 0;
      }
    }
    s_all[part][digit] = all;
    s_before[part][digit] = before;
  }
  uint32_t d[kItems], rank[kItems], total;
#pragma unroll
  for (int r = 0; r < kItems; ++r) d[r] = digit_of(w[r], pass);
  rank_tile(d, live, s_tables, rank, &total);
  uint32_t all = 0, before = 0;
  if (threadIdx.x < kDigits) {
    if (SELF) {
#pragma unroll
      for (int p = 0; p < kThreads / kDigits; ++p) {
        all += s_all[p][digit];
        before += s_before[p][digit];
      }
    } else {
      all = totals[digit];
      before = counts[tile * kDigits + digit];
    }
  }
  const uint32_t start = scan_digits(all, s_tables);
  if (threadIdx.x < kDigits) {
    s_base[digit] = start + before;
    if (tile == 0) out.digit(digit, start);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r)
    if (item_of(r) < live) out.item(s_base[d[r]] + rank[r], w[r]);
}

// All passes of a sort of one tile, by one workgroup in LDS: one launch.
template <typename Src, typename Out>
__global__ void __launch_bounds__(kThreads)
one_tile_kernel(Src src, uint32_t n, int passes, Out out) {
  __shared__ TileTables s_tables;
  __shared__ uint32_t s_base[kDigits];
  __shared__ Word s_word[kTile];
  Word w[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) w[r] = src(item_of(r) < n ? item_of(r) : n - 1);
  for (int pass = 0;; ++pass) {
    const bool last = pass == passes - 1;
    uint32_t d[kItems], rank[kItems], total;
#pragma unroll
    for (int r = 0; r < kItems; ++r) d[r] = digit_of(w[r], pass);
    rank_tile(d, n, s_tables, rank, &total);
    const uint32_t start = scan_digits(total, s_tables);
    if (threadIdx.x < kDigits) {
      s_base[threadIdx.x] = start;
      if (last) out.digit(threadIdx.x, start);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      if (item_of(r) >= n) continue;
      const uint32_t at = s_base[d[r]] + rank[r];
      if (last) out.item(at, w[r]);
      else s_word[at] = w[r];
    }
    if (last) return;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r)
      if (item_of(r) < n) w[r] = s_word[item_of(r)];
    __syncthreads();
  }
}

struct WordsOut {
  Word* word;
  __device__ __forceinline__ void digit(uint32_t, uint32_t) const {}
  __device__ __forceinline__ void item(uint32_t at, Word w) const { word[at] = w; }
};

struct Space {
  Word* word[2];      // ping and pong of all passes but the last
  uint32_t* counts;
  uint32_t* totals;
};
inline int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }
// words: of the two buffers, how many the sort needs (a last pass that writes elsewhere: passes - 1, at most 2)
inline size_t space_bytes(int64_t n, int words) {
  return words * padded(static_cast<size_t>(n) * 8) + padded(static_cast<size_t>(tiles_of(n)) * kDigits * 4) +
         padded(kDigits * 4);
}
inline void carve(Carver& ws, int64_t n, int words, Space* s) {
  for (int i = 0; i < 2; ++i) s->word[i] = i < words ? ws.take<Word>(static_cast<size_t>(n)) : nullptr;
  s->counts = ws.take<uint32_t>(static_cast<size_t>(tiles_of(n)) * kDigits);
  s->totals = ws.take<uint32_t>(kDigits);
}

template <typename Src, typename Out>
void launch_pass(Src src, int64_t n, int pass, const Space& s, Out out, hipStream_t st) {
  const int64_t tiles = tiles_of(n);
  const dim3 grid(static_cast<unsigned>(tiles));
  hipLaunchKernelGGL(count_kernel<Src>, grid, dim3(kThreads), 0, st, src, n, pass, s.counts);
  if (tiles <= kSelfTiles) {
    hipLaunchKernelGGL((pass_kernel<Src, true, Out>), grid, dim3(kThreads), 0, st, src, n, pass, tiles, s.counts,
                       s.totals, out);
  } else {
    hipLaunchKernelGGL(prefix_kernel, dim3(kDigits), dim3(kThreads), 0, st, s.counts, tiles, s.totals);
    hipLaunchKernelGGL((pass_kernel<Src, false, Out>), grid, dim3(kThreads), 0, st, src, n, pass, tiles, s.counts,
                       s.totals, out);
  }
}

// Sorts n >= 1 items (below 2^31), keys 0..num; the last pass hands every word with its place to `out`.  Where
// the sort has two passes it uses word[0] of the space, three or four word[0] and word[1].
template <typename Src, typename Out>
void sort(Src src, int64_t n, uint32_t num, const Space& s, Out out, hipStream_t st) {
  const int passes = passes_for(num);
  if (n <= kTile) {
    hipLaunchKernelGGL((one_tile_kernel<Src, Out>), dim3(1), dim3(kThreads), 0, st, src, static_cast<uint32_t>(n),
                       passes, out);
    return;
  }
  for (int p = 0; p < passes; ++p) {
    const StoredWords stored{s.word[(p + 1) & 1]};
    const WordsOut next{s.word[p & 1]};
    if (p == 0 && passes == 1) launch_pass(src, n, p, s, out, st);
    else if (p == 0) launch_pass(src, n, p, s, next, st);
    else if (p == passes - 1) launch_pass(stored, n, p, s, out, st);
    else launch_pass(stored, n, p, s, next, st);
  }
}

}  // namespace key_sort
}  // namespace gs
