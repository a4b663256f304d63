// Stable sort of the positions 0..n-1 by a key, for keys of a few bits: what the gradient of an
// embedding and the sending of rows to experts start from.  One 64-bit word per item, the key
// above its position, eight or nine bits of the key a pass; nothing here keeps a state between calls or
// waits for another workgroup, so that a call can be captured into a graph.
#pragma once

#include "gs_common.hpp"

namespace gs {
namespace key_sort {

constexpr int kItems = 4;  // of a thread
// A tile is the items of 256, 512 or 1024 threads: comparing them by ballots is what a pass takes longest
// for, and small tiles spread that over more compute units, as long as their counts are few.  Up to 16 k counts
// every workgroup of a pass adds up all of them by itself, if a thread reads no more than it asks for at once;
// more are added up by a launch between.  Us a count and pass (8 bits, 4 M keys), by itself / with that launch:
// 131 k items in 256-thread tiles 12.3 / 9.4, 512 8.5 / 9.7, 1024 10.9 / 11.0; 400 k 31.6 / 12.3, 14.9 / 10.8,
// 11.6 / 11.6; 810 k -, 31.2 / 13.9, 15.9 / 13.2; 2 M -, 106 / 21.4, 39.5 / 19.0.  (16 k items, the pass alone:
// 256 threads 4.9, 512 5.9, 1024 8.1.)
constexpr int64_t kAlone = 1024 * kItems;        // items that one workgroup sorts alone
constexpr int64_t kFewItems = 4 * kAlone;        // items that every workgroup of a pass counts by itself
constexpr int64_t kSelfCounts = int64_t(1) << 14;
constexpr int kMostDigits = 512;
constexpr int ahead_of(int bits) { return bits <= 4 ? 8 : 32; }  // counts a thread asks for at once
inline int64_t tiles_of(int64_t n, int threads) { return (n + threads * kItems - 1) / (threads * kItems); }
inline bool adds_up_itself(int64_t tiles, int bits, int threads) {
  return tiles <= ahead_of(bits) * (threads >> bits) && (tiles << bits) <= kSelfCounts;
}
// (a thread a digit at least)
inline int threads_for(int64_t n, int bits) {
  const int least = bits == 9 ? 512 : 256;
  if (n <= kAlone) return n <= 256 * kItems && least == 256 ? 256 : n <= 512 * kItems ? 512 : 1024;
  if (n <= kFewItems) return 512;
  for (int threads = least; threads <= 1024; threads *= 2)
    if (adds_up_itself(tiles_of(n, threads), bits, threads)) return threads;
  return n <= (int64_t(1) << 19) ? 512 : 1024;
}

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

// Digits of eight bits, or of nine where that is a pass less (keys of 17 and 18 bits, of 25 to 27): 400 k
// keys of 18 bits take two passes of 14 us for three of 13.  Few keys (FEW: a caller that expects some) have digits
// of four or seven bits: fewer ballots and fewer counts.
struct Digits {
  int bits, passes;
  explicit Digits(uint32_t num, bool few = false) {
    int key_bits = 1;
    while (key_bits < 32 && (num >> key_bits) != 0) ++key_bits;
    const int eight = (key_bits + 7) / 8, nine = (key_bits + 8) / 9;
    bits = nine < eight ? 9 : 8;
    passes = nine < eight ? nine : eight;
    if (few && key_bits <= 7) bits = key_bits <= 4 ? 4 : 7;
  }
};
// copies of a table of counts that many threads add to: where many items hold one digit, additions queue up
template <int BITS>
constexpr int kCopies = BITS <= 7 ? 16 : 4;
template <int BITS>
__device__ __forceinline__ uint32_t digit_of(Word w, int pass) {
  return (key_of(w) >> (BITS * pass)) & ((1u << BITS) - 1);
}

// Work that has nothing to do with the sort and runs beside it, in workgroups of their own: a sort of
// a few thousand items occupies a few compute units.
struct NoWork {
  static constexpr bool kAny = false;
  __device__ __forceinline__ void run(int64_t, int64_t, int) const {}
};

template <int BITS, int THREADS>
struct TileTables {
  static constexpr int kDigits = 1 << BITS, kWaves = THREADS / kWave;
  static_assert(kDigits <= THREADS, "a thread a digit");
  uint16_t count[kWaves][kDigits];  // of a wave's items, then of the waves before it
  uint2 scan[kDigits > kWave ? kDigits / kWave : 1];
};

// item r of this thread: a wave owns 64 * kItems consecutive items, 64 of them a round
__device__ __forceinline__ uint32_t item_of(int r) {
  return (threadIdx.x / kWave) * (kWave * kItems) + r * kWave + (threadIdx.x & (kWave - 1));
}

// Rank of each item among the earlier items of the tile with its digit, and in `total` (a thread a
// digit) how many items the tile holds of digit threadIdx.x.  A round's 64 items are compared by a
// ballot a bit; only the wave itself touches its counts until the barrier.  Items from `live`
// on are not counted.  Every thread of the workgroup calls this.
template <int BITS, int THREADS>
__device__ __forceinline__ void rank_tile(const uint32_t (&digit)[kItems], uint32_t live, TileTables<BITS, THREADS>& t,
                                          uint32_t (&rank)[kItems], uint32_t* total) {
  constexpr int kDigits = 1 << BITS, kWaves = THREADS / kWave;
  const int wave = threadIdx.x / kWave;
#pragma unroll
  for (int j = threadIdx.x; j < kWaves * kDigits / 2; j += THREADS)
    reinterpret_cast<uint32_t*>(&t.count[0][0])[j] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const bool in = item_of(r) < live;
    const unsigned long long there = __ballot(in);
    // lanes with this digit: per bit, the lanes whose bit equals this lane's (and-not-xor in one instruction)
    uint32_t lo = static_cast<uint32_t>(there), hi = static_cast<uint32_t>(there >> 32);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
      const int mine = static_cast<int>(digit[r] << (31 - b)) >> 31;
      const unsigned long long set = __ballot(mine);
      lo = __builtin_amdgcn_bitop3_b32(lo, static_cast<uint32_t>(set), mine, 0x90);
      hi = __builtin_amdgcn_bitop3_b32(hi, static_cast<uint32_t>(set >> 32), mine, 0x90);
    }
    const uint32_t in_round = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
    const uint32_t earlier = t.count[wave][digit[r]];  // (LDS operations of a wave keep their order)
    rank[r] = earlier + in_round;
    if (in && in_round == 0) t.count[wave][digit[r]] = static_cast<uint16_t>(earlier + __popc(lo) + __popc(hi));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (keeps the next round's reads behind this one's writes)
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  uint32_t sum = 0;
  if (threadIdx.x < kDigits) {
    uint32_t c[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) c[w] = t.count[w][threadIdx.x];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      t.count[w][threadIdx.x] = static_cast<uint16_t>(sum);
      sum += c[w];
    }
  }
  *total = sum;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) rank[r] += t.count[wave][digit[r]];
}

// Exclusive prefixes over the digits of two numbers, one digit a thread (the first threads hold values); every
// thread of the workgroup calls this.
template <int BITS, int THREADS>
__device__ __forceinline__ void scan_digits(uint32_t& v, uint32_t& u, TileTables<BITS, THREADS>& t) {
  constexpr int kDigits = 1 << BITS;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  uint32_t vi = v, ui = u;
  if (threadIdx.x < kDigits) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t vo = __shfl_up(vi, d, kWave), uo = __shfl_up(ui, d, kWave);
      if (lane >= d) {
        vi += vo;
        ui += uo;
      }
    }
    if (kDigits > kWave && lane == kWave - 1) t.scan[wave] = make_uint2(vi, ui);
  }
  __syncthreads();
  v = vi - v;
  u = ui - u;
  if (threadIdx.x < kDigits && kDigits > kWave) {
#pragma unroll
    for (int w = 0; w < kDigits / kWave; ++w) {
      const uint2 s = t.scan[w];
      v += w < wave ? s.x : 0;
      u += w < wave ? s.y : 0;
    }
  }
}

// counts[tile * digits + d] = items of the tile with digit d
template <int BITS, int THREADS, typename Src, typename Beside>
__global__ void __launch_bounds__(THREADS)
count_kernel(Src src, int64_t n, int pass, int64_t tiles, uint32_t* __restrict__ counts, Beside beside) {
  constexpr int kDigits = 1 << BITS;
  if (Beside::kAny && blockIdx.x >= tiles) return beside.run(blockIdx.x - tiles, gridDim.x - tiles, THREADS);
  __shared__ uint32_t s_hist[kCopies<BITS>][kDigits + 1];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (THREADS * kItems);
  Word w[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const int64_t i = base + r * THREADS + threadIdx.x;
    w[r] = src(i < n ? i : n - 1);
  }
#pragma unroll
  for (int j = threadIdx.x; j < kCopies<BITS> * (kDigits + 1); j += THREADS) (&s_hist[0][0])[j] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r)
    if (base + r * THREADS + threadIdx.x < n)
      atomicAdd(&s_hist[threadIdx.x % kCopies<BITS>][digit_of<BITS>(w[r], pass)], 1u);
  __syncthreads();
  if (threadIdx.x < kDigits) {
    uint32_t all = 0;
#pragma unroll
    for (int c = 0; c < kCopies<BITS>; ++c) all += s_hist[c][threadIdx.x];
    counts[static_cast<int64_t>(blockIdx.x) * kDigits + threadIdx.x] = all;
  }
}

// For sorts of many tiles: in place of every count, how many items of its digit the
// tiles before hold, and in totals[d] how many all hold.  A workgroup a digit.
constexpr int kPrefixThreads = 256;
static __global__ void __launch_bounds__(kPrefixThreads)
prefix_kernel(uint32_t* __restrict__ counts, int64_t tiles, int digits, uint32_t* __restrict__ totals) {
  __shared__ int64_t s_scan[kPrefixThreads / kWave + 1];
  const int digit = blockIdx.x;
  int64_t run = 0;
  for (int64_t t0 = 0; t0 < tiles; t0 += kPrefixThreads) {
    const int64_t t = t0 + threadIdx.x;
    const int64_t c = t < tiles ? counts[t * digits + digit] : 0;
    int64_t all;
    const int64_t at = block_exclusive_scan<kPrefixThreads>(c, &all, s_scan);
    if (t < tiles) counts[t * digits + digit] = static_cast<uint32_t>(run + at);
    run += all;
  }
  if (threadIdx.x == 0) totals[digit] = static_cast<uint32_t>(run);
}

// Where a pass gets the counts of all tiles from: it counts all items by itself (a launch less, for few),
// adds up the tiles' counts, or finds them added up.
enum class Counts { kHere, kTiles, kPrefixes };

// One pass over one tile.  Out: what becomes of an item at its place -- `item`, in the order of their
// places, so that neighbours are written together, and `from`, in the order in which they came -- and, of
// the first tile, of the places where the digits start.  The tile is put in order in LDS first.
template <int BITS, int THREADS, typename Src, Counts COUNTS, typename Out, typename Beside>
__global__ void __launch_bounds__(THREADS)
pass_kernel(Src src, int64_t n, int pass, int64_t tiles, const uint32_t* __restrict__ counts,
            const uint32_t* __restrict__ totals, Out out, Beside beside) {
  constexpr int kDigits = 1 << BITS, kTile = THREADS * kItems;
  constexpr int kParts = COUNTS == Counts::kHere ? 2 * kCopies<BITS> : THREADS / kDigits;
  if (Beside::kAny && blockIdx.x >= tiles) return beside.run(blockIdx.x - tiles, gridDim.x - tiles, THREADS);
  __shared__ TileTables<BITS, THREADS> s_tables;
  __shared__ uint32_t s_all[kParts][kDigits + 1], s_before[kParts][kDigits + 1];
  __shared__ uint32_t s_start[kDigits];  // where a digit's items start in the tile
  __shared__ uint32_t s_shift[kDigits];  // from a place in the tile's order to the place in memory, modulo 2^32
  __shared__ Word s_word[kTile];
  const int64_t tile = blockIdx.x, base = tile * kTile;
  const uint32_t live = n - base < kTile ? static_cast<uint32_t>(n - base) : kTile;
  Word w[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const uint32_t j = item_of(r);
    w[r] = src(base + (j < live ? j : live - 1));
  }
  const int digit = threadIdx.x & (kDigits - 1), part = threadIdx.x / kDigits;
  if constexpr (COUNTS == Counts::kHere) {
    constexpr int kAhead = 8;
#pragma unroll
    for (int j = threadIdx.x; j < kParts * (kDigits + 1); j += THREADS) (&s_all[0][0])[j] = (&s_before[0][0])[j] = 0;
    __syncthreads();
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += kAhead * THREADS) {
      Word other[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) other[k] = src(i0 + k * THREADS < n ? i0 + k * THREADS : n - 1);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t i = i0 + k * THREADS;
        if (i >= n) continue;
        atomicAdd(i < base ? &s_before[threadIdx.x % kParts][digit_of<BITS>(other[k], pass)]
                           : &s_all[threadIdx.x % kParts][digit_of<BITS>(other[k], pass)], 1u);
      }
    }
    // (s_all: of this tile and those behind it)
  } else if constexpr (COUNTS == Counts::kTiles) {  // a share of the tiles a thread, kAhead counts asked for together
    constexpr int kAhead = ahead_of(BITS);
    uint32_t all = 0, before = 0;
    for (int b0 = part; b0 < static_cast<int>(tiles); b0 += kAhead * kParts) {
      uint32_t c[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int b = b0 + k * kParts;
        c[k] = counts[(b < static_cast<int>(tiles) ? b : b0) * kDigits + digit];
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int b = b0 + k * kParts;
        all += b < static_cast<int>(tiles) && b >= static_cast<int>(tile) ? c[k] : 0;
        before += b < static_cast<int>(tile) ? c[k] : 0;
      }
    }
    s_all[part][digit] = all;
    s_before[part][digit] = before;
  }
  uint32_t d[kItems], rank[kItems], total;
#pragma unroll
  for (int r = 0; r < kItems; ++r) d[r] = digit_of<BITS>(w[r], pass);
  rank_tile<BITS, THREADS>(d, live, s_tables, rank, &total);
  uint32_t all = 0, before = 0;
  if (threadIdx.x < kDigits) {
    if (COUNTS == Counts::kPrefixes) {
      all = totals[digit];
      before = counts[tile * kDigits + digit];
    } else {
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        all += s_all[p][digit];
        before += s_before[p][digit];
      }
      all += before;
    }
  }
  uint32_t start = all, here = total;
  scan_digits(start, here, s_tables);
  if (threadIdx.x < kDigits) {
    s_start[digit] = here;
    s_shift[digit] = start + before - here;
    if (tile == 0) out.digit(digit, start);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    if (item_of(r) >= live) continue;
    const uint32_t at = s_start[d[r]] + rank[r];
    s_word[at] = w[r];
    out.from(w[r], at + s_shift[d[r]]);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const uint32_t at = r * THREADS + threadIdx.x;
    if (at >= live) continue;
    const Word word = s_word[at];
    out.item(at + s_shift[digit_of<BITS>(word, pass)], word);
  }
}

// All passes of a sort of up to kItems * THREADS items, by one workgroup in LDS: one launch.
template <int BITS, int THREADS, typename Src, typename Out, typename Beside>
__global__ void __launch_bounds__(THREADS)
alone_kernel(Src src, uint32_t n, int passes, Out out, Beside beside) {
  constexpr int kDigits = 1 << BITS;
  if (Beside::kAny && blockIdx.x >= 1) return beside.run(blockIdx.x - 1, gridDim.x - 1, THREADS);
  __shared__ TileTables<BITS, THREADS> s_tables;
  __shared__ uint32_t s_start[kDigits];
  __shared__ Word s_word[THREADS * kItems];
  Word w[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) w[r] = src(item_of(r) < n ? item_of(r) : n - 1);
  for (int pass = 0; pass < passes; ++pass) {
    const bool last = pass == passes - 1;
    uint32_t d[kItems], rank[kItems], total;
#pragma unroll
    for (int r = 0; r < kItems; ++r) d[r] = digit_of<BITS>(w[r], pass);
    rank_tile<BITS, THREADS>(d, n, s_tables, rank, &total);
    uint32_t start = total, none = 0;
    scan_digits(start, none, s_tables);
    if (threadIdx.x < kDigits) {
      s_start[threadIdx.x] = start;
      if (last) out.digit(threadIdx.x, start);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      if (item_of(r) >= n) continue;
      const uint32_t at = s_start[d[r]] + rank[r];
      s_word[at] = w[r];
      if (last) out.from(w[r], at);
    }
    __syncthreads();
    if (!last) {
#pragma unroll
      for (int r = 0; r < kItems; ++r) w[r] = s_word[item_of(r) < n ? item_of(r) : n - 1];
      __syncthreads();
    }
  }
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    const uint32_t at = r * THREADS + threadIdx.x;
    if (at < n) out.item(at, s_word[at]);
  }
}

struct WordsOut {
  Word* word;
  __device__ __forceinline__ void digit(uint32_t, uint32_t) const {}
  __device__ __forceinline__ void from(Word, uint32_t) const {}
  __device__ __forceinline__ void item(uint32_t at, Word w) const { word[at] = w; }
};

struct Space {
  Word* word[2];      // ping and pong of all passes but the last
  uint32_t* counts;
  uint32_t* totals;
};
// words: of the two buffers, how many the sort needs (a last pass that writes elsewhere: passes - 1, at most 2)
// (a tile's counts are no more than a quarter of its items: 512 of 512 threads, 256 of 256)
inline size_t most_counts(int64_t n) { return static_cast<size_t>(n / 4 + kMostDigits); }
inline size_t space_bytes(int64_t n, int words) {
  if (n <= kAlone) return 0;  // (one workgroup does it in LDS)
  return words * padded(static_cast<size_t>(n) * 8) + padded(most_counts(n) * 4) + padded(kMostDigits * 4);
}
inline void carve(Carver& ws, int64_t n, int words, Space* s) {
  *s = Space{};
  if (n <= kAlone) return;
  for (int i = 0; i < 2; ++i) s->word[i] = i < words ? ws.take<Word>(static_cast<size_t>(n)) : nullptr;
  s->counts = ws.take<uint32_t>(most_counts(n));
  s->totals = ws.take<uint32_t>(kMostDigits);
}

// a launch of `tiles` workgroups and those of the work beside it, as its next part
template <typename Beside, typename Kernel, typename... Args>
void launch_beside(Kernel kernel, int64_t tiles, int threads, hipStream_t st, Beside& beside, Args... args) {
  int64_t blocks = tiles;
  if constexpr (Beside::kAny) blocks += beside.blocks(threads);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, st, args..., beside);
  if constexpr (Beside::kAny) ++beside.part;
}

template <int BITS, int THREADS, typename Src, typename Out, typename Beside>
void launch_pass(Src src, int64_t n, int pass, const Space& s, Out out, Beside& beside, hipStream_t st) {
  const int64_t tiles = tiles_of(n, THREADS);
  const uint32_t *counts = s.counts, *totals = s.totals;
  if (n <= kFewItems) {
    launch_beside(pass_kernel<BITS, THREADS, Src, Counts::kHere, Out, Beside>, tiles, THREADS, st, beside, src, n, pass,
                  tiles, counts, totals, out);
    return;
  }
  launch_beside(count_kernel<BITS, THREADS, Src, Beside>, tiles, THREADS, st, beside, src, n, pass, tiles, s.counts);
  const bool self = adds_up_itself(tiles, BITS, THREADS);
  if (!self)
    hipLaunchKernelGGL(prefix_kernel, dim3(1 << BITS), dim3(kPrefixThreads), 0, st, s.counts, tiles, 1 << BITS, s.totals);
  launch_beside(self ? pass_kernel<BITS, THREADS, Src, Counts::kTiles, Out, Beside>
                     : pass_kernel<BITS, THREADS, Src, Counts::kPrefixes, Out, Beside>,
                tiles, THREADS, st, beside, src, n, pass, tiles, counts, totals, out);
}

template <int BITS, int THREADS, typename Src, typename Out, typename Beside>
void sort_tiles(Src src, int64_t n, int passes, const Space& s, Out out, Beside beside, hipStream_t st) {
  if constexpr (Beside::kAny) beside.parts = n <= kFewItems ? passes : 2 * passes;
  for (int p = 0; p < passes; ++p) {
    const StoredWords stored{s.word[(p + 1) & 1]};
    const WordsOut next{s.word[p & 1]};
    if (p == 0 && passes == 1) launch_pass<BITS, THREADS>(src, n, p, s, out, beside, st);
    else if (p == 0) launch_pass<BITS, THREADS>(src, n, p, s, next, beside, st);
    else if (p == passes - 1) launch_pass<BITS, THREADS>(stored, n, p, s, out, beside, st);
    else launch_pass<BITS, THREADS>(stored, n, p, s, next, beside, st);
  }
}

template <int BITS, int THREADS, typename Src, typename Out, typename Beside>
void sort_with(Src src, int64_t n, int passes, const Space& s, Out out, Beside beside, hipStream_t st) {
  if (n > kAlone) return sort_tiles<BITS, THREADS>(src, n, passes, s, out, beside, st);
  if constexpr (Beside::kAny) beside.parts = 1;
  launch_beside(alone_kernel<BITS, THREADS, Src, Out, Beside>, 1, THREADS, st, beside, src, static_cast<uint32_t>(n),
                passes, out);
}

template <int BITS, typename Src, typename Out, typename Beside>
void sort_by(Src src, int64_t n, int passes, const Space& s, Out out, Beside beside, hipStream_t st) {
  const int threads = threads_for(n, BITS);
  if constexpr (BITS <= 8) {
    if (threads == 256) return sort_with<BITS, 256>(src, n, passes, s, out, beside, st);
  }
  if (threads == 512) return sort_with<BITS, 512>(src, n, passes, s, out, beside, st);
  sort_with<BITS, 1024>(src, n, passes, s, out, beside, st);
}

// Sorts n >= 1 items (below 2^31), keys 0..num; the last pass hands every word with its place to `out`.  Where
// the sort has two passes it uses word[0] of the space, three or four word[0] and word[1].  beside: run in as many
// equal parts as there are launches.  FEW: as in Digits.
template <bool FEW, typename Src, typename Out, typename Beside = NoWork>
void sort(Src src, int64_t n, uint32_t num, const Space& s, Out out, hipStream_t st, Beside beside = Beside()) {
  const Digits digits(num, FEW);
  if constexpr (FEW) {
    if (digits.bits == 4) return sort_by<4>(src, n, 1, s, out, beside, st);
    if (digits.bits == 7) return sort_by<7>(src, n, 1, s, out, beside, st);
  }
  if (digits.bits == 9) sort_by<9>(src, n, digits.passes, s, out, beside, st);
  else sort_by<8>(src, n, digits.passes, s, out, beside, st);
}

}  // namespace key_sort
}  // namespace gs
