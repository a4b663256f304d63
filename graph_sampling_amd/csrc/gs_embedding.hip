// Embedding lookup with scaling, and its gradient by sorted ids, on gfx950.
//
//   lookup    out[n, :]  = scale * table[ids[n], :]
//   gradient  grad[v, :] = scale * sum of dout[n, :] over the n with ids[n] = v
//
// No counterpart in the reference, whose examples index feature matrices with torch.  An id outside
// the table stands for no row: zeros come out, nothing goes into the gradient, nothing is read.
// Values are fp32, fp16 or bf16; products and sums are fp32, rounded once on the way out.
//
// The gradient adds in an order that follows from the ids alone, without atomics: the positions are
// sorted by id (gs_key_sort.hpp), a group of lanes adds up a tile of consecutive sorted positions run
// by run, and writes a row when the run lies inside its tile.  Runs that cross tiles are joined in
// LDS by the workgroup's groups, and those that cross workgroups leave partial sums, at most two a
// workgroup, which are themselves a sorted list: the next launch adds them up in the same way, and
// so on until one workgroup holds all.  So a row that half of the ids name costs no more
// than any other, and sums of many addends are sums of sums, which keeps fp32 exact enough.
#include "gs_key_sort.hpp"
#include "gs_rows.hpp"

namespace gs {
namespace {

constexpr int kThreads = 256;

// ------------------------------------------------------------------ lookup ----
// A chunk a lane (ITEMS of them, asked for together); a row's id is read by all its lanes, which is one
// request.  What bounds it is the rows' bytes: random rows in, consecutive rows out.
template <typename T, typename IdT, int ITEMS>
__global__ void __launch_bounds__(kThreads)
lookup_kernel(const T* __restrict__ table, int64_t num_rows, int64_t stride, int64_t dim, Divider chunks,
              const IdT* __restrict__ ids, int64_t total, float scale, T* __restrict__ out, Past past) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * ITEMS);
  const RowRange range(chunks, first);
  int64_t id[ITEMS], to[ITEMS], at[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t j = k * kThreads + threadIdx.x;
    const bool in = first + j < total;
    uint32_t c;
    const int64_t row = range.row(in ? j : 0, &c);
    at[k] = chunk_start<T>(dim, c);
    to[k] = in ? row * dim + at[k] : -1;
    id[k] = ids[row];
  }
  Values<T> v[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    v[k] = Values<T>{};
    if (id[k] >= 0 && id[k] < num_rows) v[k] = load_chunk(table + id[k] * stride + at[k], dim);
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    // (a scale of one leaves the bits as they are)
    const Values<T> w = scale == 1.0f ? v[k] : narrow<T>(widen<T>(v[k]) * scale);
    // (0 * inf where there is no row would be NaN)
    const bool there = id[k] >= 0 && id[k] < num_rows;
    if (to[k] >= 0) store_result(out + to[k], there ? w : Values<T>{}, at[k], dim, past);
  }
}

// ---------------------------------------------------------------- gradient ----
// Zeros in the whole gradient, before the rows that are met are written: beside the sort, whose launches leave
// most of the chip idle.  16 k tokens, us: the sort alone 17.1, 64 MB of zeros alone 10.6, one after the other 27.9,
// beside each other 21.7.  64 k threads, which fill at the rate that memory takes: with 256 k the sort waits for
// memory (23.4), with 16 k it is done before the zeros are (23.3).  1 GB beside 8 k ids: 213, with 256 k 228, 16 k 279.
template <typename T>
struct Zeros {
  static constexpr bool kAny = true;
  T* out;
  int64_t n;
  int part = 0, parts = 1;
  // workgroups a launch
  int blocks(int threads) const {
    const int64_t chunks = (n / Chunk<T>::kVec + parts - 1) / parts, most = (chunks + 4 * threads - 1) / (4 * threads);
    return static_cast<int>(most < 1 ? 1 : most > (1 << 16) / threads ? (1 << 16) / threads : most);
  }
  __device__ __forceinline__ void run(int64_t block, int64_t of, int threads) const {
    const int64_t whole = n / Chunk<T>::kVec, share = (whole + parts - 1) / parts;
    const int64_t end = (part + 1) * share < whole ? (part + 1) * share : whole;
    for (int64_t i = part * share + block * threads + threadIdx.x; i < end; i += of * threads)
      store_past(out + i * Chunk<T>::kVec, Values<T>{});
    if (part == 0 && block == 0 && threadIdx.x < n - whole * Chunk<T>::kVec)
      out[whole * Chunk<T>::kVec + threadIdx.x] = T(0);
  }
};
// (alone, where there is no id)
template <typename T>
__global__ void __launch_bounds__(kThreads) zero_kernel(Zeros<T> zeros) {
  zeros.run(blockIdx.x, gridDim.x, kThreads);
}

// What a tile leaves for the next launch: which output row, and whether a partial sum goes with it.
struct Entry {
  uint32_t row;
  uint32_t state;
};
constexpr uint32_t kNone = 0, kSum = 1, kThrough = 2;  // (through: the run goes on, its sum is in the entry before)

struct RunsOut {
  float scale;
  Past past;             // (results_past)
  int64_t dim;
  int64_t chunks;        // of a row
  int slices;            // workgroups side by side over a row
  int64_t* met;          // sparse: ids of the rows by their rank
  const int64_t* heads;  // sparse: runs that begin before a workgroup's positions
  Entry* entries;        // 2 a workgroup (null where there is one)
  float* sums;           // [2 * workgroups, chunks * kVec]
};

// A workgroup is up to 64 groups of G lanes, a chunk of the row a lane, group after group along the list.
// Those that sum rows have up to 512 threads, so that four of them share a compute unit; those that
// join what is left up to 1024, so that few launches do.  (A group that took 32 entries one after the other
// needed 11 us for the 256 of 16 k ids where two a group need 4.)
constexpr int kSumMost = 512, kJoinMost = 1024;
constexpr int groups_in(int most, int lanes) { return most / lanes < 64 ? most / lanes : 64; }

template <typename T, int G, int GROUPS>
struct Runs {
  static constexpr int kEntries = 2 * GROUPS;
  struct Shared {
    Entry entry[kEntries];
    Entry left[2];  // the workgroup's own
    Wide<T> sum[kEntries][G];
  };
  const RunsOut& o;
  Shared& s;
  T* out;          // at this lane's chunk
  int64_t part;    // workgroup along the list
  int64_t chunk;
  int group, lane;
  bool in;         // whether the lane has a chunk

  __device__ __forceinline__ Runs(const RunsOut& o_, Shared& s_, T* out_) : o(o_), s(s_) {
    part = blockIdx.x / o.slices;
    group = threadIdx.x / G;
    lane = threadIdx.x & (G - 1);
    chunk = (blockIdx.x - part * o.slices) * G + lane;
    in = chunk < o.chunks;
    if (!in) chunk = 0;  // (works along, writes nothing)
    out = out_ + chunk_start<T>(o.dim, chunk);
    if (lane == 0) s.entry[2 * group] = s.entry[2 * group + 1] = Entry{0, kNone};
    if (threadIdx.x < 2) s.left[threadIdx.x] = Entry{0, kNone};
  }
  __device__ __forceinline__ void write(uint32_t row, const Wide<T>& sum) {
    if (!in) return;
    store_result(out + static_cast<int64_t>(row) * o.dim, narrow<T>(sum * o.scale), chunk_start<T>(o.dim, chunk), o.dim,
                 o.past);
  }
  // a run of this group's tile that ends; left, right: it began before the tile, goes on behind it
  __device__ __forceinline__ void finish(uint32_t row, const Wide<T>& sum, bool left, bool right) {
    if (!left && !right) return write(row, sum);
    const int slot = 2 * group + (left ? 0 : 1);
    s.sum[slot][lane] = sum;
    if (lane == 0) {
      s.entry[slot] = Entry{row, kSum};
      if (left && right) s.entry[slot + 1] = Entry{row, kThrough};
    }
  }
  // the run whose first piece here is entry i, added up over the groups it goes through
  __device__ __forceinline__ void walk(int i) {
    constexpr int kAhead = 8;  // groups asked about together
    const uint32_t row = s.entry[i].row;
    const bool left = i == 0;
    Wide<T> sum = s.sum[i][lane];
    // (on: the run goes on into the next group)
    bool on = (i & 1) != 0 || (s.entry[1].state != kNone && s.entry[1].row == row);
    for (int g0 = i / 2 + 1; on && g0 < GROUPS; g0 += kAhead) {
      Entry e[kAhead][2];
      Wide<T> v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int g = g0 + k < GROUPS ? g0 + k : GROUPS - 1;
        e[k][0] = s.entry[2 * g];
        e[k][1] = s.entry[2 * g + 1];
        v[k] = s.sum[2 * g][lane];  // (what is no sum is not added)
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (g0 + k >= GROUPS) break;
        on = on && e[k][0].state == kSum && e[k][0].row == row;
        if (on) sum += v[k];
        on = on && e[k][1].state == kThrough;
      }
    }
    const bool right = on;
    if (!left && !right) return write(row, sum);
    const int slot = left ? 0 : 1;
    if (in) {
      float* to = o.sums + ((2 * part + slot) * o.chunks + chunk) * Chunk<T>::kVec;
      __builtin_memcpy(to, &sum, sizeof(sum));
    }
    if (lane == 0) {
      s.left[slot] = Entry{row, kSum};
      if (left && right) s.left[1] = Entry{row, kThrough};
    }
  }
  // behind every group's tile: every thread of the workgroup calls this.  A run begins here in the first group's first
  // entry (it began in an earlier workgroup) or in a group's last one that holds a sum.
  __device__ __forceinline__ void join() {
    __syncthreads();
    if (group == 0 && s.entry[0].state == kSum) walk(0);
    if (s.entry[2 * group + 1].state == kSum) walk(2 * group + 1);
    __syncthreads();
    if (o.entries && threadIdx.x < 2 && blockIdx.x == part * o.slices)
      o.entries[2 * part + threadIdx.x] = s.left[threadIdx.x];
  }
};

constexpr int kBatch = 8;      // rows a group asks for together
constexpr int kMostSize = 32;  // positions of a tile at most

// A row's chunk, past the caches where rows are longer than a line: every row is read once (810 k random
// rows of 256 B, added up by 32s, from memory: 44.7 us plain, 41.5 so; by skewed ids, runs of one to 37 k: 66 and 63).
template <typename T, int G>
__device__ __forceinline__ Values<T> load_once(const T* p, int64_t dim) {
  if (G >= 16 && dim >= Chunk<T>::kVec) return load_past(p);
  return load_chunk(p, dim);
}

// Whether a run of a row that is there begins at sorted position i.
__device__ __forceinline__ bool run_begins(const key_sort::Word* __restrict__ words, int64_t i, uint32_t num_rows) {
  const uint32_t key = key_sort::key_of(words[i]), before = key_sort::key_of(words[i > 0 ? i - 1 : 0]);
  return key < num_rows && (i == 0 || before != key);
}

// Runs that begin among a workgroup's positions of the kernel below.
__global__ void __launch_bounds__(kThreads)
count_runs_kernel(const key_sort::Word* __restrict__ words, int64_t n, uint32_t num_rows, int per_part,
                  int64_t* __restrict__ counts) {
  __shared__ int s_count;
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_part;
  int count = 0;
  for (int j = threadIdx.x; j < per_part; j += kThreads)
    count += first + j < n && run_begins(words, first + j, num_rows) ? 1 : 0;
#pragma unroll
  for (int m = kWave / 2; m > 0; m /= 2) count += __shfl_xor(count, m, kWave);
  if (threadIdx.x % kWave == 0) atomicAdd(&s_count, count);
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = s_count;
}

// A tile of `size` sorted positions a group.  The workgroup's words lie in LDS as {output row, position of the
// row in grad, top bit: a run begins}; the output row is the key, or its rank among the rows that are met (SPARSE),
// and ~0 where there is none.
template <typename T, int G, bool SPARSE>
__global__ void __launch_bounds__(groups_in(kSumMost, G) * G)
sum_runs_kernel(const key_sort::Word* __restrict__ words, int64_t n, uint32_t num_rows, const T* __restrict__ grad,
                int64_t stride, int size, RunsOut o, T* __restrict__ out) {
  constexpr int kGroups = groups_in(kSumMost, G), kThreadsHere = kGroups * G, kMost = kGroups * kMostSize;
  constexpr uint32_t kNowhere = ~0u, kBegins = 1u << 31;
  __shared__ typename Runs<T, G, kGroups>::Shared s_runs;
  __shared__ uint2 s_words[kMost + 1];
  __shared__ int s_heads[SPARSE ? kMost / kWave + 1 : 1];
  Runs<T, G, kGroups> runs(o, s_runs, out);
  const int here = kGroups * size;
  const int64_t first = runs.part * here;
  for (int j0 = 0; j0 <= here; j0 += kThreadsHere) {
    const int j = j0 + threadIdx.x;
    const int64_t i = first + j;
    uint2 w = make_uint2(kNowhere, kBegins);
    if (j <= here && i < n) {
      const key_sort::Word word = words[i];
      const bool begins = i == 0 || key_sort::key_of(words[i > 0 ? i - 1 : 0]) != key_sort::key_of(word);
      w.x = key_sort::key_of(word) < num_rows ? key_sort::key_of(word) : kNowhere;
      w.y = key_sort::position_of(word) | (begins ? kBegins : 0u);
    }
    if (SPARSE) {
      const unsigned long long heads = __ballot(w.x != kNowhere && (w.y & kBegins) && j < here);
      if (j % kWave == 0 && j < here) s_heads[j / kWave] = __popcll(heads);
    }
    if (j <= here) s_words[j] = w;
  }
  __syncthreads();
  if (SPARSE) {
    const int64_t before = o.heads[runs.part];
    for (int j0 = 0; j0 < here; j0 += kThreadsHere) {
      const int j = j0 + threadIdx.x;
      const uint2 w = s_words[j < here ? j : here - 1];
      const bool begins = j < here && w.x != kNowhere && (w.y & kBegins);
      const unsigned long long heads = __ballot(begins);
      int upto = __popcll(heads & (~0ull >> (kWave - 1 - threadIdx.x % kWave)));  // up to this position
      for (int c = 0; c < j / kWave && j < here; ++c) upto += s_heads[c];
      const uint32_t rank = static_cast<uint32_t>(before + upto - 1);
      if (begins && blockIdx.x == runs.part * o.slices) o.met[rank] = w.x;
      if (j < here && w.x != kNowhere) s_words[j].x = rank;
    }
    __syncthreads();
  }
  const uint2* const mine = s_words + runs.group * size;
  const T* const from = grad + chunk_start<T>(o.dim, runs.chunk);
  uint32_t row = mine[0].x;
  if (row != kNowhere) {
    bool left = !(mine[0].y & kBegins);
    Wide<T> sum = {};
    for (int j0 = 0; j0 < size && row != kNowhere; j0 += kBatch) {
      uint2 w[kBatch];
      Values<T> v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) w[k] = mine[j0 + k];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const uint32_t at = w[k].x != kNowhere ? w[k].y & ~kBegins : w[0].y & ~kBegins;
        v[k] = load_once<T, G>(from + at * stride, o.dim);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if ((w[k].y & kBegins) && j0 + k > 0) {
          runs.finish(row, sum, left, false);
          left = false;
          row = w[k].x;
          if (row == kNowhere) break;  // (no rows from here on)
          sum = Wide<T>{};
        }
        sum += widen<T>(v[k]);
      }
    }
    if (row != kNowhere) runs.finish(row, sum, left, !(mine[size].y & kBegins));
  }
  runs.join();
}

// Two entries that an earlier launch left a group, of m; sums_in as RunsOut::sums.
template <typename T, int G>
__global__ void __launch_bounds__(groups_in(kJoinMost, G) * G)
join_runs_kernel(const Entry* __restrict__ in, int64_t m, const float* __restrict__ sums_in, RunsOut o,
                 T* __restrict__ out) {
  constexpr int kGroups = groups_in(kJoinMost, G);
  __shared__ typename Runs<T, G, kGroups>::Shared s_runs;
  Runs<T, G, kGroups> runs(o, s_runs, out);
  const int64_t base = 2 * (runs.part * kGroups + runs.group);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (base + k >= m) continue;
    const Entry e = in[base + k];
    Wide<T> v;  // (asked for before it is known whether there is one: nothing is added where there is none)
    __builtin_memcpy(&v, sums_in + ((base + k) * o.chunks + runs.chunk) * Chunk<T>::kVec, sizeof(v));
    s_runs.sum[2 * runs.group + k][runs.lane] = v;
    if (runs.lane == 0) s_runs.entry[2 * runs.group + k] = e;
  }
  runs.join();
}

// ------------------------------------------------------------------- plans ----
// The workgroups of every launch: a function of the sizes alone.
constexpr int kMaxLevels = 8;
// n below 2^31 (short tiles are for lists of fewer than 2^23 lanes, which need no more levels than the longest one)
constexpr int most_levels(int lanes) {
  const int64_t joins = groups_in(kJoinMost, lanes);
  int64_t p = (int64_t(1) << 31) / (kMostSize * groups_in(kSumMost, lanes));
  int levels = 1;
  for (; p > 1; p = (p + joins - 1) / joins) ++levels;
  return levels;
}
static_assert(most_levels(1) <= kMaxLevels && most_levels(16) <= kMaxLevels && most_levels(32) <= kMaxLevels &&
              most_levels(kWave) <= kMaxLevels, "launches of the longest list");
// Whether a call takes these sizes: what it does not take has no plan.
bool has_plan(int64_t n, int64_t dim, int type) {
  return n > 0 && n < (int64_t(1) << 31) && dim < (int64_t(1) << 24) && (type == GS_F32 || type == GS_F16 || type == GS_BF16);
}

struct SumPlan {
  int64_t n, chunks;
  int group, slices;  // lanes a group, workgroups over a row
  int size;           // positions a group of the first launch
  int levels;
  int64_t parts[kMaxLevels];  // workgroups along the list

  SumPlan(int64_t n_, int64_t dim, int type) : n(n_) {
    chunks = type == GS_F32 ? chunks_of<float>(dim) : chunks_of<_Float16>(dim);
    group = 1;
    while (group < kWave && group < chunks) group *= 2;
    slices = static_cast<int>((chunks + group - 1) / group);
    const int groups = groups_in(kSumMost, group), joins = groups_in(kJoinMost, group);
    // as long as there are waves enough for the chip, longer tiles leave fewer partial sums
    size = kMostSize;
    while (size > 8 && (n / size) * slices * group < int64_t(256) * 16 * kWave) size /= 2;
    levels = 0;
    int64_t p = (n + int64_t(size) * groups - 1) / (int64_t(size) * groups);
    parts[levels++] = p;
    while (p > 1) {
      p = (p + joins - 1) / joins;
      parts[levels++] = p;
    }
  }
  int vec(int type) const { return 16 / value_bytes(type); }
  size_t sums_bytes(int level, int type) const {
    return static_cast<size_t>(2 * parts[level]) * chunks * vec(type) * sizeof(float);
  }
};

struct GradSpace {
  key_sort::Space sort;
  key_sort::Word* sorted;
  int64_t* counts;      // sparse: runs that begin in each workgroup's positions
  int64_t* heads;       // sparse: and before them
  int64_t* scan_tiles;  // sparse
  Entry* entries[2];
  float* sums[2];
};

// even levels write buffer 0, odd ones buffer 1, each sized for the first of them
size_t grad_bytes(const SumPlan& p, int type, bool sparse) {
  // (sorted lies in one of the sort's own buffers where it has any)
  size_t bytes = p.n <= key_sort::kAlone ? padded(static_cast<size_t>(p.n) * 8) : key_sort::space_bytes(p.n, 2);
  if (sparse)
    bytes += padded(static_cast<size_t>(p.parts[0]) * 8) + padded(static_cast<size_t>(p.parts[0] + 1) * 8) +
             scan_workspace_bytes(p.parts[0]);
  for (int l = 0; l < 2 && l + 1 < p.levels; ++l)
    bytes += padded(static_cast<size_t>(2 * p.parts[l]) * sizeof(Entry)) + padded(p.sums_bytes(l, type));
  return bytes;
}

bool carve_grad(Carver& ws, const SumPlan& p, int type, uint32_t num_rows, bool sparse, GradSpace* s) {
  key_sort::carve(ws, p.n, 2, &s->sort);
  s->sorted = p.n <= key_sort::kAlone ? ws.take<key_sort::Word>(static_cast<size_t>(p.n))
                                      : s->sort.word[(key_sort::Digits(num_rows).passes - 1) & 1];
  s->counts = sparse ? ws.take<int64_t>(static_cast<size_t>(p.parts[0])) : nullptr;
  s->heads = sparse ? ws.take<int64_t>(static_cast<size_t>(p.parts[0] + 1)) : nullptr;
  s->scan_tiles = sparse ? ws.take<int64_t>(scan_workspace_bytes(p.parts[0]) / 8) : nullptr;
  for (int l = 0; l < 2; ++l) {
    s->entries[l] = nullptr;
    s->sums[l] = nullptr;
    if (l + 1 < p.levels) {
      s->entries[l] = ws.take<Entry>(static_cast<size_t>(2 * p.parts[l]));
      s->sums[l] = ws.take<float>(p.sums_bytes(l, type) / sizeof(float));
    }
  }
  return ws.ok;
}

template <typename F>
void with_group(int group, F&& f) {
  switch (group) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    case 16: f(std::integral_constant<int, 16>()); break;
    case 32: f(std::integral_constant<int, 32>()); break;
    default: f(std::integral_constant<int, 64>()); break;
  }
}

template <typename T>
void launch_sums(const SumPlan& p, const GradSpace& s, uint32_t num_rows, const T* grad, int64_t stride, int64_t dim,
                 float scale, int64_t* met, T* out, hipStream_t st) {
  with_group(p.group, [&](auto g) {
    constexpr int G = decltype(g)::value;
    for (int l = 0; l < p.levels; ++l) {
      const bool last = l == p.levels - 1;
      const RunsOut o{scale, results_past(out, dim, false), dim, p.chunks, p.slices, met, s.heads,
                      last ? nullptr : s.entries[l & 1], last ? nullptr : s.sums[l & 1]};
      const dim3 grid(static_cast<unsigned>(p.parts[l] * p.slices));
      if (l == 0)
        hipLaunchKernelGGL((met ? sum_runs_kernel<T, G, true> : sum_runs_kernel<T, G, false>), grid,
                           dim3(groups_in(kSumMost, G) * G), 0, st, s.sorted, p.n, num_rows, grad, stride, p.size, o, out);
      else
        hipLaunchKernelGGL((join_runs_kernel<T, G>), grid, dim3(groups_in(kJoinMost, G) * G), 0, st,
                           s.entries[(l - 1) & 1], 2 * p.parts[l - 1], s.sums[(l - 1) & 1], o, out);
    }
  });
}

struct Numbers {
  const int64_t* number;
  __device__ __forceinline__ int64_t operator()(int64_t i) const { return number[i]; }
};

template <typename IdT, typename Beside>
void sort_ids(const IdT* ids, int64_t n, uint32_t num_rows, const GradSpace& s, Beside beside, hipStream_t st) {
  const key_sort::IdWords<IdT> src{ids, num_rows};
  key_sort::sort<false>(src, n, num_rows, s.sort, key_sort::WordsOut{s.sorted}, st, beside);
}

int check_rows(const char* what, const void* rows, int64_t stride, int64_t dim, int type, int64_t n, int64_t num_rows) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16, "%s: value type %d is none of GS_F32, GS_F16, GS_BF16",
             what, type);
  GS_REQUIRE(n >= 0 && n < (int64_t(1) << 31), "%s: %lld ids, at most 2^31 - 1 are taken", what, static_cast<long long>(n));
  GS_REQUIRE(num_rows >= 0 && num_rows < (int64_t(1) << 32) - 1, "%s: %lld rows, at most 2^32 - 2 are taken", what,
             static_cast<long long>(num_rows));
  GS_REQUIRE(dim >= 0 && dim < (int64_t(1) << 24), "%s: rows of %lld values, at most 2^24 - 1 are taken", what,
             static_cast<long long>(dim));
  GS_REQUIRE(stride >= 0, "%s: negative stride", what);
  GS_REQUIRE(aligned_to(rows, value_bytes(type)), "%s: rows not aligned to their type", what);
  return GS_OK;
}
int check_ids(const char* what, const void* ids, int id_bytes, int64_t n) {
  GS_REQUIRE(valid_id_bytes(id_bytes), "%s: id_bytes must be 4 or 8, got %d", what, id_bytes);
  GS_REQUIRE(n == 0 || ids, "%s: ids is null", what);
  GS_REQUIRE(aligned_to(ids, id_bytes), "%s: ids not aligned to their type", what);
  return GS_OK;
}
// whether every launch of the sums has a grid that can be launched
int check_plan(const char* what, const SumPlan& p) {
  GS_RETURN_IF_ERROR(check_grid(what, p.parts[0] * p.slices, groups_in(kSumMost, p.group) * p.group));
  return p.levels > 1 ? check_grid(what, p.parts[1] * p.slices, groups_in(kJoinMost, p.group) * p.group) : int(GS_OK);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

int gs_embedding_lookup(const void* table, int64_t num_rows, int64_t row_stride, int64_t dim, int type,
                        const void* ids, int id_bytes, int64_t n, float scale, void* out, void* stream) {
  GS_RETURN_IF_ERROR(check_rows("gs_embedding_lookup", table, row_stride, dim, type, n, num_rows));
  GS_RETURN_IF_ERROR(check_ids("gs_embedding_lookup", ids, id_bytes, n));
  if (n == 0 || dim == 0) return GS_OK;
  GS_REQUIRE(out && (table || num_rows == 0), "gs_embedding_lookup: null array");
  GS_REQUIRE(aligned_to(out, value_bytes(type)), "gs_embedding_lookup: out not aligned to its type");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return with_value_type(type, "gs_embedding_lookup", [&](auto zero) {
    using T = decltype(zero);
    const int64_t chunks = chunks_of<T>(dim), total = n * chunks;
    // four chunks a lane where that still leaves a workgroup for every compute unit
    constexpr int kMany = 4;
    const bool many = total >= int64_t(256) * kThreads * kMany;
    const int64_t blocks = (total + kThreads * (many ? kMany : 1) - 1) / (kThreads * (many ? kMany : 1));
    GS_RETURN_IF_ERROR(check_grid("gs_embedding_lookup", blocks, kThreads));
    const Divider by(static_cast<uint32_t>(chunks));
    return with_id_type(id_bytes, [&](auto id) {
      using IdT = decltype(id);
      auto* kernel = many ? lookup_kernel<T, IdT, kMany> : lookup_kernel<T, IdT, 1>;
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st,
                         static_cast<const T*>(table), num_rows, row_stride, dim, by, static_cast<const IdT*>(ids), total,
                         scale, static_cast<T*>(out), results_past(static_cast<const T*>(out), dim, true));
      return check_launch("embedding_lookup");
    });
  });
}

size_t gs_embedding_grad_workspace_bytes(int64_t n, int64_t dim, int type) {
  if (!has_plan(n, dim, type) || dim <= 0) return 256;  // (the call needs none, or refuses)
  return grad_bytes(SumPlan(n, dim, type), type, false);
}

int gs_embedding_grad(const void* grad, int64_t grad_stride, int64_t dim, int type, const void* ids, int id_bytes,
                      int64_t n, int64_t num_rows, float scale, void* out, void* workspace, size_t workspace_bytes,
                      void* stream) {
  GS_RETURN_IF_ERROR(check_rows("gs_embedding_grad", grad, grad_stride, dim, type, n, num_rows));
  GS_RETURN_IF_ERROR(check_ids("gs_embedding_grad", ids, id_bytes, n));
  if (num_rows == 0 || dim == 0) return GS_OK;
  GS_REQUIRE(out && (grad || n == 0), "gs_embedding_grad: null array");
  GS_REQUIRE(aligned_to(out, value_bytes(type)), "gs_embedding_grad: out not aligned to its type");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const SumPlan plan(n > 0 ? n : 1, dim, type);
  GS_RETURN_IF_ERROR(check_plan("gs_embedding_grad", plan));
  GradSpace space;
  if (n > 0) {
    Carver ws(workspace, workspace_bytes);
    if (!carve_grad(ws, plan, type, static_cast<uint32_t>(num_rows), false, &space)) {
      set_error_text("gs_embedding_grad: workspace needs %zu bytes, 256-byte aligned",
                     gs_embedding_grad_workspace_bytes(n, dim, type));
      return GS_ERR_WORKSPACE;
    }
  }
  return with_value_type(type, "gs_embedding_grad", [&](auto zero) {
    using T = decltype(zero);
    Zeros<T> zeros{static_cast<T*>(out), num_rows * dim};
    if (n > 0) {
      with_id_type(id_bytes, [&](auto id) {
        using IdT = decltype(id);
        sort_ids(static_cast<const IdT*>(ids), n, static_cast<uint32_t>(num_rows), space, zeros, st);
        return 0;
      });
      launch_sums(plan, space, static_cast<uint32_t>(num_rows), static_cast<const T*>(grad), grad_stride, dim, scale,
                  nullptr, static_cast<T*>(out), st);
    } else {
      hipLaunchKernelGGL(zero_kernel<T>, dim3(zeros.blocks(kThreads)), dim3(kThreads), 0, st, zeros);
    }
    return check_launch("embedding_grad");
  });
}

size_t gs_embedding_sparse_grad_workspace_bytes(int64_t n, int64_t dim, int type) {
  if (!has_plan(n, dim, type)) return 256;
  return grad_bytes(SumPlan(n, dim > 0 ? dim : 1, type), type, true);
}

int gs_embedding_sparse_grad_count(const void* ids, int id_bytes, int64_t n, int64_t num_rows, int64_t dim, int type,
                                   gs_mailbox* mailbox, int64_t ticket, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  GS_RETURN_IF_ERROR(check_rows("gs_embedding_sparse_grad_count", nullptr, 0, dim, type, n, num_rows));
  GS_RETURN_IF_ERROR(check_ids("gs_embedding_sparse_grad_count", ids, id_bytes, n));
  GS_REQUIRE(n > 0, "gs_embedding_sparse_grad_count: no ids");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const SumPlan plan(n, dim > 0 ? dim : 1, type);
  GradSpace space;
  Carver ws(workspace, workspace_bytes);
  const uint32_t rows = static_cast<uint32_t>(num_rows);
  if (!carve_grad(ws, plan, type, rows, true, &space)) {
    set_error_text("gs_embedding_sparse_grad_count: workspace needs %zu bytes, 256-byte aligned",
                   gs_embedding_sparse_grad_workspace_bytes(n, dim, type));
    return GS_ERR_WORKSPACE;
  }
  with_id_type(id_bytes, [&](auto id) {
    using IdT = decltype(id);
    sort_ids(static_cast<const IdT*>(ids), n, rows, space, key_sort::NoWork(), st);
    return 0;
  });
  hipLaunchKernelGGL(count_runs_kernel, dim3(static_cast<unsigned>(plan.parts[0])), dim3(kThreads), 0, st, space.sorted, n,
                     rows, plan.size * groups_in(kSumMost, plan.group), space.counts);
  return exclusive_scan(Numbers{space.counts}, plan.parts[0], space.heads, space.scan_tiles, st, mailbox, ticket);
}

int gs_embedding_sparse_grad_fill(const void* grad, int64_t grad_stride, int64_t dim, int type, int64_t n,
                                  int64_t num_rows, float scale, int64_t* met, void* values, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  GS_RETURN_IF_ERROR(check_rows("gs_embedding_sparse_grad_fill", grad, grad_stride, dim, type, n, num_rows));
  GS_REQUIRE(n > 0 && met && ((grad && values) || dim == 0), "gs_embedding_sparse_grad_fill: no ids or null array");
  GS_REQUIRE(aligned_to(values, value_bytes(type)), "gs_embedding_sparse_grad_fill: values not aligned to their type");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const SumPlan plan(n, dim > 0 ? dim : 1, type);
  GS_RETURN_IF_ERROR(check_plan("gs_embedding_sparse_grad_fill", plan));
  GradSpace space;
  Carver ws(workspace, workspace_bytes);
  const uint32_t rows = static_cast<uint32_t>(num_rows);
  if (!carve_grad(ws, plan, type, rows, true, &space)) {
    set_error_text("gs_embedding_sparse_grad_fill: workspace needs %zu bytes, 256-byte aligned",
                   gs_embedding_sparse_grad_workspace_bytes(n, dim, type));
    return GS_ERR_WORKSPACE;
  }
  return with_value_type(type, "gs_embedding_sparse_grad_fill", [&](auto zero) {
    using T = decltype(zero);
    launch_sums(plan, space, rows, static_cast<const T*>(grad), grad_stride, dim, scale, met, static_cast<T*>(values), st);
    return check_launch("embedding_sparse_grad_fill");
  });
}

}  // extern "C"
