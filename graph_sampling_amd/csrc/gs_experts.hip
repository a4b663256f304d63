// Rows sorted by expert and back, with weights applied, and the gradients, on gfx950.
//
// T tokens choose K experts of E each; item t * K + k is token t's k-th choice.  The items sorted by
// expert, stably, are the order in which the experts' rows lie:
//   place[t, k]            where item t * K + k lies, -1 when its choice names no expert
//   order[place[t, k]]     = t * K + k, -1 behind the last
//   gather   rows[place[t, k], :] = x[t, :], zeros behind the last
//   combine  out[t, :]     = sum over k of weights[t, k] * y[place[t, k], :]
//   its gradient: dy[place[t, k], :] = weights[t, k] * dout[t, :], dweights[t, k] = <dout[t, :], y[place[t, k], :]>
//   (the gradient of the gather is a combine without weights).
// No counterpart in the reference.  With one choice each, the experts may be node types or relations.
// Every row moves once: the kernels go by token, read its row once, and reach the experts' rows through
// `place`.  What bounds them is the rows' bytes; products and sums are fp32, rounded once at the end.
#include "gs_key_sort.hpp"
#include "gs_rows.hpp"

namespace gs {
namespace {

constexpr int kThreads = 256;

// -------------------------------------------------------------------- sort ----
// Sorted items of fewer than 512 experts (one pass, which knows where every expert begins).
struct OrderOut {
  int32_t* order;
  int32_t* place;
  int64_t* offsets;
  uint32_t experts;
  __device__ __forceinline__ void digit(uint32_t d, uint32_t start) const {
    if (d <= experts) offsets[d] = start;
  }
  __device__ __forceinline__ void from(key_sort::Word w, uint32_t at) const {
    place[key_sort::position_of(w)] = key_sort::key_of(w) < experts ? static_cast<int32_t>(at) : -1;
  }
  __device__ __forceinline__ void item(uint32_t at, key_sort::Word w) const {
    order[at] = key_sort::key_of(w) < experts ? static_cast<int32_t>(key_sort::position_of(w)) : -1;
  }
};

// The same from words sorted in several passes, and where the experts begin, by search.
__global__ void __launch_bounds__(kThreads)
order_kernel(const key_sort::Word* __restrict__ words, int64_t n, OrderOut out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i < n) {
    out.from(words[i], static_cast<uint32_t>(i));
    out.item(static_cast<uint32_t>(i), words[i]);
  }
  if (i <= static_cast<int64_t>(out.experts)) {
    int64_t lo = 0, hi = n;  // items of the experts before i
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (key_sort::key_of(words[mid]) < static_cast<uint32_t>(i)) lo = mid + 1; else hi = mid;
    }
    out.offsets[i] = lo;
  }
}
__global__ void __launch_bounds__(kThreads) no_items_kernel(int64_t* __restrict__ offsets, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    offsets[i] = 0;
}

// ------------------------------------------------------------------ gather ----
// Zeros in the rows from `from` to n, a share of them by every workgroup.
template <int THREADS = kThreads, typename T>
__device__ __forceinline__ void zero_rows_behind(int64_t from, int64_t n, int64_t dim, const Divider& chunks,
                                                 T* __restrict__ rows, Past past) {
  if (from >= n || from < 0) return;
  const int64_t total = (n - from) * chunks.d, stride = static_cast<int64_t>(gridDim.x) * THREADS;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x; i < total; i += stride) {
    const int64_t row = i / chunks.d;
    const int64_t at = chunk_start<T>(dim, i - row * chunks.d);
    store_result(rows + (from + row) * dim + at, Values<T>{}, at, dim, past);
  }
}

// A chunk of a token a lane (ITEMS of them): read once, written to every choice's place.
template <typename T, int ITEMS>
__global__ void __launch_bounds__(kThreads)
gather_kernel(const T* __restrict__ x, int64_t stride, int64_t dim, Divider chunks, const int32_t* __restrict__ place,
              int64_t total, int choices, int64_t n, const int64_t* __restrict__ live, T* __restrict__ rows, Past past) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kThreads * ITEMS);
  const RowRange range(chunks, first);
  int64_t token[ITEMS], at[ITEMS];
  Values<T> v[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const uint32_t j = i * kThreads + threadIdx.x;
    uint32_t c;
    token[i] = range.row(first + j < total ? j : 0, &c);
    at[i] = chunk_start<T>(dim, c);
    v[i] = load_chunk(x + token[i] * stride + at[i], dim);
    if (first + j >= total) token[i] = -1;
  }
  for (int k = 0; k < choices; ++k) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      if (token[i] < 0) continue;
      const int64_t to = place[token[i] * choices + k];
      if (to >= 0 && to < n) store_result(rows + to * dim + at[i], v[i], at[i], dim, past);
    }
  }
  zero_rows_behind(*live, n, dim, chunks, rows, past);
}

// The same with the sort, for a few items: every workgroup ranks all of them in LDS, which takes less than a launch,
// and goes on with its chunks; the first one writes the order down.  16 items of 64 experts: 4 us where two launches
// take 6 and the space between them; 8 of 256 experts, the whole call: 8.9 us for 16.5.
constexpr int64_t kDispatchItems = kThreads * key_sort::kItems;
constexpr int dispatch_threads(int bits) { return bits == 9 ? 512 : kThreads; }  // (a thread a digit)

template <typename T, typename IdT, int BITS>
__global__ void __launch_bounds__(dispatch_threads(BITS))
sort_gather_kernel(const IdT* __restrict__ experts, const T* __restrict__ x, int64_t stride, int64_t dim, Divider chunks,
                   int64_t total, int choices, uint32_t n, OrderOut out, T* __restrict__ rows, Past past) {
  constexpr int kDigits = 1 << BITS, kThreadsHere = dispatch_threads(BITS);
  __shared__ key_sort::TileTables<BITS, kThreadsHere> s_tables;
  __shared__ uint32_t s_start[kDigits];
  __shared__ int32_t s_place[kDispatchItems];
  // the token's chunk is on its way meanwhile
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreadsHere;
  const bool in = first + threadIdx.x < total;
  const RowRange range(chunks, first);
  uint32_t c;
  const int64_t token = range.row(in ? threadIdx.x : 0, &c), at = chunk_start<T>(dim, c);
  const Values<T> v = load_chunk(x + token * stride + at, dim);

  const key_sort::IdWords<IdT> src{experts, out.experts};
  key_sort::Word w[key_sort::kItems];
  uint32_t d[key_sort::kItems], rank[key_sort::kItems], here;
#pragma unroll
  for (int r = 0; r < key_sort::kItems; ++r) {
    const uint32_t i = key_sort::item_of(r);
    w[r] = src(i < n ? i : n - 1);
    d[r] = key_sort::digit_of<BITS>(w[r], 0);
  }
  key_sort::rank_tile<BITS, kThreadsHere>(d, n, s_tables, rank, &here);
  uint32_t start = here, none = 0;
  key_sort::scan_digits(start, none, s_tables);
  if (threadIdx.x < kDigits) {
    s_start[threadIdx.x] = start;
    if (blockIdx.x == 0) out.digit(threadIdx.x, start);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < key_sort::kItems; ++r) {
    const uint32_t i = key_sort::item_of(r);
    if (i >= n) continue;
    const uint32_t to = s_start[d[r]] + rank[r];
    s_place[i] = key_sort::key_of(w[r]) < out.experts ? static_cast<int32_t>(to) : -1;
    if (blockIdx.x == 0) {
      out.from(w[r], to);
      out.item(to, w[r]);
    }
  }
  __syncthreads();
  if (in) {
    for (int k = 0; k < choices; ++k) {
      const int32_t to = s_place[token * choices + k];
      if (to >= 0) store_result(rows + to * dim + at, v, at, dim, past);
    }
  }
  const int64_t live = s_start[out.experts];
  if (live < n) zero_rows_behind<kThreadsHere>(live, static_cast<int64_t>(n), dim, chunks, rows, past);
}

// ----------------------------------------------------------------- combine ----
template <typename W>
__device__ __forceinline__ float weight_of(const W* weights, int64_t item) {
  return weights ? static_cast<float>(weights[item]) : 1.0f;
}

// A chunk of a token's sum a lane; the rows of KU choices are asked for together.
template <typename T, typename W, int KU>
__global__ void __launch_bounds__(kThreads)
combine_kernel(const T* __restrict__ y, int64_t stride, int64_t dim, Divider chunks, const int32_t* __restrict__ place,
               int64_t total, int choices, int64_t n, const W* __restrict__ weights, T* __restrict__ out, Past past) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads;
  if (first + threadIdx.x >= total) return;
  const RowRange range(chunks, first);
  uint32_t c;
  const int64_t token = range.row(threadIdx.x, &c), at = chunk_start<T>(dim, c);
  Wide<T> sum = {};
  for (int k0 = 0; k0 < choices; k0 += KU) {
    Values<T> v[KU];
    float w[KU];
    bool there[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const int64_t item = token * choices + (k0 + u < choices ? k0 + u : k0);
      const int64_t from = place[item];
      there[u] = k0 + u < choices && from >= 0 && from < n;
      w[u] = weight_of(weights, item);
      v[u] = Values<T>{};
      if (there[u]) v[u] = load_chunk(y + from * stride + at, dim);
    }
#pragma unroll
    for (int u = 0; u < KU; ++u)
      if (there[u]) sum += widen<T>(v[u]) * w[u];
  }
  store_result(out + token * dim + at, narrow<T>(sum), at, dim, past);
}

// ---------------------------------------------------- gradient of the combine ----
// A group of G lanes a token (or a whole workgroup, WAVES = 4): dout's chunk is read once for KU
// choices, y's rows give the weights' gradients, dy's rows are written.
template <typename T, typename W, int G, int WAVES, int KU>
__global__ void __launch_bounds__(kThreads)
combine_grad_kernel(const T* __restrict__ dout, int64_t dout_stride, const T* __restrict__ y, int64_t y_stride,
                    int64_t dim, Divider chunks, const int32_t* __restrict__ place, int64_t tokens, int choices,
                    int64_t n, const int64_t* __restrict__ live, const W* __restrict__ weights, T* __restrict__ dy,
                    W* __restrict__ dweights, Past past) {
  constexpr int kLanes = G * WAVES;               // of a token
  constexpr int kTokens = kThreads / kLanes;      // of a workgroup
  __shared__ float s_dots[WAVES > 1 ? WAVES * KU : 1];
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int64_t token = t < tokens ? t : tokens - 1;  // (works along, writes nothing)
  for (int k0 = 0; k0 < choices; k0 += KU) {
    int64_t from[KU];
    float w[KU], dot[KU];
#pragma unroll
    for (int u = 0; u < KU; ++u) {
      const int64_t item = token * choices + (k0 + u < choices ? k0 + u : k0);
      from[u] = place[item];
      w[u] = weight_of(weights, item);
      dot[u] = 0.0f;
      if (k0 + u >= choices || from[u] < 0 || from[u] >= n || t >= tokens) from[u] = -1;
    }
    for (int64_t c = lane; c < chunks.d; c += kLanes) {
      const int64_t at = chunk_start<T>(dim, c);
      const int64_t overlap = c * Chunk<T>::kVec - at;  // values of the chunk before
      const Wide<T> d = widen<T>(load_chunk(dout + token * dout_stride + at, dim));
      Values<T> v[KU];
      if (dweights) {
#pragma unroll
        for (int u = 0; u < KU; ++u) {
          v[u] = Values<T>{};
          // (past the caches: y is read for the last time, and dy needs their room: 50 k tokens, 4 rows of 512
          // bf16 each, from memory 91 us plain and 86 so; of 500, whose dy is written plainly, 101 and 106, and the same
          // rows every call 100 and 88)
          const T* const at_y = y + (from[u] >= 0 ? from[u] * y_stride + at : 0);
          if (from[u] >= 0) v[u] = dim >= Chunk<T>::kVec ? load_past(at_y) : load_chunk(at_y, dim);
        }
      }
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        if (dweights && from[u] >= 0) {
          const Wide<T> b = widen<T>(v[u]);
#pragma unroll
          for (int i = 0; i < Chunk<T>::kVec; ++i)
            if (i >= overlap) dot[u] = __fmaf_rn(d[i], b[i], dot[u]);
        }
        if (dy && from[u] >= 0) store_result(dy + from[u] * dim + at, narrow<T>(d * w[u]), at, dim, past);
      }
    }
    if (!dweights) continue;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
      for (int m = G / 2; m > 0; m /= 2) dot[u] += __shfl_xor(dot[u], m, kWave);
    if (WAVES > 1) {
      if (lane % kWave == 0) {
#pragma unroll
        for (int u = 0; u < KU; ++u) s_dots[(lane / kWave) * KU + u] = dot[u];
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < KU; ++u) {
        dot[u] = 0.0f;
        for (int wv = 0; wv < WAVES; ++wv) dot[u] += s_dots[wv * KU + u];
      }
      __syncthreads();
    }
    if (lane == 0 && t < tokens) {
#pragma unroll
      for (int u = 0; u < KU; ++u)
        if (k0 + u < choices) dweights[token * choices + k0 + u] = static_cast<W>(from[u] >= 0 ? dot[u] : 0.0f);
    }
  }
  if (dy) zero_rows_behind(*live, n, dim, chunks, dy, past);
}

// ------------------------------------------------------------------- checks ----
int check_shape(const char* what, int64_t tokens, int64_t choices, int64_t experts) {
  GS_REQUIRE(tokens >= 0 && choices >= 0 && experts >= 0, "%s: negative size", what);
  GS_REQUIRE(choices < (int64_t(1) << 31) && (choices == 0 || tokens <= ((int64_t(1) << 31) - 1) / choices),
             "%s: tokens x choices, at most 2^31 - 1 are taken", what);
  GS_REQUIRE(experts < (int64_t(1) << 31), "%s: %lld experts, at most 2^31 - 1 are taken", what,
             static_cast<long long>(experts));
  return GS_OK;
}
int check_values(const char* what, int type, int64_t dim, int64_t stride) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16, "%s: value type %d is none of GS_F32, GS_F16, GS_BF16",
             what, type);
  GS_REQUIRE(dim >= 0 && dim < (int64_t(1) << 24), "%s: rows of %lld values, at most 2^24 - 1 are taken", what,
             static_cast<long long>(dim));
  GS_REQUIRE(stride >= 0, "%s: negative stride", what);
  return GS_OK;
}

// weights are fp32 or of the rows' type
template <typename T, typename F>
int with_weight_type(int type, int weight_type, const char* what, F&& f) {
  if (weight_type == GS_F32) return f(float(0));
  if (weight_type == type) return f(T(0));
  set_error_text("%s: weights are fp32 or of the rows' type", what);
  return GS_ERR_INVALID_ARG;
}
template <typename F>
void with_choices(int64_t choices, F&& f) {
  if (choices <= 1) f(std::integral_constant<int, 1>());
  else if (choices == 2) f(std::integral_constant<int, 2>());
  else if (choices <= 4) f(std::integral_constant<int, 4>());
  else f(std::integral_constant<int, 8>());
}

template <typename T>
int launch_gather(const T* x, int64_t stride, int64_t dim, const int32_t* place, int64_t tokens, int64_t choices,
                  const int64_t* live, T* rows, hipStream_t st, const char* what) {
  const int64_t chunks = chunks_of<T>(dim), total = tokens * chunks;
  constexpr int kMany = 4;
  const bool many = total >= int64_t(256) * 4 * kThreads * kMany;
  const int64_t blocks = (total + kThreads * (many ? kMany : 1) - 1) / (kThreads * (many ? kMany : 1));
  GS_RETURN_IF_ERROR(check_grid(what, blocks, kThreads));
  auto* kernel = many ? gather_kernel<T, kMany> : gather_kernel<T, 1>;
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, st, x, stride, dim,
                     Divider(static_cast<uint32_t>(chunks)), place, total, static_cast<int>(choices), tokens * choices, live,
                     rows, results_past(rows, dim, false));
  return check_launch(what);
}

template <typename T, typename W, int G, int WAVES>
int launch_combine_grad(const T* dout, int64_t dout_stride, const T* y, int64_t y_stride, int64_t dim,
                        const int32_t* place, int64_t tokens, int64_t choices, const int64_t* live, const W* weights,
                        T* dy, W* dweights, hipStream_t st) {
  constexpr int kTokens = kThreads / (G * WAVES);
  constexpr int64_t kMost = most_blocks(kThreads) * kTokens;  // tokens a launch
  const auto past = results_past(dy, dim, false);
  // (rows of eight choices at once take registers that waves need: 25 k tokens, 8 choices of 500 bf16, 123 us; four 107)
  for (int64_t t = 0; t < tokens; t += kMost) {
    const int64_t here = tokens - t < kMost ? tokens - t : kMost, item = t * choices;
    const dim3 grid(static_cast<unsigned>((here + kTokens - 1) / kTokens));
    with_choices(choices < 4 ? choices : 4, [&](auto ku) {
      hipLaunchKernelGGL((combine_grad_kernel<T, W, G, WAVES, decltype(ku)::value>), grid, dim3(kThreads), 0, st,
                         dout + t * dout_stride, dout_stride, y, y_stride, dim,
                         Divider(static_cast<uint32_t>(chunks_of<T>(dim))), place + item, here,
                         static_cast<int>(choices), tokens * choices, live, weights ? weights + item : nullptr, dy,
                         dweights ? dweights + item : nullptr, past);
    });
    GS_RETURN_IF_ERROR(check_launch("expert_combine_grad"));
  }
  return GS_OK;
}

template <typename IdT>
int sort_items(const IdT* experts, int64_t n, int64_t num_experts, const OrderOut& out, void* workspace,
               size_t workspace_bytes, hipStream_t st) {
  if (n == 0) {
    const int64_t offsets = num_experts + 1;
    hipLaunchKernelGGL(no_items_kernel, dim3(blocks_for(offsets < (1 << 20) ? offsets : (1 << 20), kThreads)),
                       dim3(kThreads), 0, st, out.offsets, offsets);
    return check_launch("expert_sort");
  }
  const uint32_t num = static_cast<uint32_t>(num_experts);
  const int passes = key_sort::Digits(num).passes;
  Carver ws(workspace, workspace_bytes);
  key_sort::Space space;
  key_sort::carve(ws, n, passes > 1 ? 2 : 0, &space);
  key_sort::Word* sorted = nullptr;  // (in one of the sort's own buffers where it has any)
  if (passes > 1)
    sorted = n <= key_sort::kAlone ? ws.take<key_sort::Word>(static_cast<size_t>(n)) : space.word[(passes - 1) & 1];
  if (!ws.ok) {
    set_error_text("gs_expert_sort: workspace needs %zu bytes, 256-byte aligned",
                   gs_expert_sort_workspace_bytes(n, num_experts));
    return GS_ERR_WORKSPACE;
  }
  const key_sort::IdWords<IdT> src{experts, num};
  if (passes == 1) {
    key_sort::sort<true>(src, n, num, space, out, st);
  } else {
    key_sort::sort<false>(src, n, num, space, key_sort::WordsOut{sorted}, st);
    const int64_t threads = n > num_experts + 1 ? n : num_experts + 1;
    hipLaunchKernelGGL(order_kernel, dim3(static_cast<unsigned>((threads + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                       st, sorted, n, out);
  }
  return check_launch("expert_sort");
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

size_t gs_expert_sort_workspace_bytes(int64_t n, int64_t num_experts) {
  if (n <= 0 || num_experts < 0) return 256;
  const uint32_t num = static_cast<uint32_t>(num_experts);
  const bool words = key_sort::Digits(num).passes > 1;
  if (n <= key_sort::kAlone) return words ? padded(static_cast<size_t>(n) * 8) : 0;
  return key_sort::space_bytes(n, words ? 2 : 0);
}

int gs_expert_sort(const void* experts, int id_bytes, int64_t n, int64_t num_experts, int32_t* order, int32_t* place,
                   int64_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  GS_RETURN_IF_ERROR(check_shape("gs_expert_sort", n, 1, num_experts));
  GS_REQUIRE(valid_id_bytes(id_bytes), "gs_expert_sort: id_bytes must be 4 or 8, got %d", id_bytes);
  GS_REQUIRE(offsets && (n == 0 || (experts && order && place)), "gs_expert_sort: null array");
  GS_REQUIRE(aligned_to(experts, id_bytes), "gs_expert_sort: ids not aligned to their type");
  const OrderOut out{order, place, offsets, static_cast<uint32_t>(num_experts)};
  return with_id_type(id_bytes, [&](auto id) {
    using IdT = decltype(id);
    return sort_items(static_cast<const IdT*>(experts), n, num_experts, out, workspace, workspace_bytes,
                      static_cast<hipStream_t>(stream));
  });
}

int gs_expert_gather(const void* x, int64_t x_stride, int64_t dim, int type, const int32_t* place, int64_t tokens,
                     int64_t choices, const int64_t* live, void* rows, void* stream) {
  GS_RETURN_IF_ERROR(check_shape("gs_expert_gather", tokens, choices, 0));
  GS_RETURN_IF_ERROR(check_values("gs_expert_gather", type, dim, x_stride));
  if (tokens == 0 || choices == 0 || dim == 0) return GS_OK;
  GS_REQUIRE(x && place && live && rows, "gs_expert_gather: null array");
  GS_REQUIRE(aligned_to(x, value_bytes(type)) && aligned_to(rows, value_bytes(type)),
             "gs_expert_gather: rows not aligned to their type");
  return with_value_type(type, "gs_expert_gather", [&](auto zero) {
    using T = decltype(zero);
    return launch_gather(static_cast<const T*>(x), x_stride, dim, place, tokens, choices, live, static_cast<T*>(rows),
                         static_cast<hipStream_t>(stream), "gs_expert_gather");
  });
}

int gs_expert_dispatch(const void* x, int64_t x_stride, int64_t dim, int type, const void* experts, int id_bytes,
                       int64_t tokens, int64_t choices, int64_t num_experts, int32_t* order, int32_t* place,
                       int64_t* offsets, void* rows, void* workspace, size_t workspace_bytes, void* stream) {
  GS_RETURN_IF_ERROR(check_shape("gs_expert_dispatch", tokens, choices, num_experts));
  GS_RETURN_IF_ERROR(check_values("gs_expert_dispatch", type, dim, x_stride));
  const int64_t n = tokens * choices;
  if (n == 0 || n > kDispatchItems || num_experts >= 512 || dim == 0) {
    GS_RETURN_IF_ERROR(gs_expert_sort(experts, id_bytes, n, num_experts, order, place, offsets, workspace,
                                      workspace_bytes, stream));
    return gs_expert_gather(x, x_stride, dim, type, place, tokens, choices, offsets + num_experts, rows, stream);
  }
  GS_REQUIRE(valid_id_bytes(id_bytes), "gs_expert_dispatch: id_bytes must be 4 or 8, got %d", id_bytes);
  GS_REQUIRE(x && experts && order && place && offsets && rows, "gs_expert_dispatch: null array");
  GS_REQUIRE(aligned_to(experts, id_bytes) && aligned_to(x, value_bytes(type)) && aligned_to(rows, value_bytes(type)),
             "gs_expert_dispatch: ids or rows not aligned to their type");
  const OrderOut out{order, place, offsets, static_cast<uint32_t>(num_experts)};
  return with_value_type(type, "gs_expert_dispatch", [&](auto zero) {
    using T = decltype(zero);
    return with_id_type(id_bytes, [&](auto id) {
      using IdT = decltype(id);
      const int bits = key_sort::Digits(static_cast<uint32_t>(num_experts), true).bits, threads = dispatch_threads(bits);
      const int64_t chunks = chunks_of<T>(dim), total = tokens * chunks, blocks = (total + threads - 1) / threads;
      GS_RETURN_IF_ERROR(check_grid("gs_expert_dispatch", blocks, threads));
      auto* kernel = bits == 4   ? sort_gather_kernel<T, IdT, 4>
                     : bits == 7 ? sort_gather_kernel<T, IdT, 7>
                     : bits == 8 ? sort_gather_kernel<T, IdT, 8>
                                 : sort_gather_kernel<T, IdT, 9>;
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(threads), 0,
                         static_cast<hipStream_t>(stream), static_cast<const IdT*>(experts), static_cast<const T*>(x),
                         x_stride, dim, Divider(static_cast<uint32_t>(chunks)), total, static_cast<int>(choices),
                         static_cast<uint32_t>(n), out, static_cast<T*>(rows),
                         results_past(static_cast<const T*>(rows), dim, false));
      return check_launch("expert_dispatch");
    });
  });
}

int gs_expert_combine(const void* y, int64_t y_stride, int64_t dim, int type, const int32_t* place, int64_t tokens,
                      int64_t choices, const void* weights, int weight_type, void* out, void* stream) {
  GS_RETURN_IF_ERROR(check_shape("gs_expert_combine", tokens, choices, 0));
  GS_RETURN_IF_ERROR(check_values("gs_expert_combine", type, dim, y_stride));
  if (tokens == 0 || dim == 0) return GS_OK;
  GS_REQUIRE(out && (choices == 0 || (y && place)), "gs_expert_combine: null array");
  GS_REQUIRE(aligned_to(y, value_bytes(type)) && aligned_to(out, value_bytes(type)),
             "gs_expert_combine: rows not aligned to their type");
  return with_value_type(type, "gs_expert_combine", [&](auto zero) {
    using T = decltype(zero);
    return with_weight_type<T>(type, weights ? weight_type : GS_F32, "gs_expert_combine", [&](auto wzero) {
      using W = decltype(wzero);
      const int64_t chunks = chunks_of<T>(dim), most = most_blocks(kThreads) * kThreads / chunks;  // tokens a launch
      const auto past = results_past(static_cast<const T*>(out), dim, true);
      for (int64_t t = 0; t < tokens; t += most) {
        const int64_t here = tokens - t < most ? tokens - t : most, total = here * chunks, item = t * choices;
        const dim3 grid(static_cast<unsigned>((total + kThreads - 1) / kThreads));
        with_choices(choices, [&](auto ku) {
          hipLaunchKernelGGL((combine_kernel<T, W, decltype(ku)::value>), grid, dim3(kThreads), 0,
                             static_cast<hipStream_t>(stream), static_cast<const T*>(y), y_stride, dim,
                             Divider(static_cast<uint32_t>(chunks)), place ? place + item : nullptr, total,
                             static_cast<int>(choices), tokens * choices,
                             weights ? static_cast<const W*>(weights) + item : nullptr,
                             static_cast<T*>(out) + t * dim, past);
        });
        GS_RETURN_IF_ERROR(check_launch("expert_combine"));
      }
      return static_cast<int>(GS_OK);
    });
  });
}

int gs_expert_combine_grad(const void* dout, int64_t dout_stride, const void* y, int64_t y_stride, int64_t dim, int type,
                           const int32_t* place, int64_t tokens, int64_t choices, const int64_t* live,
                           const void* weights, int weight_type, void* dy, void* dweights, void* stream) {
  GS_RETURN_IF_ERROR(check_shape("gs_expert_combine_grad", tokens, choices, 0));
  GS_RETURN_IF_ERROR(check_values("gs_expert_combine_grad", type, dim, dout_stride));
  GS_REQUIRE(y_stride >= 0, "gs_expert_combine_grad: negative stride");
  if (tokens == 0 || choices == 0 || (!dy && !dweights)) return GS_OK;
  GS_REQUIRE(place && live, "gs_expert_combine_grad: null array");
  GS_REQUIRE(dim == 0 || (dout && (!dweights || y)), "gs_expert_combine_grad: null array");
  GS_REQUIRE(aligned_to(dout, value_bytes(type)) && aligned_to(y, value_bytes(type)) && aligned_to(dy, value_bytes(type)),
             "gs_expert_combine_grad: rows not aligned to their type");
  return with_value_type(type, "gs_expert_combine_grad", [&](auto zero) {
    using T = decltype(zero);
    return with_weight_type<T>(type, weights || dweights ? weight_type : GS_F32, "gs_expert_combine_grad", [&](auto wzero) {
      using W = decltype(wzero);
      const int64_t chunks = chunks_of<T>(dim);
      auto go = [&](auto lanes, auto waves) {
        return launch_combine_grad<T, W, decltype(lanes)::value, decltype(waves)::value>(
            static_cast<const T*>(dout), dout_stride, static_cast<const T*>(y), y_stride, dim, place, tokens, choices,
            live, static_cast<const W*>(weights), static_cast<T*>(dy), static_cast<W*>(dweights),
            static_cast<hipStream_t>(stream));
      };
      using One = std::integral_constant<int, 1>;
      if (chunks <= 4) return go(std::integral_constant<int, 4>(), One());
      if (chunks <= 16) return go(std::integral_constant<int, 16>(), One());
      // (half a wave, too, where a whole one would idle for a third of its time: rows of 77 chunks, 8192 tokens of 3
      // choices 18.5 us for 22.4, 20 k of 4 62.6 for 61.6 from memory and 50.8 for 54.7 from the caches, 50 k of 2 86 for 77
      // and 62 for 64)
      if (chunks <= 32 || (tokens >= 4096 && chunks > kWave && chunks <= 85))
        return go(std::integral_constant<int, 32>(), One());
      if (chunks <= kWave || tokens >= 4096) return go(std::integral_constant<int, kWave>(), One());
      return go(std::integral_constant<int, kWave>(), std::integral_constant<int, kThreads / kWave>());
    });
  });
}

}  // extern "C"
