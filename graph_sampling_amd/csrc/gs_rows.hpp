// Rows of values moved by ids (embedding rows, rows sent to experts): the pieces that
// gs_embedding.hip and gs_experts.hip share.
#pragma once

#include "gs_common.hpp"

namespace gs {

// A row is moved in chunks of 16 bytes, one a lane.  Chunks are aligned like the values, not like
// themselves: rows of an odd width are read in the same way (the memory pipeline takes 16 bytes from
// any address here).  The last chunk of a row whose width is no multiple of the chunk starts
// earlier and overlaps the one before; its values are read, or written the same, twice.
template <typename T>
struct Chunk {
  static constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  typedef T Values __attribute__((ext_vector_type(kVec)));
  typedef float Wide __attribute__((ext_vector_type(kVec)));
};
template <typename T>
using Values = typename Chunk<T>::Values;
template <typename T>
using Wide = typename Chunk<T>::Wide;

// chunks of a row, at least one
template <typename T>
constexpr int64_t chunks_of(int64_t dim) {
  return dim <= Chunk<T>::kVec ? 1 : (dim + Chunk<T>::kVec - 1) / Chunk<T>::kVec;
}
// where chunk c of a row begins
template <typename T>
__device__ __forceinline__ int64_t chunk_start(int64_t dim, int64_t c) {
  const int64_t at = c * Chunk<T>::kVec, last = dim - Chunk<T>::kVec;
  return at < last ? at : (last > 0 ? last : 0);
}

// p: the chunk's first value; dim: the row's width (narrower rows than a chunk go value by value)
template <typename T>
__device__ __forceinline__ Values<T> load_chunk(const T* p, int64_t dim) {
  Values<T> v = {};
  if (dim >= Chunk<T>::kVec) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Chunk<T>::kVec; ++i)
      if (i < dim) v[i] = p[i];
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, Values<T> v, int64_t dim) {
  if (dim >= Chunk<T>::kVec) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Chunk<T>::kVec; ++i)
      if (i < dim) p[i] = v[i];
  }
}
// The same past the caches, of a whole chunk.
template <typename T>
__device__ __forceinline__ void store_past(T* p, Values<T> v) {
  typedef Values<T> Loose __attribute__((aligned(sizeof(T))));
  __builtin_nontemporal_store(v, reinterpret_cast<Loose*>(p));
}
template <typename T>
__device__ __forceinline__ Values<T> load_past(const T* p) {
  typedef Values<T> Loose __attribute__((aligned(sizeof(T))));
  return __builtin_nontemporal_load(reinterpret_cast<const Loose*>(p));
}
// Whether results go past the caches, and leave those to what is read: as they come, where rows fill whole lines; in
// the lines that lie inside a row, where no chunk crosses a line; or not at all.  Kernel times, other ids and results
// every call, so that nothing is left in the memory-side cache: 600 k rows of 256 B looked up in 627 MB 60 us with plain
// stores, 48 so (with plain stores and loads past the caches 58), and with a kernel behind that reads the result 115 and
// 113; 75 k rows 12.0 and 10.0.  94 k rows of 400 B sent to 4 experts each, and the gradient: 45 + 53 plain, 48 + 43 with
// the inner lines so, 67 + 36 with all.  Rows that are no multiple of 16 bytes, whose lines are written in two parts, go
// plainly: 30 k rows of 2002 B sent to experts 29 us either way (the same rows every call 20 and 22); a
// lookup alone is the other way round, 162 k rows of 1286 B 78 plain and 69 so.
enum class Past { kNo, kInside, kAll };

// p: the chunk `at` values into a row of dim values
template <typename T>
__device__ __forceinline__ void store_result(T* p, Values<T> v, int64_t at, int64_t dim, Past past) {
  bool whole = past == Past::kAll;
  if (past == Past::kInside) {
    constexpr int64_t kLine = 128;
    constexpr int64_t kSize = static_cast<int64_t>(sizeof(T));
    const int64_t in_line = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) % kLine);
    whole = in_line <= at * kSize && kLine - in_line <= (dim - at) * kSize;
  }
  if (whole) store_past(p, v);
  else store_chunk(p, v, dim);
}
// contiguous: the rows lie side by side and are written in order
template <typename T>
Past results_past(const T* rows, int64_t dim, bool contiguous) {
  constexpr int64_t kLine = 128;
  const int64_t bytes = dim * static_cast<int64_t>(sizeof(T));
  const uintptr_t base = reinterpret_cast<uintptr_t>(rows);
  if (dim <= 0 || bytes % 16 != 0 || base % 16 != 0) return Past::kNo;
  if (base % kLine == 0 && (contiguous || bytes % kLine == 0)) return Past::kAll;
  return bytes >= 2 * kLine ? Past::kInside : Past::kNo;
}
template <typename T>
__device__ __forceinline__ Wide<T> widen(Values<T> v) {
  return __builtin_convertvector(v, Wide<T>);
}
template <typename T>  // one rounding, to nearest, ties to even
__device__ __forceinline__ Values<T> narrow(Wide<T> v) {
  return __builtin_convertvector(v, Values<T>);
}

// x / d for x < 2^31 by a product (Granlund and Montgomery, "Division by invariant integers using
// multiplication", 1994), 1 <= d < 2^31.
struct Divider {
  uint32_t mul = 1, shift = 0, d = 1;
  Divider() = default;
  explicit Divider(uint32_t by) : d(by) {
    while ((uint64_t(1) << shift) < by) ++shift;
    mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - by)) / by + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    return (__umulhi(mul, x) + x) >> shift;
  }
};

// The chunks of all rows side by side, a workgroup a range of them: the row and the chunk in it of the
// j-th chunk (j below 2^31 - d) behind the range's first one.
struct RowRange {
  Divider by;
  int64_t row0;
  uint32_t c0;
  __device__ __forceinline__ RowRange(const Divider& chunks, int64_t first) : by(chunks) {
    if (first < (int64_t(1) << 31)) {
      const uint32_t q = chunks.quotient(static_cast<uint32_t>(first));
      row0 = q;
      c0 = static_cast<uint32_t>(first) - q * chunks.d;
    } else {
      row0 = first / chunks.d;
      c0 = static_cast<uint32_t>(first - row0 * chunks.d);
    }
  }
  __device__ __forceinline__ int64_t row(uint32_t j, uint32_t* chunk) const {
    const uint32_t x = c0 + j, q = by.quotient(x);
    *chunk = x - q * by.d;
    return row0 + q;
  }
};

// Which value type an entry point was given: calls f with a zero of the type.
template <typename F>
int with_value_type(int type, const char* what, F&& f) {
  switch (type) {
    case GS_F32:
      return f(float(0));
    case GS_F16:
      return f(_Float16(0));
    case GS_BF16:
      return f(__bf16(0));
    default:
      set_error_text("%s: value type %d is none of GS_F32, GS_F16, GS_BF16", what, type);
      return GS_ERR_INVALID_ARG;
  }
}
template <typename F>
int with_id_type(int id_bytes, F&& f) {
  return id_bytes == 4 ? f(int32_t(0)) : f(int64_t(0));
}
// Workgroups of `threads` that one launch takes: it counts its threads in 32 bits.
constexpr int64_t most_blocks(int threads) { return ((int64_t(1) << 32) - 1) / threads; }
inline int check_grid(const char* what, int64_t blocks, int threads) {
  if (blocks <= most_blocks(threads)) return GS_OK;
  set_error_text("%s: more rows and values than one launch takes", what);
  return GS_ERR_UNSUPPORTED;
}
inline int value_bytes(int type) { return type == GS_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & static_cast<uintptr_t>(bytes - 1)) == 0;
}

}  // namespace gs
