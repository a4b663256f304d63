// Products of tiles on the matrix cores of gfx950: the pieces that the products of experts' rows and
// the gradients of their matrices share.
//
// A workgroup makes a tile of C[m, n] = sum over k of A[m, k] * B[k, n].  It goes along k in steps of
// 128 bytes (64 values of 16 bits, 32 fp32 values), which lie in LDS, two steps at a time: one is worked on
// while the next is fetched.  Either operand comes in one of two orders: along k, where the values of one row (or
// column) of C lie side by side, or across k, where the rows of one k do.  Sums are fp32 in the
// matrix cores' accumulators, in the order of k, rounded once at the end.
#pragma once

#include "gs_rows.hpp"

namespace gs {
namespace products {

constexpr int kStepBytes = 128;
template <typename T>
constexpr int kStep = kStepBytes / static_cast<int>(sizeof(T));  // values of k a step

typedef float Acc __attribute__((ext_vector_type(4)));

// What a lane holds for 16 rows (or columns) of C and 64 bytes of k: row lane % 16, k from lane / 16 * 16 bytes on.  The
// product of two of those: lane l gets C's row (l % 16) of a, columns (l / 16) * 4 .. + 3 of b.
__device__ __forceinline__ Acc multiply(Values<__bf16> b, Values<__bf16> a, Acc c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
}
__device__ __forceinline__ Acc multiply(Values<_Float16> b, Values<_Float16> a, Acc c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(b, a, c, 0, 0, 0);
}
// (fp32: four instructions, each with one value of every lane's four, the same for a and b)
__device__ __forceinline__ Acc multiply(Values<float> b, Values<float> a, Acc c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(b[i], a[i], c, 0, 0, 0);
  return c;
}

// How an operand's WIDTH rows (or columns) of a step lie in LDS, in slots of 16 bytes.
template <typename T, bool ACROSS, int WIDTH>
struct Layout {
  static constexpr int kVec = Chunk<T>::kVec;
  static constexpr int kSlots = WIDTH * (kStepBytes / 16);
  static constexpr int kBytes = kSlots * 16;
  static constexpr int kRowSlots = ACROSS ? WIDTH / kVec : kStepBytes / 16;  // slots of a row of the step

  // Along k, row r holds 8 slots; a fragment's 16 rows are 128 bytes apart, so slot s keeps chunk s ^ (r % 8): the rows
  // of a fragment then lie in different banks.  Across k, row k holds WIDTH values; fragments take 32 bytes (16 bits) or 64
  // (fp32) of each of several rows, and such units trade places for the same reason.
  static __device__ __forceinline__ int chunk_in(int row, int slot) {
    if (!ACROSS) return slot ^ (row & 7);
    if (sizeof(T) == 4) return (((slot >> 2) ^ ((row >> 2) & (WIDTH >= 64 ? 3 : 0))) << 2) | (slot & 3);
    return (((slot >> 1) ^ turn(row)) << 1) | (slot & 1);
  }
  static __device__ __forceinline__ int turn(int row) {
    if (WIDTH >= 128) return (row & 3) | (((row >> 3) & 1) << 2);
    if (WIDTH == 64) return ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
    return 0;
  }

  // the fragment of rows at .. at + 15 (a multiple of 16) and the step's half `half`
  static __device__ __forceinline__ Values<T> fragment(const char* lds, int at, int half) {
    const int lane = threadIdx.x % kWave, row16 = lane % 16, quarter = lane / 16;
    if constexpr (!ACROSS) {
      const int row = at + row16;
      return *reinterpret_cast<const Values<T>*>(lds + row * kStepBytes + chunk_in(row, half * 4 + quarter) * 16);
    } else if constexpr (sizeof(T) == 4) {
      Values<T> v;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = half * 16 + quarter * 4 + i;
        const int unit = (at / 16) ^ ((k >> 2) & (WIDTH >= 64 ? 3 : 0));
        v[i] = *reinterpret_cast<const T*>(lds + (k * WIDTH + unit * 16 + row16) * 4);
      }
      return v;
    } else {
      // (a transposing read: 16 lanes take 4 rows of 16 values and get a column of 4 each)
      typedef short Four __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) Four LdsFour;
      union {
        Four part[2];
        Values<T> v;
      } u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = half * 32 + quarter * 8 + i * 4 + row16 / 4;
        const int unit = (at / 16) ^ turn(k);
        const char* p = lds + k * (WIDTH * 2) + unit * 32 + (lane % 4) * 8;
        u.part[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour*)(p));
      }
      return u.v;
    }
  }
};

// A chunk of which the first `there` values exist; zeros for the others.
template <typename T>
__device__ __forceinline__ Values<T> load_part(const T* p, int64_t there) {
  Values<T> v = {};
  if (there >= Chunk<T>::kVec) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Chunk<T>::kVec; ++i)
      if (i < there) v[i] = p[i];
  }
  return v;
}

// An operand of a tile: `rows` rows (along k: of C; across k: of k), `stride` values apart, of `width` values.
template <typename T>
struct Operand {
  const T* base;
  int64_t stride, rows, width;
};

// Fetches an operand step by step through registers.
template <typename T, bool ACROSS, int WIDTH, int THREADS>
struct Fetch {
  using L = Layout<T, ACROSS, WIDTH>;
  static constexpr int kEach = (L::kSlots + THREADS - 1) / THREADS;
  Values<T> held[kEach];

  __device__ __forceinline__ void load(const Operand<T>& x, int64_t k0) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int q = i * THREADS + threadIdx.x;
      const int r = q / L::kRowSlots, c = L::chunk_in(r, q % L::kRowSlots) * L::kVec;
      const int64_t row = ACROSS ? k0 + r : r, col = ACROSS ? c : k0 + c;
      const bool in = q < L::kSlots && row < x.rows;
      held[i] = load_part(x.base + row * x.stride + col, in ? x.width - col : 0);
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int q = i * THREADS + threadIdx.x;
      if (L::kSlots % THREADS == 0 || q < L::kSlots) *reinterpret_cast<Values<T>*>(lds + q * 16) = held[i];
    }
  }
};

// A tile of BM x BN by WM x WN waves.
template <typename T, bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN>
struct Tile {
  using LA = Layout<T, A_ACROSS, BM>;
  using LB = Layout<T, B_ACROSS, BN>;
  static constexpr int kThreads = WM * WN * kWave;
  static constexpr int kMI = BM / WM / 16, kNI = BN / WN / 16;
  static constexpr int kBytes = 2 * (LA::kBytes + LB::kBytes);  // of LDS
  Acc acc[kMI][kNI];

  static __device__ __forceinline__ int row0() { return static_cast<int>(threadIdx.x) / kWave / WN * (BM / WM); }
  static __device__ __forceinline__ int col0() { return static_cast<int>(threadIdx.x) / kWave % WN * (BN / WN); }

  __device__ __forceinline__ void work(const char* a_lds, const char* b_lds) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Values<T> a[kMI], b[kNI];
#pragma unroll
      for (int i = 0; i < kMI; ++i) a[i] = LA::fragment(a_lds, row0() + i * 16, half);
#pragma unroll
      for (int j = 0; j < kNI; ++j) b[j] = LB::fragment(b_lds, col0() + j * 16, half);
#pragma unroll
      for (int i = 0; i < kMI; ++i)
#pragma unroll
        for (int j = 0; j < kNI; ++j) acc[i][j] = multiply(b[j], a[i], acc[i][j]);
    }
  }

  // lds: kBytes
  __device__ __forceinline__ void run(const Operand<T>& a, const Operand<T>& b, int64_t depth, char* lds) {
#pragma unroll
    for (int i = 0; i < kMI; ++i)
#pragma unroll
      for (int j = 0; j < kNI; ++j) acc[i][j] = Acc{};
    if (depth <= 0) return;
    Fetch<T, A_ACROSS, BM, kThreads> fa;
    Fetch<T, B_ACROSS, BN, kThreads> fb;
    char* const a_lds[2] = {lds, lds + LA::kBytes};
    char* const b_lds[2] = {lds + 2 * LA::kBytes, lds + 2 * LA::kBytes + LB::kBytes};
    fa.load(a, 0);
    fb.load(b, 0);
    fa.store(a_lds[0]);
    fb.store(b_lds[0]);
    __syncthreads();
    int now = 0;
    for (int64_t k = kStep<T>; ; k += kStep<T>) {
      const bool more = k < depth;
      if (more) {
        fa.load(a, k);
        fb.load(b, k);
      }
      work(a_lds[now], b_lds[now]);
      if (!more) break;
      now ^= 1;  // (whose last readers are behind the barrier of the step before)
      fa.store(a_lds[now]);
      fb.store(b_lds[now]);
      __syncthreads();
    }
  }

  // f(m, n, four values of row m from column n on)
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int i = 0; i < kMI; ++i)
#pragma unroll
      for (int j = 0; j < kNI; ++j) f(row0() + i * 16 + lane % 16, col0() + j * 16 + lane / 16 * 4, acc[i][j]);
  }
};

// `there` of four values, rounded once, to nearest, ties to even
template <typename T>
__device__ __forceinline__ void store_four(T* p, Acc v, int64_t there) {
  typedef T Four __attribute__((ext_vector_type(4)));
  const Four r = __builtin_convertvector(v, Four);
  if (there >= 4) {
    __builtin_memcpy(p, &r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < there) p[i] = r[i];
  }
}

// Where an expert's rows begin and end, inside [0, n] whatever the offsets hold.  Expert `experts` has the rows behind the last.
struct Group {
  int64_t begin, end;
  __device__ __forceinline__ int64_t rows() const { return end > begin ? end - begin : 0; }
};
__device__ __forceinline__ int64_t inside(int64_t v, int64_t n) { return v < 0 ? 0 : (v < n ? v : n); }
__device__ __forceinline__ Group group_of(const int64_t* __restrict__ offsets, int64_t experts, int64_t n, int64_t e) {
  return {inside(offsets[e], n), e < experts ? inside(offsets[e + 1], n) : n};
}

}  // namespace products
}  // namespace gs
