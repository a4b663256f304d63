// Products of tiles on the matrix cores of gfx950: the pieces that the products of experts' rows and
// the gradients of their matrices share.
//
// A workgroup makes a tile of C[m, n] = sum over k of A[m, k] * B[k, n].  It goes along k in steps of
// 64 bytes (32 values of 16 bits, 16 fp32 values), three to six of which have room in LDS: one is worked on, the next has
// arrived, or is about to, the others are on their way.  Either operand comes in one of two orders: along k, where the values of one row (or
// column) of C lie side by side, or across k, where the rows of one k do.  Sums are fp32 in the
// matrix cores' accumulators, in the order of k (what is left of the last step first), rounded once at the end.
#pragma once

#include "gs_rows.hpp"

namespace gs {
namespace products {

constexpr int kStepBytes = 64;
template <typename T>
constexpr int kStep = kStepBytes / static_cast<int>(sizeof(T));  // values of k a step

// A fragment is what a wave holds of 16 rows (or columns) of C and a step: lane l has row l % 16, 16 bytes of k from
// l / 16 * 16 bytes on.  The product of two: lane l gets C's row l % 16 of a, columns l / 16 * 4 .. + 3 of b.  (Products of
// 32 x 32 and half the depth read and write their sums twice as often, and are 5 % slower with as many cycles busy.)
typedef float Acc __attribute__((ext_vector_type(4)));

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
  static constexpr int kVec = Chunk<T>::kVec, kSize = static_cast<int>(sizeof(T));
  static constexpr int kSlots = WIDTH * (kStepBytes / 16);
  static constexpr int kBytes = kSlots * 16;
  static constexpr int kRowSlots = ACROSS ? WIDTH / kVec : kStepBytes / 16;  // slots of a row of the step
  static constexpr int kUnitSlots = kSize == 4 ? 4 : 2;  // of a unit of 16 values

  // What is read together lies in different banks (64 of 4 bytes).  Along k, row r holds 4 slots, and slot s keeps chunk
  // s ^ (r / 2 % 4): lanes 0 - 3, 12 - 15 and 20 - 27 are served together, then the others.  Across k, row k holds WIDTH
  // values in units of 16 that trade places: 32 lanes read a unit of rows k .. k + 3 and k + 8 .. k + 11 (16 bits), 64 lanes
  // one of rows k, k + 4, k + 8 and k + 12 (fp32).
  static_assert(WIDTH >= 64, "four units of a row trade places");
  static __device__ __forceinline__ int turn(int row) {
    if (!ACROSS) return (row >> 1) & 3;
    if (kSize == 4) return (row >> 2) & 3;
    return WIDTH >= 128 ? (row & 3) | (((row >> 3) & 1) << 2) : ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
  }
  static __device__ __forceinline__ int chunk_in(int row, int slot) {
    if (!ACROSS) return slot ^ turn(row);
    return ((slot / kUnitSlots) ^ turn(row)) * kUnitSlots + slot % kUnitSlots;
  }
};

// Reads a wave's fragments out of LDS.
template <typename T, bool ACROSS, int WIDTH>
struct Reader {
  using L = Layout<T, ACROSS, WIDTH>;
  template <typename V>
  using Lds = const __attribute__((address_space(3))) V;
  static constexpr int kRow = WIDTH * L::kSize;  // bytes, across k
  uint32_t base;  // the lane's part of the addresses

  // lds: where the operand's part of the ring begins; first: the wave's first row, a multiple of its number of rows, which
  // is a power of two
  __device__ __forceinline__ Reader(uint32_t lds, int first) {
    const int lane = threadIdx.x % kWave, row16 = lane % 16, quarter = lane / 16;
    if (!ACROSS) {
      base = lds + (first + row16) * kStepBytes + (quarter ^ L::turn(row16)) * 16;
    } else {
      const int k = L::kSize == 4 ? quarter * 4 : quarter * 8 + row16 / 4;
      base = lds + k * kRow + ((first / 16) ^ L::turn(k)) * (16 * L::kSize) + (L::kSize == 4 ? row16 * 4 : lane % 4 * 8);
    }
  }
  // the wave's j-th fragment of a step that lies `step` bytes into the ring
  __device__ __forceinline__ Values<T> fragment(int j, uint32_t step) const {
    if constexpr (!ACROSS) {
      return *reinterpret_cast<Lds<Values<T>>*>(base + step + j * 16 * kStepBytes);
    } else if constexpr (L::kSize == 4) {
      Values<T> v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<Lds<T>*>((base ^ (j * 64)) + step + i * kRow);
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
      for (int i = 0; i < 2; ++i)
        u.part[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<LdsFour*>((base ^ (j * 32)) + step + i * 4 * kRow));
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

// Writes some values.  Lanes whose 16 bytes begin inside a word do so by an instruction of their own, because one such lane
// slows all of its instruction's down: the gradient of 160 matrices of 1001 x 333, fp16, 187 rows each, 56 us and 61.  (Written as
// three stores, of which the compiler makes one, so that it does not see that both branches are the same.)
template <typename T, typename V>
__device__ __forceinline__ void store_all(T* p, V v) {
  if constexpr (sizeof(T) == 2 && sizeof(V) == 16) {
    struct Words {
      uint32_t w[3];
    };
    typedef Words __attribute__((aligned(4), may_alias)) Aliasing;
    if (reinterpret_cast<uintptr_t>(p) % 4 != 0) {
      typedef T Six __attribute__((ext_vector_type(6)));
      const Six six = {v[1], v[2], v[3], v[4], v[5], v[6]};
      Words words;
      __builtin_memcpy(&words, &six, sizeof(words));
      p[0] = v[0];
      *reinterpret_cast<Aliasing*>(p + 1) = words;
      p[7] = v[7];
      return;
    }
  }
  __builtin_memcpy(p, &v, sizeof(V));
}

// Writes the first `there` of some values.
template <typename T, typename V>
__device__ __forceinline__ void store_part(T* p, V v, int64_t there) {
  constexpr int kMany = static_cast<int>(sizeof(V) / sizeof(T));
  if (there >= kMany) {
    store_all(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < kMany - 1; ++i)
      if (i < there) p[i] = v[i];
  }
}

// Where a value of the last chunk of a row (or column) of `there` values has its place, if that chunk was fetched from as far
// in front of it as it lacks; others stay.
template <int VEC>
__device__ __forceinline__ int64_t moved(int64_t n, int64_t there) {
  const int64_t first = n / VEC * VEC;
  return first + VEC > there ? n + there - VEC - first : n;
}

// Rounds a lane's sums, columns j * 16 + (l / 16) * 4 .. of a row, once, to nearest, ties to even, and writes the first
// `there` columns of the row.  MOVED: the columns' chunks have that many values, and the last one was moved.
template <int FRAGMENTS, int MOVED = 0, typename O>
__device__ __forceinline__ void write_row(const Acc* acc, O* row, int64_t there) {
  typedef O Four __attribute__((ext_vector_type(4)));
  const int quarter = threadIdx.x % kWave / 16;
  auto put = [&](int n, auto v) {
    if constexpr (MOVED != 0) {
      if (n / MOVED * MOVED < there) store_all(row + moved<MOVED>(n, there), v);
    } else {
      store_part(row + n, v, there - n);
    }
  };
  if constexpr (sizeof(O) == 2 && FRAGMENTS % 2 == 0) {
    // two fragments' neighbouring quarters trade places, so that a lane has eight columns side by side
#pragma unroll
    for (int j = 0; j < FRAGMENTS; j += 2) {
      typedef uint32_t Two __attribute__((ext_vector_type(2)));
      const Two a = __builtin_bit_cast(Two, __builtin_convertvector(acc[j], Four));
      const Two b = __builtin_bit_cast(Two, __builtin_convertvector(acc[j + 1], Four));
      const Two x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
      const Two y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
      union {
        uint32_t word[4];
        Values<O> v;
      } u = {{x[0], y[0], x[1], y[1]}};
      put((j + quarter % 2) * 16 + quarter / 2 * 8, u.v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < FRAGMENTS; ++j) put(j * 16 + quarter * 4, __builtin_convertvector(acc[j], Four));
  }
}

// An operand of a tile: `rows` rows (along k: of C; across k: of k), `stride` values apart, of `width` values.
template <typename T>
struct Operand {
  const T* base;
  int64_t stride, rows, width;
};

// The values of a chunk from the s-th on, zeros behind them.
template <typename T>
__device__ __forceinline__ Values<T> shifted(Values<T> v, int s) {
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  Words w = __builtin_bit_cast(Words, v);
  const int words = sizeof(T) == 4 ? s : s / 2;
  if (words & 2) w = Words{w[2], w[3], 0, 0};
  if (words & 1) w = Words{w[1], w[2], w[3], 0};
  if (sizeof(T) == 2 && (s & 1)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (w[i] >> 16) | (i < 3 ? w[i < 3 ? i + 1 : 3] << 16 : 0);
  }
  return __builtin_bit_cast(Values<T>, w);
}

// How an operand comes: straight into LDS, or, where there is no whole chunk or a step's chunks lie more than 2^31 bytes
// apart, value by value through registers.
enum class Way { kDirect, kValues };

// Fetches an operand value by value, kHeld steps ahead of their stores to LDS.
constexpr int kHeld = 4;
template <typename T, bool ACROSS, int WIDTH, int THREADS>
struct Staged {
  using L = Layout<T, ACROSS, WIDTH>;
  static constexpr int kEach = L::kSlots / THREADS;
  static_assert(L::kSlots % THREADS == 0, "every lane has as many chunks");
  Operand<T> x;
  int64_t k0 = 0;  // of the next step
  Values<T> held[kHeld][kEach];

  static __device__ __forceinline__ int row(int i) { return (i * THREADS + static_cast<int>(threadIdx.x)) / L::kRowSlots; }
  static __device__ __forceinline__ int chunk(int i) {
    return L::chunk_in(row(i), (i * THREADS + static_cast<int>(threadIdx.x)) % L::kRowSlots) * L::kVec;
  }
  __device__ __forceinline__ explicit Staged(const Operand<T>& operand) : x(operand) {}
  // The first step: the last part of the depth, `rest` of a step, so that all others are whole.
  __device__ __forceinline__ void load_rest(int64_t whole_steps, int64_t rest) {
    k0 = whole_steps * kStep<T>;
#pragma unroll
    for (int i = 0; i < kEach; ++i) held[0][i] = part(i, rest);
    k0 = 0;
  }
  __device__ __forceinline__ Values<T> part(int i, int64_t left) const {
    const int64_t r = ACROSS ? k0 + row(i) : row(i), c = ACROSS ? chunk(i) : k0 + chunk(i);
    const bool in = ACROSS ? row(i) < left : r < x.rows;
    return load_part(x.base + r * x.stride + c, in ? (ACROSS ? x.width - c : left - chunk(i)) : 0);
  }
  // The next step; more: it is not the last one (which is read again, and not used, behind the end).  whole: there is one.
  template <int SLOT>
  __device__ __forceinline__ void load(bool whole, bool more) {
    if (!whole) return;
#pragma unroll
    for (int i = 0; i < kEach; ++i) held[SLOT][i] = part(i, kStep<T>);
    if (more) k0 += kStep<T>;
  }
  template <int SLOT>
  __device__ __forceinline__ void store(char* lds) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) *reinterpret_cast<Values<T>*>(lds + (i * THREADS + threadIdx.x) * 16) = held[SLOT][i];
  }
};

// Fetches an operand step by step straight into LDS, 16 bytes a lane.  Chunks that do not exist are fetched from beyond
// the buffer's end, and come as zeros.  One of which a part exists is fetched from as far in front of it as it lacks: along the
// depth it is shifted in LDS (it is in the first step), across it its values change places in C, which is known when C is
// written.  Rows hold a chunk at least, and a step of a tile lies within 2^31 bytes; they need no alignment, but chunks that are not
// aligned come at half the rate, or less, from the caches: 23 TB/s, 11.5 (to 4 bytes) and 9.3 (to 2).
template <typename T, bool ACROSS, int WIDTH, int THREADS>
struct Direct {
  using L = Layout<T, ACROSS, WIDTH>;
  typedef int Buffer __attribute__((ext_vector_type(4)));
  static constexpr int kEach = L::kSlots / THREADS, kRowsApart = THREADS / L::kRowSlots;
  static_assert(L::kSlots % THREADS == 0 && THREADS % L::kRowSlots == 0, "every lane has as many chunks");
  static constexpr int kNowhere = static_cast<int>(0x80000000u), kSize = static_cast<int>(sizeof(T));
  uint64_t base;  // aligned, 16 to 31 bytes in front of the operand
  int64_t step;   // bytes between steps
  int at[kEach];

  __device__ __forceinline__ explicit Direct(const Operand<T>& x) {
    const uint64_t from = reinterpret_cast<uint64_t>(x.base) - 16;
    base = from & ~uint64_t(15);
    step = ACROSS ? kStep<T> * x.stride * kSize : kStepBytes;
    const int64_t across = ACROSS ? x.width : x.rows;
    const int front = static_cast<int>(from & 15) + 16;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int lack = ACROSS && across < chunk(i) + L::kVec ? chunk(i) + L::kVec - static_cast<int>(across) : 0;
      at[i] = static_cast<int>(row(i) * x.stride + chunk(i) - lack) * kSize + front;
      if ((ACROSS ? chunk(i) : row(i)) >= across) at[i] = kNowhere;
    }
  }
  static __device__ __forceinline__ int row(int i) { return static_cast<int>(threadIdx.x) / L::kRowSlots + i * kRowsApart; }
  static __device__ __forceinline__ int chunk(int i) { return L::chunk_in(row(i), threadIdx.x % L::kRowSlots) * L::kVec; }
  // Written as instructions because the compiler, which cannot tell the ring's steps apart, would wait for all of them before
  // each read of LDS; who reads waits by arrived().  (m0, where the place in LDS goes, is set by the compiler, which so knows what it
  // holds; the instruction behind has to wait for a cycle.)
  static __device__ __forceinline__ void put(uint64_t base, int bytes, int from, uint32_t lds, int offset) {
    const Buffer buffer = {static_cast<int>(base), static_cast<int>(base >> 32), bytes, 0x00020000};
    register uint32_t place asm("m0") = lds + offset;
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(place), "v"(from), "s"(buffer) : "memory");
  }
  // Puts a part of the next step on its way to lds (an offset); bytes: all there are, or none, for zeros.
  __device__ __forceinline__ void part(int i, uint32_t lds, int bytes) const {
    put(base, bytes, at[i], lds, i * THREADS * 16);
  }
  __device__ __forceinline__ void advance() { base += step; }
  // The first step: the last part of the depth, `rest` of a step, so that all others are whole.
  __device__ __forceinline__ void first(int64_t whole_steps, int rest, uint32_t lds) const {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int left = rest - (ACROSS ? row(i) : chunk(i));
      const int less = !ACROSS && left < L::kVec ? (L::kVec - left) * kSize : 0;
      put(base + whole_steps * step, kAll, left > 0 && at[i] >= 0 ? at[i] - less : kNowhere, lds, i * THREADS * 16);
    }
  }
  // When the lane's part of that step is there, what came from in front of its place is shifted.
  __device__ __forceinline__ void settle(int rest, char* lds) const {
#pragma unroll
    for (int i = 0; i < kEach && !ACROSS; ++i) {
      const int left = rest - chunk(i);
      auto* const slot = reinterpret_cast<Values<T>*>(lds + (i * THREADS + threadIdx.x) * 16);
      if (left > 0 && left < L::kVec) *slot = shifted<T>(*slot, L::kVec - left);
    }
  }
  static constexpr int kAll = 0x7fffffff;
};

// How rows of `width` values, `stride` apart, come, up to `rows` of them a step.
template <typename T>
Way way_of(int64_t stride, int64_t width, int64_t rows) {
  const bool far = stride >= (int64_t(1) << 31) / (rows * static_cast<int64_t>(sizeof(T)));
  return width < Chunk<T>::kVec || far ? Way::kValues : Way::kDirect;
}
// Whether their chunks are aligned; apart: other matrices' distance.
template <typename T>
bool aligned_rows(const T* base, int64_t stride, int64_t apart) {
  constexpr int64_t kVec = Chunk<T>::kVec;
  return aligned_to(base, 16) && stride % kVec == 0 && apart % kVec == 0;
}
inline Way slower(Way a, Way b) { return a > b ? a : b; }

// All but the last LEFT of a wave's fetches have arrived, and all waves of the workgroup have come here.
template <int LEFT>
__device__ __forceinline__ void arrived() {
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"(LEFT) : "memory");
}

// A tile of BM x BN by WM x WN waves, RING steps in LDS, three at least.
template <typename T, bool A_ACROSS, bool B_ACROSS, int BM, int BN, int WM, int WN, int RING, Way WAY>
struct Tile {
  using LA = Layout<T, A_ACROSS, BM>;
  using LB = Layout<T, B_ACROSS, BN>;
  using RA = Reader<T, A_ACROSS, BM>;
  using RB = Reader<T, B_ACROSS, BN>;
  static constexpr int kThreads = WM * WN * kWave;
  static constexpr int kMI = BM / WM / 16, kNI = BN / WN / 16, kFirst = kMI / 2;
  static_assert(kFirst >= 1, "either half of a step has rows");
  static constexpr int kStage = LA::kBytes + LB::kBytes, kBytes = RING * kStage;  // of LDS
  static constexpr bool kDirect = WAY == Way::kDirect;
  using FA = std::conditional_t<kDirect, Direct<T, A_ACROSS, BM, kThreads>, Staged<T, A_ACROSS, BM, kThreads>>;
  using FB = std::conditional_t<kDirect, Direct<T, B_ACROSS, BN, kThreads>, Staged<T, B_ACROSS, BN, kThreads>>;
  Acc acc[kMI][kNI];

  static __device__ __forceinline__ int row0() { return static_cast<int>(threadIdx.x) / kWave / WN * (BM / WM); }
  static __device__ __forceinline__ int col0() { return static_cast<int>(threadIdx.x) / kWave % WN * (BN / WN); }
  static __device__ __forceinline__ uint32_t lds_offset(char* lds) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)lds));
  }

  // Step s is multiplied in two halves of the wave's rows.  In front of the second one, step s + 1 has arrived everywhere,
  // and nobody reads step s - 1 any more, whose place step s + RING - 1 takes: its fetches, and the reads of the fragments
  // that step s + 1 begins with, stand between the products of the second half, in an order that is kept as it is written.
  struct Fragments {
    Values<T> a[kMI], b[2][kNI];
  };
  static constexpr int kFirstProducts = kFirst * kNI, kSecondProducts = (kMI - kFirst) * kNI;
  static constexpr int kLater = kMI - kFirst, kAhead = kFirst + kNI, kFetches = FA::kEach + FB::kEach;
  // The items of `many` that stand in front of product q of `products`, spread evenly; what is read ahead, in the first
  // three quarters, so that it has come when the next step begins; what is fetched, a little behind what is read, since a
  // wave finds time for three instructions behind a product, no more.
  static constexpr int due(int q, int many, int products) { return (q * many + products - 1) / products; }
  static constexpr int due_ahead(int q) {
    const int r = (q * kAhead * 4 + 3 * kSecondProducts - 1) / (3 * kSecondProducts);
    return r < kAhead ? r : kAhead;
  }
  static constexpr int due_fetch(int q) {
    if (q >= kSecondProducts) return kFetches;
    const int r = (4 * q * kFetches - kSecondProducts + 4 * kSecondProducts - 1) / (4 * kSecondProducts);
    return r < 0 ? 0 : r;
  }

  struct Steps {
    RA ra;
    RB rb;
    FA fa;
    FB fb;
    char* lds;
    int64_t ahead;  // steps that are not on their way yet
    bool whole;     // there are whole ones

    __device__ __forceinline__ void fetch(int i, uint32_t to, int bytes) {
      if (i < FA::kEach) fa.part(i, to, bytes);
      else fb.part(i - FA::kEach, to + LA::kBytes, bytes);
    }
    template <int SLOT>
    __device__ __forceinline__ void load() {  // (through registers)
      fa.template load<SLOT>(whole, ahead > 1);
      fb.template load<SLOT>(whole, ahead > 1);
      --ahead;
    }
    template <int SLOT>
    __device__ __forceinline__ void store(char* to) {
      fa.template store<SLOT>(to);
      fb.template store<SLOT>(to + LA::kBytes);
    }
    __device__ __forceinline__ void advance() {
      fa.advance();
      fb.advance();
      --ahead;
    }
  };

  // a step in ring place `now`, its fragments of b in f.b[TURN % 2]
  template <int TURN>
  __device__ __forceinline__ void step(Fragments& f, Steps& s, uint32_t now) {
    const uint32_t next = now + kStage == kBytes ? 0 : now + kStage;
#pragma unroll
    for (int q = 0; q < kFirstProducts; ++q) {
#pragma unroll
      for (int r = due(q, kLater, kFirstProducts); r < due(q + 1, kLater, kFirstProducts); ++r)
        f.a[kFirst + r] = s.ra.fragment(kFirst + r, now);
      acc[q / kNI][q % kNI] = multiply(f.b[TURN % 2][q % kNI], f.a[q / kNI], acc[q / kNI][q % kNI]);
      __builtin_amdgcn_sched_barrier(0);
    }
    uint32_t to = 0;
    int bytes = 0;
    if constexpr (kDirect) {
      arrived<(RING - 3) * kFetches>();
      to = lds_offset(s.lds) + (now == 0 ? kBytes - kStage : now - kStage) +
           __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * (kWave * 16);
      bytes = s.ahead > 0 ? FA::kAll : 0;
    } else {
      __syncthreads();
      s.template store<(TURN + 2) % kHeld>(s.lds + (now + 2 * kStage) % kBytes);
      s.template load<(TURN + 2) % kHeld>();
    }
#pragma unroll
    for (int q = 0; q < kSecondProducts; ++q) {
      const int i = kFirst + q / kNI, j = q % kNI;
#pragma unroll
      for (int r = due_ahead(q); r < due_ahead(q + 1); ++r) {
        if (r < kFirst) f.a[r] = s.ra.fragment(r, next);
        else f.b[(TURN + 1) % 2][r - kFirst] = s.rb.fragment(r - kFirst, next);
      }
      if constexpr (kDirect) {
#pragma unroll
        for (int r = due_fetch(q); r < due_fetch(q + 1); ++r) s.fetch(r, to, bytes);
      }
      acc[i][j] = multiply(f.b[TURN % 2][j], f.a[i], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kDirect) s.advance();
  }

  // lds: kBytes, aligned to 1024 (parts of addresses are exchanged by exclusive or)
  __device__ __forceinline__ void run(const Operand<T>& a, const Operand<T>& b, int64_t depth, char* lds) {
#pragma unroll
    for (int i = 0; i < kMI; ++i)
#pragma unroll
      for (int j = 0; j < kNI; ++j) acc[i][j] = Acc{};
    int64_t steps = (depth + kStep<T> - 1) / kStep<T>;
    if (steps <= 0) return;
    Steps s{RA(lds_offset(lds), row0()), RB(lds_offset(lds) + LA::kBytes, col0()), FA(a), FB(b), lds, steps, depth >= kStep<T>};
    if constexpr (kDirect) {
      const uint32_t to = lds_offset(lds) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * (kWave * 16);
      const int64_t whole = depth / kStep<T>;
      const int rest = static_cast<int>(depth % kStep<T>);
      if (rest > 0) {
        s.fa.first(whole, rest, to);
        s.fb.first(whole, rest, to + LA::kBytes);
        --s.ahead;
      }
#pragma unroll
      for (int i = 0; i < RING - 1; ++i) {
        if (i == 0 && rest > 0) continue;
#pragma unroll
        for (int r = 0; r < kFetches; ++r) s.fetch(r, to + i * kStage, s.ahead > 0 ? FA::kAll : 0);
        s.advance();
      }
      if (rest % LA::kVec != 0 && !(A_ACROSS && B_ACROSS)) {
        asm volatile("s_waitcnt vmcnt(%0)" : : "n"((RING - 2) * kFetches) : "memory");
        s.fa.settle(rest, lds);
        s.fb.settle(rest, lds + LA::kBytes);
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      }
      arrived<(RING - 2) * kFetches>();
    } else {
      const int64_t whole = depth / kStep<T>, rest = depth % kStep<T>;
      if (rest > 0) {
        s.fa.load_rest(whole, rest);
        s.fb.load_rest(whole, rest);
        --s.ahead;
      } else {
        s.template load<0>();
      }
      s.template load<1>();
      s.template load<2>();
      s.template load<3>();
      s.template store<0>(lds);
      s.template load<0>();
      s.template store<1>(lds + kStage);
      s.template load<1>();
      __syncthreads();
    }
    Fragments f;
#pragma unroll
    for (int j = 0; j < kNI; ++j) f.b[0][j] = s.rb.fragment(j, 0);
#pragma unroll
    for (int i = 0; i < kFirst; ++i) f.a[i] = s.ra.fragment(i, 0);
    // (two steps a turn, or four, so that what is read ahead stays in its registers; straight into LDS, one behind the last
    // is zeros)
    uint32_t now = 0;
    auto place = [&] {
      const uint32_t here = now;
      now = now + kStage == kBytes ? 0 : now + kStage;
      return here;
    };
    if constexpr (kDirect) {
      for (; steps > 0; steps -= 2) {
        step<0>(f, s, place());
        step<1>(f, s, place());
      }
    } else {
      while (true) {
        step<0>(f, s, place());
        if (--steps == 0) break;
        step<1>(f, s, place());
        if (--steps == 0) break;
        step<2>(f, s, place());
        if (--steps == 0) break;
        step<3>(f, s, place());
        if (--steps == 0) break;
      }
    }
    if constexpr (kDirect) arrived<0>();  // (nothing is on its way into LDS that the next workgroup has by then)
  }

  // Rounds the sums, once, to nearest, ties to even, and writes rows 0 .. rows - 1 and columns 0 .. cols - 1 of the tile to out.
  // (Some rows and columns are written twice where chunks across the depth were moved, the same values.)
  template <typename O>
  __device__ __forceinline__ void write(O* out, int64_t stride, int64_t rows, int64_t cols) const {
    constexpr int kVec = LA::kVec;
    constexpr bool kRowsMoved = kDirect && A_ACROSS, kColsMoved = kDirect && B_ACROSS;
#pragma unroll
    for (int i = 0; i < kMI; ++i) {
      const int m = row0() + i * 16 + static_cast<int>(threadIdx.x) % 16;
      const bool in = (kRowsMoved ? m / kVec * kVec : m) < rows;
      write_row<kNI, kColsMoved ? kVec : 0>(acc[i], out + (kRowsMoved ? moved<kVec>(m, rows) : m) * stride + col0(),
                                            in ? cols - col0() : 0);
    }
  }
};

// Every workgroup looks through all experts' offsets for its own rows, up to half a megabyte.
constexpr int64_t kMostExperts = 1 << 16;

// Where an expert's rows begin and end, inside [0, n] whatever the offsets hold.  Expert `experts` has the rows behind the last.
struct Group {
  int64_t begin, end;
  __device__ __forceinline__ int64_t rows() const { return end > begin ? end - begin : 0; }
};
__device__ __forceinline__ int64_t uniform(int64_t v) {  // (the same in all lanes)
  const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
}
__device__ __forceinline__ int64_t inside(int64_t v, int64_t n) { return v < 0 ? 0 : (v < n ? v : n); }
__device__ __forceinline__ Group group_of(const int64_t* __restrict__ offsets, int64_t experts, int64_t n, int64_t e) {
  return {inside(offsets[e], n), e < experts ? inside(offsets[e + 1], n) : n};
}

// Launches a kernel of one argument for so many workgroups, in turns where one launch does not take them.
template <typename Args>
int launch_blocks(void (*kernel)(Args), Args args, int64_t blocks, int threads, const char* what, hipStream_t st) {
  const int64_t most = most_blocks(threads) / kXcds * kXcds;  // (every turn begins at the first die)
  for (args.first_block = 0; args.first_block < blocks; args.first_block += most) {
    const int64_t here = blocks - args.first_block < most ? blocks - args.first_block : most;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(here)), dim3(threads), 0, st, args);
    GS_RETURN_IF_ERROR(check_launch(what));
  }
  return GS_OK;
}

}  // namespace products
}  // namespace gs
