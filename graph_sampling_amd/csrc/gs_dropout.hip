// Dropout by counter-based draws, on gfx950.
//
//   out[i] = residual[i] + (draw(seed, 6, 0, i) >= floor(p * 2^32) ? x[i] / (1 - p) : 0)
//
// The draw is the samplers' own (Philox4x32-10, four positions a block), so the mask is a function of seed and position
// and is never stored: the gradient draws it again.  Memory bounds it; with a chunk a lane there are waves enough to hide the
// draws, ten rounds of two products each: 600 000 x 64 fp32, 52 us, 5.9 TB/s; 16384 x 2048 bf16 with a residual, 38 us, 5.3.
// No counterpart in the reference.
#include "gs_rows.hpp"

namespace gs {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kTagDropout = 6u;

// A chunk of values a lane.  LATER: a launch behind the first, whose values begin at block0 of the draws (the first one does without
// the sum: 16384 x 2048 bf16 21.1 us with it, 20.6 without).
template <typename T, bool LATER>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, int64_t n, uint32_t least, bool none, float scale,
               uint64_t seed, const int64_t* __restrict__ seed_at, T* __restrict__ out, uint64_t block0) {
  constexpr int kVec = Chunk<T>::kVec;
  if (seed_at) seed = static_cast<uint64_t>(*seed_at);
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kVec;
  if (first >= n) return;
  const int64_t there = n - first < kVec ? n - first : kVec;
  const Wide<T> v = widen<T>(load_chunk(x + first, there));
  Wide<T> r = {};
  if (residual) r = widen<T>(load_chunk(residual + first, there));
#pragma unroll
  for (int i = 0; i < kVec; i += 4) {
    const U4 draws = draw_block(seed, kTagDropout, 0, (LATER ? block0 : 0) + (static_cast<uint64_t>(first + i) >> 2));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (draws.v[j] >= least && !none) r[i + j] = __fmaf_rn(v[i + j], scale, r[i + j]);
  }
  store_chunk(out + first, narrow<T>(r), there);
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" int gs_dropout(const void* x, const void* residual, int64_t n, int type, double p, uint64_t seed,
                          const int64_t* seed_at, void* out, void* stream) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16,
             "gs_dropout: value type %d is none of GS_F32, GS_F16, GS_BF16", type);
  GS_REQUIRE(n >= 0, "gs_dropout: negative size");
  GS_REQUIRE(p >= 0.0 && p <= 1.0, "gs_dropout: p = %g is no probability", p);
  if (n == 0) return GS_OK;
  GS_REQUIRE(x && out, "gs_dropout: null array");
  GS_REQUIRE(aligned_to(x, value_bytes(type)) && aligned_to(residual, value_bytes(type)) && aligned_to(out, value_bytes(type)) &&
                 aligned_to(seed_at, 8),
             "gs_dropout: values not aligned to their type");
  const bool none = p == 1.0;
  const uint32_t least = none ? 0 : static_cast<uint32_t>(p * 4294967296.0);
  const float scale = none ? 0.0f : static_cast<float>(1.0 / (1.0 - p));
  return with_value_type(type, "gs_dropout", [&](auto zero) {
    using T = decltype(zero);
    constexpr int64_t kBlock = kThreads * Chunk<T>::kVec, kMost = most_blocks(kThreads) * kBlock;  // values a launch
    for (int64_t base = 0; base < n; base += kMost) {
      const int64_t here = n - base < kMost ? n - base : kMost;
      const dim3 grid(static_cast<unsigned>((here + kBlock - 1) / kBlock));
      hipLaunchKernelGGL((base == 0 ? dropout_kernel<T, false> : dropout_kernel<T, true>), grid, dim3(kThreads), 0,
                         static_cast<hipStream_t>(stream), static_cast<const T*>(x) + base,
                         residual ? static_cast<const T*>(residual) + base : nullptr, here, least, none, scale, seed, seed_at,
                         static_cast<T*>(out) + base, static_cast<uint64_t>(base) / 4);
      GS_RETURN_IF_ERROR(check_launch("dropout"));
    }
    return static_cast<int>(GS_OK);
  });
}
