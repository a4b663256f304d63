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

// A chunk of values a lane.
template <typename T>
__global__ void __launch_bounds__(kThreads)
dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, int64_t n, uint32_t least, bool none, float scale,
               uint64_t seed, const int64_t* __restrict__ seed_at, T* __restrict__ out) {
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
    const U4 draws = draw_block(seed, kTagDropout, 0, static_cast<uint64_t>(first + i) >> 2);
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
    constexpr int64_t kBlock = kThreads * Chunk<T>::kVec;
    const int64_t blocks = (n + kBlock - 1) / kBlock;
    GS_RETURN_IF_ERROR(check_grid("gs_dropout", blocks, kThreads));
    hipLaunchKernelGGL((dropout_kernel<T>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), static_cast<const T*>(x), static_cast<const T*>(residual), n, least,
                       none, scale, seed, seed_at, static_cast<T*>(out));
    return check_launch("dropout");
  });
}
