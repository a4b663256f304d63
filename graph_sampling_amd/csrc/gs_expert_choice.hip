// The choice of experts from a router's logits, and its gradient, on gfx950.
//
//   experts[t, :] = the K experts with the largest of logits[t, :], largest first, the lower one of equals
//   weights[t, k] = exp(logits[t, experts[t, k]] - top) / sum,  the sum over the chosen ones (normalized) or over all
//   d logits[t, j] = weight_j * (dweights_j - d)   normalized: j chosen, d = sum over k of weights_k * dweights_k, else 0
//                  = weight_j * dweights_j - share_j * d   otherwise (share: of all; weight_j: 0 where not chosen)
//
// A logit of -infinity stands for an expert that the token may not choose: it is never taken, and where no other is
// left, experts[t, k] = -1 with weight 0.  NaN is larger than everything, and makes the token's weights NaN.  No
// counterpart in the reference.
#include "gs_rows.hpp"

namespace gs {
namespace {

constexpr int kThreads = 256;

// Order-preserving, both zeros the same, NaN the largest; 0: not to be chosen.
__device__ __forceinline__ uint32_t rank_of(float f) {
  if (f == -__builtin_inff()) return 0;
  if (f != f) return 0xFFFFFFFFu;
  return float_to_ordered(f == 0.0f ? 0.0f : f);
}

template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int m = G / 2; m > 0; m /= 2) {
    const uint32_t other = __shfl_xor(v, m, kWave);
    v = other > v ? other : v;
  }
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int m = G / 2; m > 0; m /= 2) v += __shfl_xor(v, m, kWave);
  return v;
}

// G lanes a token, EACH experts a lane, side by side: of equals the first lane has the lower ones.  A choice is the group's
// maximum; lane k keeps the k-th.
template <typename T, int G, int EACH>
__global__ void __launch_bounds__(kThreads)
choose_kernel(const T* __restrict__ logits, int64_t stride, int64_t tokens, int experts, int choices, bool normalize,
              int32_t* __restrict__ chosen, float* __restrict__ weights) {
  const int lane = threadIdx.x % G, group0 = threadIdx.x % kWave / G * G;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  const T* const row = logits + (t < tokens ? t : tokens - 1) * stride;  // (works along, writes nothing)
  float v[EACH];
  uint32_t rank[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int e = lane * EACH + j;
    v[j] = e < experts ? static_cast<float>(row[e]) : -__builtin_inff();
    rank[j] = rank_of(v[j]);
  }
  float top = 0.0f, mine = 0.0f;
  int32_t which = -1;
  for (int k = 0; k < choices; ++k) {
    uint32_t best = rank[0];
    float value = v[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < EACH; ++j) {
      if (rank[j] > best) {
        best = rank[j];
        value = v[j];
        at = j;
      }
    }
    const uint32_t most = group_max<G>(best);
    if (most == 0) break;  // (nothing is left for this token)
    uint64_t equal = __ballot(best == most) >> group0;
    if (G < kWave) equal &= (uint64_t(1) << (G % kWave)) - 1;
    const int winner = __ffsll(static_cast<unsigned long long>(equal)) - 1;
    const float taken = __shfl(value, group0 + winner, kWave);
    const int expert = __shfl(lane * EACH + at, group0 + winner, kWave);
    if (k == 0) top = taken;
    if (lane == k) {
      which = expert;
      mine = taken;
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (lane == winner && j == at) rank[j] = 0;
  }
  const float share = which >= 0 ? expf(mine - top) : 0.0f;
  float sum = share;
  if (!normalize) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += v[j] == -__builtin_inff() ? 0.0f : expf(v[j] - top);
  }
  sum = group_sum<G>(sum);
  if (t < tokens && lane < choices) {
    chosen[t * choices + lane] = which;
    weights[t * choices + lane] = which >= 0 ? share / sum : 0.0f;
  }
}

// G lanes a token: its row is put together in LDS, and written in chunks.
template <typename T, int G>
__global__ void __launch_bounds__(kThreads)
choose_grad_kernel(const T* __restrict__ logits, int64_t stride, const int32_t* __restrict__ chosen,
                   const float* __restrict__ weights, const float* __restrict__ dweights, int64_t tokens, int experts,
                   int choices, bool normalize, T* __restrict__ dlogits) {
  extern __shared__ float s_rows[];
  const int lane = threadIdx.x % G, group0 = threadIdx.x % kWave / G * G;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  if (t >= tokens) return;
  float* const s_row = s_rows + threadIdx.x / G * experts;
  float w = 0.0f, dw = 0.0f;
  int32_t which = -1;
  if (lane < choices) {
    which = chosen[t * choices + lane];
    w = weights[t * choices + lane];
    dw = dweights[t * choices + lane];
  }
  const bool there = which >= 0 && which < experts;
  const float d = group_sum<G>(there ? w * dw : 0.0f);
  const int32_t first = __shfl(which, group0, kWave);
  const bool any = first >= 0 && first < experts;
  if (normalize || !any) {
    for (int e = lane; e < experts; e += G) s_row[e] = 0.0f;
  } else {
    const T* const row = logits + t * stride;
    const float top = static_cast<float>(row[first]), per = __shfl(w, group0, kWave) * d;
    for (int e = lane; e < experts; e += G) {
      const float v = static_cast<float>(row[e]);
      s_row[e] = v == -__builtin_inff() ? 0.0f : -(expf(v - top) * per);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (a group is inside a wave, whose LDS accesses stay in order)
  if (there) s_row[which] += w * (normalize ? dw - d : dw);
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  for (int e = lane; e < experts; e += G) dlogits[t * experts + e] = static_cast<T>(s_row[e]);
}

int check_choice(const char* what, int64_t tokens, int64_t experts, int64_t choices, int type, int64_t stride) {
  GS_REQUIRE(type == GS_F32 || type == GS_F16 || type == GS_BF16,
             "%s: value type %d is none of GS_F32, GS_F16, GS_BF16", what, type);
  GS_REQUIRE(tokens >= 0 && experts >= 0 && choices >= 0 && stride >= 0, "%s: negative size", what);
  GS_REQUIRE(experts <= 4096, "%s: %lld experts, at most 4096 are taken", what, static_cast<long long>(experts));
  GS_REQUIRE(choices <= 64 && choices <= experts, "%s: %lld choices of %lld experts, at most 64 and no more than there are "
             "experts are taken", what, static_cast<long long>(choices), static_cast<long long>(experts));
  GS_REQUIRE(choices == 0 || tokens <= ((int64_t(1) << 31) - 1) / choices,
             "%s: tokens x choices, at most 2^31 - 1 are taken", what);
  return GS_OK;
}

}  // namespace
}  // namespace gs

using namespace gs;

extern "C" {

int gs_expert_choose(const void* logits, int64_t stride, int type, int64_t tokens, int64_t experts, int64_t choices,
                     int normalize, int32_t* chosen, float* weights, void* stream) {
  GS_RETURN_IF_ERROR(check_choice("gs_expert_choose", tokens, experts, choices, type, stride));
  if (tokens == 0 || choices == 0) return GS_OK;
  GS_REQUIRE(logits && chosen && weights, "gs_expert_choose: null array");
  GS_REQUIRE(aligned_to(logits, value_bytes(type)), "gs_expert_choose: logits not aligned to their type");
  return with_value_type(type, "gs_expert_choose", [&](auto zero) {
    using T = decltype(zero);
    auto go = [&](auto lanes, auto each) {
      constexpr int G = decltype(lanes)::value, kTokens = kThreads / G;
      const int64_t blocks = (tokens + kTokens - 1) / kTokens;
      GS_RETURN_IF_ERROR(check_grid("gs_expert_choose", blocks, kThreads));
      hipLaunchKernelGGL((choose_kernel<T, G, decltype(each)::value>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads),
                         0, static_cast<hipStream_t>(stream), static_cast<const T*>(logits), stride, tokens,
                         static_cast<int>(experts), static_cast<int>(choices), normalize != 0, chosen, weights);
      return check_launch("expert_choose");
    };
    using Few = std::integral_constant<int, 16>;
    using All = std::integral_constant<int, kWave>;
    if (choices <= 16 && experts <= 256) {
      if (experts <= 16) return go(Few(), std::integral_constant<int, 1>());
      if (experts <= 64) return go(Few(), std::integral_constant<int, 4>());
      return go(Few(), std::integral_constant<int, 16>());
    }
    if (experts <= 256) return go(All(), std::integral_constant<int, 4>());
    if (experts <= 1024) return go(All(), std::integral_constant<int, 16>());
    return go(All(), std::integral_constant<int, 64>());
  });
}

int gs_expert_choose_grad(const void* logits, int64_t stride, int type, const int32_t* chosen, const float* weights,
                          const float* dweights, int64_t tokens, int64_t experts, int64_t choices, int normalize,
                          void* dlogits, void* stream) {
  GS_RETURN_IF_ERROR(check_choice("gs_expert_choose_grad", tokens, experts, choices, type, stride));
  if (tokens == 0 || experts == 0) return GS_OK;
  GS_REQUIRE(dlogits && (normalize || logits) && (choices == 0 || (chosen && weights && dweights)),
             "gs_expert_choose_grad: null array");
  GS_REQUIRE(aligned_to(logits, value_bytes(type)) && aligned_to(dlogits, value_bytes(type)),
             "gs_expert_choose_grad: logits not aligned to their type");
  return with_value_type(type, "gs_expert_choose_grad", [&](auto zero) {
    using T = decltype(zero);
    auto go = [&](auto lanes) {
      constexpr int G = decltype(lanes)::value, kTokens = kThreads / G;
      const int64_t blocks = (tokens + kTokens - 1) / kTokens;
      GS_RETURN_IF_ERROR(check_grid("gs_expert_choose_grad", blocks, kThreads));
      hipLaunchKernelGGL((choose_grad_kernel<T, G>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads),
                         kTokens * static_cast<size_t>(experts) * sizeof(float), static_cast<hipStream_t>(stream),
                         static_cast<const T*>(logits), stride, chosen, weights, dweights, tokens,
                         static_cast<int>(experts), static_cast<int>(choices), normalize != 0, static_cast<T*>(dlogits));
      return check_launch("expert_choose_grad");
    };
    return choices <= 16 && experts <= 256 ? go(std::integral_constant<int, 16>())
                                           : go(std::integral_constant<int, kWave>());
  });
}

}  // extern "C"
