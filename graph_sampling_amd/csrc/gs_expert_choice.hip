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
template <int V>
using N = std::integral_constant<int, V>;

// Order-preserving, both zeros the same, NaN the largest; 0: not to be chosen.
__device__ __forceinline__ uint32_t rank_of(float f) {
  if (f == -__builtin_inff()) return 0;
  if (f != f) return 0xFFFFFFFFu;
  return float_to_ordered(f == 0.0f ? 0.0f : f);
}
// The value that a rank stands for (no difference is left between the zeros).
__device__ __forceinline__ float value_of(uint32_t rank) {
  return __uint_as_float(rank & 0x80000000u ? rank & 0x7FFFFFFFu : ~rank);
}
// A 16-bit value's rank and its expert in one number: of equals the lower expert's is the larger.
template <typename T>
__device__ __forceinline__ uint32_t key_of(T f, int expert) {
  uint32_t b = __builtin_bit_cast(uint16_t, f);
  if (b == 0x8000u) b = 0;
  const uint32_t rank = f != f ? 0xFFFFu : (b & 0x8000u ? ~b & 0xFFFFu : b | 0x8000u);
  return f == static_cast<T>(-__builtin_inff()) ? 0 : rank << 16 | (0xFFFFu - static_cast<uint32_t>(expert));
}
template <typename T>
__device__ __forceinline__ float value_of_key(uint32_t key) {
  const uint32_t rank = key >> 16;
  return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(rank & 0x8000u ? rank & 0x7FFFu : ~rank)));
}

// Lanes of a row of 16 exchange within the instruction, larger groups by shuffles on top.
template <int CTRL>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xf, 0xf, false));
}
constexpr int kSwapNeighbours = 0xb1, kSwapPairs = 0x4e, kMirrorEight = 0x141, kMirrorRow = 0x140;
template <int G, typename F>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, F&& f) {
  if (G >= 2) v = f(v, from_lane<kSwapNeighbours>(v));
  if (G >= 4) v = f(v, from_lane<kSwapPairs>(v));
  if (G >= 8) v = f(v, from_lane<kMirrorEight>(v));
  if (G >= 16) v = f(v, from_lane<kMirrorRow>(v));
#pragma unroll
  for (int m = 16; m < G; m *= 2) v = f(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m, kWave)));
  return v;
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  return __uint_as_float(group_reduce<G>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// G lanes a token, EACH experts a lane, side by side.  A choice is the group's maximum; lane k keeps the k-th.
//   16-bit logits: what is left is what lies below the last choice's key; less that key, with the borrow lost, it comes
//   before all others, so that a look at an expert is a subtraction and a maximum, and nothing is taken out.
//   fp32: the rank that was chosen is taken out in its lane, the first of equals, which has the lowest experts.
// Both are bound by those instructions, and by what is exchanged: as few lanes as there are choices have the fewest experts
// each that will do.  100 003 x 160 fp16, 6 choices, 7 us of bytes, 23 us, vector units issuing in 73 % of the cycles; 16384 x 256
// fp32, 8 choices, shares of all, 3.6 us of bytes, 14 us, 42 %, with four waves a unit in all;
// 500 000 x 27 bf16, 4 choices, 10 us of bytes, 18 us with 4 lanes of 8, 41 with 16 of 4; 500 000 x 264, 140 us with 16 of 20, 403
// with 64 of 16.
template <typename T, int G, int EACH>
__global__ void __launch_bounds__(kThreads)
choose_kernel(const T* __restrict__ logits, int64_t stride, int64_t tokens, int experts, int choices, bool normalize,
              int32_t* __restrict__ chosen, float* __restrict__ weights) {
  const int lane = threadIdx.x % G, group0 = threadIdx.x % kWave / G * G;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  const T* const row = logits + (t < tokens ? t : tokens - 1) * stride;  // (works along, writes nothing)
  constexpr bool kKeys = sizeof(T) == 2;
  constexpr int kRun = EACH % Chunk<T>::kVec == 0 ? Chunk<T>::kVec : EACH % 4 == 0 ? 4 : EACH % 2 == 0 ? 2 : 1;  // read at once
  typedef T Run __attribute__((ext_vector_type(kRun)));
  float v[kKeys ? 1 : EACH];
  uint32_t rank[EACH];  // or keys
#pragma unroll
  for (int j = 0; j < EACH; j += kRun) {
    const int e = lane * EACH + j;
    Run run;
    if (e + kRun <= experts) {
      __builtin_memcpy(&run, row + e, sizeof(Run));
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i) run[i] = e + i < experts ? row[e + i] : static_cast<T>(-__builtin_inff());
    }
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      if constexpr (kKeys) {
        rank[j + i] = key_of(run[i], e + i);
      } else {
        v[j + i] = run[i];
        rank[j + i] = rank_of(run[i]);
      }
    }
  }
  uint32_t top = 0, mine = 0, last = 0;
  int32_t which = -1;
  for (int k = 0; k < choices; ++k) {
    if constexpr (kKeys) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) most = rank[j] - last > most ? rank[j] - last : most;
      const uint32_t next = group_max<G>(most) + last;
      const bool there = next != 0 && (k == 0 || next < last);
      if (!__any(there)) break;  // (nothing is left for any of the wave's tokens)
      if (there) last = next;
      if (there && lane == k) {
        mine = next;
        which = static_cast<int32_t>(0xFFFFu - (next & 0xFFFFu));
      }
      if (k == 0) top = there ? next : 0;
    } else {
      uint32_t best = rank[0];
      int at = 0;
#pragma unroll
      for (int j = 1; j < EACH; ++j) {
        if (rank[j] > best) {
          best = rank[j];
          at = j;
        }
      }
      const uint32_t most = group_max<G>(best);
      if (!__any(most != 0)) break;
      uint64_t equal = __ballot(best == most) >> group0;
      if (G < kWave) equal &= (uint64_t(1) << (G % kWave)) - 1;
      const int winner = __ffsll(static_cast<unsigned long long>(equal)) - 1;
      const int expert = __shfl(lane * EACH + at, group0 + winner, kWave);
      if (k == 0) top = most;
      if (lane == k && most != 0) {
        which = expert;
        mine = most;
      }
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        if (lane == winner && j == at) rank[j] = 0;
    }
  }
  float value, most;
  if constexpr (kKeys) {
    value = value_of_key<T>(mine);
    most = value_of_key<T>(top);
  } else {
    value = value_of(mine);
    most = value_of(top);
  }
  if (top == 0) most = 0.0f;
  const float share = which >= 0 ? expf(value - most) : 0.0f;
  float sum = share;
  if (!normalize) {
    // (By expf, as in the gradient.  exp2 of a product with log2(e), rounded once, is 1.3e-8 of the difference too small, to
    // the same side for all; without normalize 16384 x 256 fp32 takes 12.1 us by expf and 11.0 so, 100 003 x 160 fp16 27 and 24.)
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      if constexpr (kKeys) sum += rank[j] ? expf(value_of_key<T>(rank[j]) - most) : 0.0f;
      else sum += v[j] == -__builtin_inff() ? 0.0f : expf(v[j] - most);
    }
  }
  sum = group_sum<G>(sum);
  if (t < tokens && lane < choices) {
    chosen[t * choices + lane] = which;
    weights[t * choices + lane] = which >= 0 ? share / sum : 0.0f;
  }
}

// G lanes a token: what the chosen experts get is put to its place in LDS, and read, and written, in chunks with the rest.
// Memory bounds large ones: 500 000 x 264 bf16, 264 MB written, 64 us, and as much read without normalize, 128; groups of lanes
// about as many as a third of the chunks lose least at a row's end (500 000 x 27: 14 us with 4, 87 with 64).
template <typename T, int G>
__global__ void __launch_bounds__(kThreads)
choose_grad_kernel(const T* __restrict__ logits, int64_t stride, const int32_t* __restrict__ chosen,
                   const float* __restrict__ weights, const float* __restrict__ dweights, int64_t tokens, int experts,
                   int choices, bool normalize, T* __restrict__ dlogits) {
  extern __shared__ __attribute__((aligned(16))) float s_rows[];
  constexpr int kVec = Chunk<T>::kVec;
  const int lane = threadIdx.x % G, group0 = threadIdx.x % kWave / G * G;
  const int chunks = (experts + kVec - 1) / kVec;
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (kThreads / G) + threadIdx.x / G;
  if (t >= tokens) return;
  float* const s_row = s_rows + threadIdx.x / G * (chunks * kVec);
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
  for (int c = lane; c < chunks; c += G) *reinterpret_cast<Wide<T>*>(s_row + c * kVec) = Wide<T>{};
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // (a group is inside a wave, whose LDS accesses stay in order)
  if (there) s_row[which] += w * (normalize ? dw - d : dw);
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const T* const row = logits + t * stride;
  const bool rest = !normalize && first >= 0 && first < experts;  // all others have shares, too
  const float top = rest ? static_cast<float>(row[first]) : 0.0f, per = __shfl(w, group0, kWave) * d;
  for (int c = lane; c < chunks; c += G) {
    const int e = c * kVec;
    Wide<T> sum = *reinterpret_cast<const Wide<T>*>(s_row + e);
    if (rest) {
      const Wide<T> v = widen<T>(load_chunk(row + e, experts - e));
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum[i] -= v[i] == -__builtin_inff() ? 0.0f : expf(v[i] - top) * per;
    }
    store_chunk(dlogits + t * experts + e, narrow<T>(sum), experts - e);
  }
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
      constexpr int64_t kMost = most_blocks(kThreads) * kTokens;  // tokens a launch
      for (int64_t t = 0; t < tokens; t += kMost) {
        const int64_t here = tokens - t < kMost ? tokens - t : kMost;
        hipLaunchKernelGGL((choose_kernel<T, G, decltype(each)::value>), dim3(static_cast<unsigned>((here + kTokens - 1) / kTokens)),
                           dim3(kThreads), 0, static_cast<hipStream_t>(stream), static_cast<const T*>(logits) + t * stride, stride,
                           here, static_cast<int>(experts), static_cast<int>(choices), normalize != 0, chosen + t * choices,
                           weights + t * choices);
        GS_RETURN_IF_ERROR(check_launch("expert_choose"));
      }
      return static_cast<int>(GS_OK);
    };
    auto four = [&](auto g, auto a, auto b, auto c, auto d) {  // the fewest experts a lane that will do
      constexpr int G = decltype(g)::value;
      if (experts <= G * decltype(a)::value) return go(g, a);
      if (experts <= G * decltype(b)::value) return go(g, b);
      return experts <= G * decltype(c)::value ? go(g, c) : go(g, d);
    };
    if (choices <= 4 && experts <= 32) return four(N<4>(), N<2>(), N<4>(), N<6>(), N<8>());
    if (choices <= 8 && experts <= 64) return four(N<8>(), N<4>(), N<6>(), N<8>(), N<8>());
    if (choices <= 16 && experts <= 192) return four(N<16>(), N<4>(), N<6>(), N<8>(), N<12>());
    if (choices <= 16 && experts <= 384) return four(N<16>(), N<16>(), N<20>(), N<24>(), N<24>());
    if (choices <= 32 && experts <= 512) return four(N<32>(), N<4>(), N<8>(), N<12>(), N<16>());
    if (experts <= 1024) return four(N<kWave>(), N<4>(), N<8>(), N<12>(), N<16>());
    return four(N<kWave>(), N<24>(), N<32>(), N<48>(), N<64>());
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
    const int64_t chunks = (experts + Chunk<T>::kVec - 1) / Chunk<T>::kVec;
    auto go = [&](auto lanes) {
      constexpr int G = decltype(lanes)::value, kTokens = kThreads / G;
      constexpr int64_t kMost = most_blocks(kThreads) * kTokens;
      for (int64_t t = 0; t < tokens; t += kMost) {
        const int64_t here = tokens - t < kMost ? tokens - t : kMost, item = t * choices;
        hipLaunchKernelGGL((choose_grad_kernel<T, G>), dim3(static_cast<unsigned>((here + kTokens - 1) / kTokens)), dim3(kThreads),
                           static_cast<size_t>(kTokens * chunks * Chunk<T>::kVec) * sizeof(float), static_cast<hipStream_t>(stream),
                           logits ? static_cast<const T*>(logits) + t * stride : nullptr, stride, chosen ? chosen + item : nullptr,
                           weights ? weights + item : nullptr, dweights ? dweights + item : nullptr, here,
                           static_cast<int>(experts), static_cast<int>(choices), normalize != 0,
                           static_cast<T*>(dlogits) + t * experts);
        GS_RETURN_IF_ERROR(check_launch("expert_choose_grad"));
      }
      return static_cast<int>(GS_OK);
    };
    if (choices <= 4 && chunks <= 8) return go(N<4>());
    if (choices <= 8 && chunks <= 24) return go(N<8>());
    if (choices <= 16 && chunks <= 64) return go(N<16>());
    if (choices <= 32 && chunks <= 128) return go(N<32>());
    return go(N<kWave>());
  });
}

}  // extern "C"
