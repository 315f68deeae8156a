// MoE router training terms for gfx950, beside the router top-k: the balance
// loss with the experts' route counts, and the gradient of the raw scores.
//
// With b = exp(s - max) (softmax) or sqrt(softplus(s)) and p = b / sum(b):
//   c_e = routes to expert e,  P_e = 1/T sum_t p_te,
//   L   = coefficient E / (T k) sum_e c_e P_e;
//   dL/ds_te = b'_te / sum(b) (g_e - sum_j g_j p_tj),
//              g_e = dL coefficient E / (T^2 k) c_e,
// b' = db/ds: b itself (softmax; the shift by the maximum cancels), and for
// sqrt(softplus) sigmoid(s) / (2 b) = b/2 sigmoid(s)/softplus(s).  The route
// weights w_j = scale b_j / sum over the k selected (both modes) add
//   b'_j scale / S (dw_j - sum_i dw_i b_i / S),  S = sum of the selected b.
//
// Both passes are one read of the scores (and one write): a wavefront per
// row, lane l holds experts l, l + 64, ... as the top-k kernel does, the row
// sums by xor shuffles.  The affinities' sums stay in each wave's registers
// over its rows, are added over the block's waves in LDS and over the blocks
// by the second launch, in a fixed order and in fp32; the counts are integer
// adds, whose order does not show.
//
// Error bits: 1 non-finite score, 2 id >= E, 4 affinities that sum to 0.
#include <algorithm>

#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kMaxExperts = 1024, kMaxTopk = 32;
constexpr uint32_t kWaves = 4;
// rows per wave below which another block costs more than it saves
constexpr uint32_t kBlocks = 256;

// b(s) and its derivative
template <int MODE>
__device__ __forceinline__ void affinity(float s, float top, float& b, float& slope) {
  if constexpr (MODE == kRouterSoftmax) {
    b = expf(s - top);
    slope = b;
  } else {
    const float e = expf(-fabsf(s));  // <= 1
    const float sp = fmaxf(s, 0.0f) + log1pf(e);
    const float sig = s >= 0.0f ? 1.0f / (1.0f + e) : e / (1.0f + e);
    b = sqrtf(sp);
    // sigmoid / softplus tends to 1 where both underflow
    slope = sp > 1e-30f ? 0.5f * sig / b : 0.5f * b;
  }
}

// the row's b, b' and their sum; bits of what is wrong with it (then the sum
// is 1 and every b is 0)
template <int MODE, int PER>
__device__ __forceinline__ uint32_t row_affinities(const float* s, uint32_t lane, uint32_t experts, float (&b)[PER],
                                                   float (&slope)[PER], float& sum) {
  float raw[PER], top = -INFINITY;
  bool finite = true;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t e = lane + 64u * j;
    raw[j] = e < experts ? s[e] : 0.0f;
    if (e < experts) {
      finite &= __builtin_isfinite(raw[j]);
      top = fmaxf(top, raw[j]);
    }
  }
  const bool bad = __builtin_amdgcn_ballot_w64(!finite) != 0;
  if constexpr (MODE == kRouterSoftmax) top = reduce_max_xor<64>(top);
  float part = 0.0f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t e = lane + 64u * j;
    b[j] = slope[j] = 0.0f;
    if (e < experts && !bad) {
      affinity<MODE>(raw[j], top, b[j], slope[j]);
      part += b[j];
    }
  }
  sum = reduce_sum_xor<64>(part);
  if (bad || sum == 0.0f) {
    sum = 1.0f;
    return bad ? 1u : 4u;
  }
  return 0u;
}

template <int MODE, int PER>
__global__ __launch_bounds__(64 * kWaves) void router_balance_kernel(const float* scores, const uint32_t* ids,
                                                                     float* part_sum, uint32_t* part_count,
                                                                     uint32_t* err, uint32_t tokens, uint32_t experts,
                                                                     uint32_t topk) {
  __shared__ float sums[kWaves][64 * PER];
  __shared__ uint32_t counts[64 * PER];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
  for (uint32_t e = tid; e < 64 * PER; e += 64 * kWaves) counts[e] = 0;
  __syncthreads();
  float acc[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) acc[j] = 0.0f;
  uint32_t bad = 0;
  for (uint32_t t = blockIdx.x * kWaves + wave; t < tokens; t += gridDim.x * kWaves) {
    if (lane < topk) {
      const uint32_t id = ids[(uint64_t)t * topk + lane];
      if (id < experts) atomicAdd(&counts[id], 1u);
      else bad |= 2u;
    }
    float b[PER], slope[PER], sum;
    bad |= row_affinities<MODE, PER>(scores + (uint64_t)t * experts, lane, experts, b, slope, sum);
    const float inv = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[j] += b[j] * inv;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) sums[wave][lane + 64u * j] = acc[j];
  __syncthreads();
  for (uint32_t e = tid; e < experts; e += 64 * kWaves) {
    float v = sums[0][e];
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) v += sums[w][e];
    part_sum[(uint64_t)blockIdx.x * experts + e] = v;
    part_count[(uint64_t)blockIdx.x * experts + e] = counts[e];
  }
  if (bad) atomicOr(err, bad);
}

// The blocks' partial sums, and the loss: one block, thread (e, part) adds
// every parts-th block's partial of expert e.
__global__ __launch_bounds__(1024) void router_balance_finish_kernel(const float* part_sum, const uint32_t* part_count,
                                                                     float* loss, uint32_t* counts, float* mean,
                                                                     uint32_t blocks, uint32_t tokens,
                                                                     uint32_t experts, float weight) {
  __shared__ float s_sum[1024];
  __shared__ uint32_t s_count[1024];
  __shared__ float s_term[16];
  const uint32_t tid = threadIdx.x, parts = 1024 / experts, e = tid % experts, part = tid / experts;
  float v = 0.0f;
  uint32_t c = 0;
  if (part < parts)
    for (uint32_t i = part; i < blocks; i += parts) {
      v += part_sum[(uint64_t)i * experts + e];
      c += part_count[(uint64_t)i * experts + e];
    }
  s_sum[tid] = v;
  s_count[tid] = c;
  __syncthreads();
  float term = 0.0f;
  if (tid < experts) {
    for (uint32_t q = 1; q < parts; ++q) {
      v += s_sum[q * experts + tid];
      c += s_count[q * experts + tid];
    }
    const float m = v / (float)tokens;
    counts[tid] = c;
    mean[tid] = m;
    term = (float)c * m;
  }
  term = reduce_sum_xor<64>(term);
  if ((tid & 63u) == 0) s_term[tid >> 6] = term;
  __syncthreads();
  if (tid == 0) {
    float total = s_term[0];
    for (int w = 1; w < 16; ++w) total += s_term[w];
    *loss = total * weight;
  }
}

template <int MODE, int PER>
__global__ __launch_bounds__(64 * kWaves) void router_backward_kernel(
    const float* scores, const uint32_t* ids, const uint32_t* counts, const float* loss_grad,
    const float* weights_grad, float* scores_grad, uint32_t* err, uint32_t tokens, uint32_t experts, uint32_t topk,
    float weight, float scale) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  float g[PER];
  const float up = loss_grad ? *loss_grad * weight : 0.0f;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const uint32_t e = lane + 64u * j;
    g[j] = loss_grad && e < experts ? (float)counts[e] * up : 0.0f;
  }
  uint32_t bad = 0;
  for (uint32_t t = blockIdx.x * kWaves + wave; t < tokens; t += gridDim.x * kWaves) {
    float b[PER], slope[PER], sum;
    const uint32_t wrong =
        row_affinities<MODE, PER>(scores + (uint64_t)t * experts, lane, experts, b, slope, sum);
    bad |= wrong;
    const float inv = 1.0f / sum;
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) dot += g[j] * (b[j] * inv);
    dot = reduce_sum_xor<64>(dot);
    float d[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) d[j] = slope[j] * inv * (g[j] - dot);
    uint32_t id = 0xffffffffu;
    if (lane < topk) {
      id = ids[(uint64_t)t * topk + lane];
      if (id >= experts) {
        bad |= 2u;
        id = 0xffffffffu;
      }
    }
    if (weights_grad) {
      // lane r < k holds route r; its b comes from the lane that owns the expert
      float dw = lane < topk && id != 0xffffffffu ? weights_grad[(uint64_t)t * topk + lane] : 0.0f;
      float mine = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float v = __shfl(b[j], (int)(id & 63u), 64);
        if (id != 0xffffffffu && (id >> 6) == (uint32_t)j) mine = v;
      }
      const float chosen = reduce_sum_xor<64>(mine);
      const float scaled = chosen > 0.0f ? 1.0f / chosen : 0.0f;
      const float back = reduce_sum_xor<64>(dw * (mine * scaled));
      const float term = scale * scaled * (dw - back);
      for (uint32_t r = 0; r < topk; ++r) {
        const uint32_t rid = (uint32_t)__builtin_amdgcn_readlane((int)id, r);
        if (rid == 0xffffffffu) continue;
        const float v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, term), r));
        if ((rid & 63u) == lane) {
#pragma unroll
          for (int j = 0; j < PER; ++j)
            if ((rid >> 6) == (uint32_t)j) d[j] += slope[j] * v;
        }
      }
    }
    float* out = scores_grad + (uint64_t)t * experts;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint32_t e = lane + 64u * j;
      if (e < experts) out[e] = wrong ? 0.0f : d[j];
    }
  }
  if (bad) atomicOr(err, bad);
}

uint32_t balance_blocks(uint32_t tokens) { return std::min(kBlocks, (tokens + kWaves - 1) / kWaves); }

bool shape_ok(uint32_t tokens, uint32_t topk, uint32_t experts) {
  return tokens && experts && experts <= kMaxExperts && topk && topk <= kMaxTopk && topk <= experts;
}

template <typename F>
void with_per(uint32_t experts, F&& f) {
  const uint32_t per = (experts + 63) / 64;
  if (per <= 1) f(std::integral_constant<int, 1>{});
  else if (per <= 2) f(std::integral_constant<int, 2>{});
  else if (per <= 4) f(std::integral_constant<int, 4>{});
  else if (per <= 8) f(std::integral_constant<int, 8>{});
  else f(std::integral_constant<int, 16>{});
}

}  // namespace

uint64_t RouterBalanceWorkspaceBytes(uint32_t tokens, uint32_t topk, uint32_t experts) {
  if (!shape_ok(tokens, topk, experts)) return 0;
  return (uint64_t)balance_blocks(tokens) * experts * 8;
}

St LaunchRouterBalance(const RouterBalanceArgs& a) {
  if (!a.scores || !a.ids || !a.loss || !a.counts || !a.mean || !a.workspace || !a.error_flag || !a.stream)
    return Invalid("router_balance_null_argument");
  if (!shape_ok(a.tokens, a.topk, a.experts)) return Invalid("router_balance_shape_invalid");
  if (a.mode != kRouterSoftmax && a.mode != kRouterSqrtSoftplus) return Invalid("router_balance_mode_invalid");
  if (!__builtin_isfinite(a.coefficient)) return Invalid("router_balance_coefficient_invalid");
  if (a.workspace_bytes < RouterBalanceWorkspaceBytes(a.tokens, a.topk, a.experts) ||
      reinterpret_cast<uintptr_t>(a.workspace) % 4)
    return Invalid("router_balance_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  const uint32_t blocks = balance_blocks(a.tokens);
  float* sums = static_cast<float*>(a.workspace);
  uint32_t* counts = reinterpret_cast<uint32_t*>(sums + (uint64_t)blocks * a.experts);
  with_per(a.experts, [&](auto per) {
    constexpr int PER = decltype(per)::value;
    auto kernel = a.mode == kRouterSoftmax ? router_balance_kernel<kRouterSoftmax, PER>
                                           : router_balance_kernel<kRouterSqrtSoftplus, PER>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, a.stream, a.scores, a.ids, sums, counts,
                       a.error_flag, a.tokens, a.experts, a.topk);
  });
  const float weight = (float)((double)a.coefficient * a.experts / ((double)a.tokens * a.topk));
  hipLaunchKernelGGL(router_balance_finish_kernel, dim3(1), dim3(1024), 0, a.stream, sums, counts, a.loss, a.counts,
                     a.mean, blocks, a.tokens, a.experts, weight);
  return AfterLaunch("router_balance_launch_failed");
}

St LaunchRouterBackward(const RouterBackwardArgs& a) {
  if (!a.scores || !a.ids || !a.scores_grad || !a.error_flag || !a.stream || (a.loss_grad && !a.counts) ||
      (!a.loss_grad && !a.weights_grad))
    return Invalid("router_backward_null_argument");
  if (!shape_ok(a.tokens, a.topk, a.experts)) return Invalid("router_backward_shape_invalid");
  if (a.mode != kRouterSoftmax && a.mode != kRouterSqrtSoftplus) return Invalid("router_backward_mode_invalid");
  if (!__builtin_isfinite(a.coefficient)) return Invalid("router_backward_coefficient_invalid");
  if (!__builtin_isfinite(a.scale) || a.scale <= 0.0f) return Invalid("router_backward_scale_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  // of a score's own term: the loss's weight over T
  const float weight = (float)((double)a.coefficient * a.experts / ((double)a.tokens * a.tokens * a.topk));
  const uint32_t blocks = std::min<uint32_t>(2048, (a.tokens + kWaves - 1) / kWaves);
  with_per(a.experts, [&](auto per) {
    constexpr int PER = decltype(per)::value;
    auto kernel = a.mode == kRouterSoftmax ? router_backward_kernel<kRouterSoftmax, PER>
                                           : router_backward_kernel<kRouterSqrtSoftplus, PER>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, a.stream, a.scores, a.ids, a.counts, a.loss_grad,
                       a.weights_grad, a.scores_grad, a.error_flag, a.tokens, a.experts, a.topk, weight, a.scale);
  });
  return AfterLaunch("router_backward_launch_failed");
}

}  // namespace pih_amd
