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
// Both passes are one read of the scores (and one write); what costs is the
// instructions beside it, so a row is 16 lanes (E <= 256), whose sums are four
// in-register rotations for four rows at once, or 32 or 64 where a lane would
// hold more than 16 values.  (A wave per row with its sums by wave shuffles:
// 28 us for the gradient of 32768 x 256 scores, 62 us for the loss.)  A lane
// holds 4 neighbouring experts of every 4 LANES.  The affinities' sums stay in
// each lane's registers over its rows, are added over the block in LDS and over
// the blocks by the second launch, in a fixed order and in fp32; the counts
// are integer adds, whose order does not show.  The route weights' part of the
// gradient is added up per row in LDS, since its places are any experts.
//
// Measured at 256 experts: 32768 rows (34 MB) 12.7 us for the loss's pass and 5 for
// the block that finishes it, 18 us for the gradient with the route weights'
// (3.7 TB/s), where the 7 sums and the exponentials of a row take as long as its
// bytes; 57 rows 6.5 us, one launch.
//
// Error bits: 1 non-finite score, 2 id >= E, 4 affinities that sum to 0 (with the
// route weights' gradient also those of a row's routes).
#include <algorithm>
#include <type_traits>

#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kMaxExperts = 1024, kMaxTopk = 32, kNoId = 0xffffffffu;
constexpr uint32_t kMaxTokens = (1u << 27) - 1;  // times kMaxTopk below 2^32, the counts' range
constexpr uint32_t kWaves = 4;          // of the gradient's blocks
constexpr uint32_t kBalanceWaves = 16;  // of the loss's, whose partial sums one block adds up:
constexpr uint32_t kBlocks = 128;       // few and large
constexpr float kLog2e = 1.44269504088896340736f;

// log(1 + e) for e in [0, 1]: 2 atanh(z) with z = e / (2 + e) <= 1/3, its
// series up to z^15 (the next term is 2^-27 of the sum at most)
__device__ __forceinline__ float log1p01(float e) {
  const float z = e * __builtin_amdgcn_rcpf(2.0f + e), y = z * z;
  float s = 1.0f / 15.0f;
  s = __builtin_fmaf(s, y, 1.0f / 13.0f);
  s = __builtin_fmaf(s, y, 1.0f / 11.0f);
  s = __builtin_fmaf(s, y, 1.0f / 9.0f);
  s = __builtin_fmaf(s, y, 1.0f / 7.0f);
  s = __builtin_fmaf(s, y, 1.0f / 5.0f);
  s = __builtin_fmaf(s, y, 1.0f / 3.0f);
  s = __builtin_fmaf(s, y, 1.0f);
  return 2.0f * z * s;
}

// b(s) and its derivative.  2^(s log2 e) by the hardware exponential: off by
// 2^-23 of itself and |s| 2^-24 from the exponent's rounding.
template <int MODE>
__device__ __forceinline__ void affinity(float s, float top, float& b, float& slope) {
  if constexpr (MODE == kRouterSoftmax) {
    b = __builtin_amdgcn_exp2f((s - top) * kLog2e);
    slope = b;
  } else {
    const float e = __builtin_amdgcn_exp2f(-fabsf(s) * kLog2e);  // <= 1
    const float sp = fmaxf(s, 0.0f) + log1p01(e);
    const float sig = (s >= 0.0f ? 1.0f : e) * __builtin_amdgcn_rcpf(1.0f + e);
    b = __builtin_amdgcn_sqrtf(sp);
    // sigmoid / softplus tends to 1 where both underflow
    slope = sp > 1e-30f ? 0.5f * sig * __builtin_amdgcn_rcpf(b) : 0.5f * b;
  }
}
// The same for sqrt(softplus) of a score below -80: e^s leaves the normal
// numbers at -87, its root e^(s/2), which b is there to 2^-117 of itself, at -174.
constexpr float kFarScore = -80.0f;
__device__ __forceinline__ void far_affinity(float s, float& b, float& slope) {
  const float x = 0.5f * kLog2e * s;
  b = x >= -126.0f ? __builtin_amdgcn_exp2f(x) : 0.0f;
  slope = 0.5f * b;
}

// the sum or maximum over a row's lanes, in every one of them
template <int ROR>
__device__ __forceinline__ float rotated(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + ROR, 0xf, 0xf, true));
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
  v += rotated<8>(v);
  v += rotated<4>(v);
  v += rotated<2>(v);
  v += rotated<1>(v);
  if constexpr (LANES > 16) v += __shfl_xor(v, 16, 64);
  if constexpr (LANES > 32) v += __shfl_xor(v, 32, 64);
  return v;
}
template <int LANES>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, rotated<8>(v));
  v = fmaxf(v, rotated<4>(v));
  v = fmaxf(v, rotated<2>(v));
  v = fmaxf(v, rotated<1>(v));
  if constexpr (LANES > 16) v = fmaxf(v, __shfl_xor(v, 16, 64));
  if constexpr (LANES > 32) v = fmaxf(v, __shfl_xor(v, 32, 64));
  return v;
}

// Row t of the wave's, LANES lanes of it: lane i holds experts 4 (LANES q + i)
// + c, q < Q.  vec: rows are 16-byte aligned.
template <int MODE, int LANES, int Q>
struct Row {
  static constexpr int N = 4 * Q;
  float b[N], slope[N], top, sum;
  uint32_t wrong;
  bool far;  // some row of the wave has scores below kFarScore
  // scores outside the row
  static constexpr float kOutside = MODE == kRouterSoftmax ? -INFINITY : 0.0f;

  static __device__ __forceinline__ uint32_t expert(int j) {
    return 4 * (LANES * (j / 4) + (threadIdx.x & (LANES - 1))) + j % 4;
  }
  __device__ __forceinline__ void load(const float* s, uint32_t experts, bool vec) {
    // (raw scores in slope)
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const uint32_t e = expert(4 * q);
      if (vec) {
        v4f v{kOutside, kOutside, kOutside, kOutside};
        if (e < experts) v = *reinterpret_cast<const v4f*>(s + e);
#pragma unroll
        for (int c = 0; c < 4; ++c) slope[4 * q + c] = v[c];
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) slope[4 * q + c] = e + c < experts ? s[e + c] : kOutside;
      }
    }
  }
  // the affinities, their derivatives and sum of the row s; what is wrong with
  // it (then the sum is 1 and every affinity 0)
  __device__ __forceinline__ void work(const float* s, uint32_t experts) {
    float bad = 0.0f, least = 0.0f;
    top = 0.0f;
    if constexpr (MODE == kRouterSoftmax) {
      top = slope[0];
#pragma unroll
      for (int j = 1; j < N; ++j) top = fmaxf(top, slope[j]);
      top = row_max<LANES>(top);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) least = fminf(least, slope[j]);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      // 0 for a finite score, else NaN
      const float nan = slope[j] * 0.0f;
      bad += kOutside == 0.0f || expert(j) < experts ? nan : 0.0f;
    }
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float score = slope[j];
      affinity<MODE>(score, top, b[j], slope[j]);
      // (outside the row; of -inf the derivative is a NaN)
      if (expert(j) >= experts) b[j] = slope[j] = 0.0f;
      sum += b[j];
    }
    far = MODE == kRouterSqrtSoftplus && __builtin_amdgcn_ballot_w64(least < kFarScore);
    if (far) {
      // (rare: the scores again, one at a time, for registers of no more)
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float score = expert(j) < experts ? s[expert(j)] : 0.0f;
        if (score < kFarScore) far_affinity(score, b[j], slope[j]);
        sum += b[j];
        asm volatile("" ::: "memory");
      }
    }
    sum = row_sum<LANES>(sum);
    wrong = row_sum<LANES>(bad) == 0.0f ? (sum == 0.0f ? 4u : 0u) : 1u;
    if (wrong) {
      sum = 1.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) b[j] = slope[j] = 0.0f;
    }
  }
};

// what the entry writes, and the loss's weight of a count times a mean affinity
struct Balance {
  float* loss;
  uint32_t* counts;
  float* mean;
  float weight;
};
// the loss from every thread's part of it, by a block of 1024
__device__ __forceinline__ void write_loss(const Balance& to, float term) {
  __shared__ float s_term[16];
  const uint32_t tid = threadIdx.x;
  term = reduce_sum_xor<64>(term);
  if ((tid & 63u) == 0) s_term[tid >> 6] = term;
  __syncthreads();
  if (tid == 0) {
    float total = s_term[0];
    for (int w = 1; w < 16; ++w) total += s_term[w];
    *to.loss = total * to.weight;
  }
}

// A block by itself also finishes: 57 rows of 256 scores 15.3 us a call and
// 27.0 us alone, against 19.2 and 28.9 us with the second launch.  (Two rounds
// of rows in one block: 15.4 and 29.4 us against 19.2 and 28.9.)
template <int MODE, int LANES, int Q>
__global__ __launch_bounds__(64 * kBalanceWaves) void router_balance_kernel(const float* scores, const uint32_t* ids,
                                                                            float* part_sum, uint32_t* part_count,
                                                                            Balance to, uint32_t* err,
                                                                            uint32_t tokens, uint32_t experts,
                                                                            uint32_t topk, bool vec) {
  using R = Row<MODE, LANES, Q>;
  constexpr uint32_t kRows = 64 / LANES, kAll = LANES * R::N;  // rows of a wave, experts held
  constexpr uint32_t kParts = kBalanceWaves * kRows;
  static_assert(kParts * kAll <= 16384, "64 KB of partial sums");
  __shared__ float sums[kParts][kAll];
  __shared__ uint32_t counts[kAll];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, part = wave * kRows + lane / LANES;
  for (uint32_t e = tid; e < kAll; e += 64 * kBalanceWaves) counts[e] = 0;
  __syncthreads();
  float acc[R::N];
#pragma unroll
  for (int j = 0; j < R::N; ++j) acc[j] = 0.0f;
  uint32_t bad = 0;
  for (uint32_t t = blockIdx.x * kParts + part; t < tokens; t += gridDim.x * kParts) {
    R row;
    row.load(scores + (uint64_t)t * experts, experts, vec);
    for (uint32_t k = tid & (LANES - 1); k < topk; k += LANES) {
      const uint32_t id = ids[(uint64_t)t * topk + k];
      if (id < experts) atomicAdd(&counts[id], 1u);
      else bad |= 2u;
    }
    row.work(scores + (uint64_t)t * experts, experts);
    bad |= row.wrong;
    const float inv = 1.0f / row.sum;
#pragma unroll
    for (int j = 0; j < R::N; ++j) acc[j] += row.b[j] * inv;
  }
  // the parts' sums, added up by expert
  float total = 0.0f;
#pragma unroll
  for (int j = 0; j < R::N; ++j) sums[part][R::expert(j)] = acc[j];
  __syncthreads();
  if (tid < experts)
    for (uint32_t i = 0; i < kParts; ++i) total += sums[i][tid];
  if (bad) atomicOr(err, bad);
  if (gridDim.x == 1) {
    float term = 0.0f;
    if (tid < experts) {
      const float m = total / (float)tokens;
      to.counts[tid] = counts[tid];
      to.mean[tid] = m;
      term = (float)counts[tid] * m;
    }
    write_loss(to, term);
  } else if (tid < experts) {
    part_sum[(uint64_t)blockIdx.x * experts + tid] = total;
    part_count[(uint64_t)blockIdx.x * experts + tid] = counts[tid];
  }
}

// The blocks' partial sums, and the loss: one block, whose thread (column,
// part) adds every parts-th block's partials of V neighbouring experts.
template <int V>
__global__ __launch_bounds__(1024) void router_balance_finish_kernel(const float* part_sum, const uint32_t* part_count,
                                                                     Balance to, uint32_t blocks, uint32_t tokens,
                                                                     uint32_t experts) {
  typedef float Sums __attribute__((ext_vector_type(V)));
  typedef uint32_t Counts __attribute__((ext_vector_type(V)));
  __shared__ Sums s_sum[1024];
  __shared__ Counts s_count[1024];
  const uint32_t tid = threadIdx.x, columns = experts / V, parts = 1024 / columns, c = tid % columns, part = tid / columns;
  Sums v = 0.0f;
  Counts n = 0u;
  if (part < parts)
#pragma unroll 8
    for (uint32_t i = part; i < blocks; i += parts) {
      v += *reinterpret_cast<const Sums*>(part_sum + (uint64_t)i * experts + V * c);
      n += *reinterpret_cast<const Counts*>(part_count + (uint64_t)i * experts + V * c);
    }
  s_sum[tid] = v;
  s_count[tid] = n;
  __syncthreads();
  float term = 0.0f;
  if (tid < columns) {
#pragma unroll 4
    for (uint32_t q = 1; q < parts; ++q) {
      v += s_sum[q * columns + tid];
      n += s_count[q * columns + tid];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float m = v[e] / (float)tokens;
      to.counts[V * tid + e] = n[e];
      to.mean[V * tid + e] = m;
      term += (float)n[e] * m;
    }
  }
  write_loss(to, term);
}

template <int MODE, int LANES, int Q>
__global__ __launch_bounds__(64 * kWaves) void router_backward_kernel(
    const float* scores, const uint32_t* ids, const uint32_t* counts, const float* loss_grad,
    const float* weights_grad, float* scores_grad, uint32_t* err, uint32_t tokens, uint32_t experts, uint32_t topk,
    float weight, float scale, bool vec) {
  using R = Row<MODE, LANES, Q>;
  constexpr uint32_t kRows = 64 / LANES, kAll = LANES * R::N, kRoutes = (kMaxTopk + LANES - 1) / LANES;
  __shared__ __align__(16) float extra[kWaves * kRows][kAll];
  const uint32_t lane = threadIdx.x & 63u, part = (threadIdx.x >> 6) * kRows + lane / LANES, i = lane & (LANES - 1);
  float* const mine = extra[part];
  float g[R::N];
  const float up = loss_grad ? *loss_grad * weight : 0.0f;
#pragma unroll
  for (int j = 0; j < R::N; ++j) {
    const uint32_t e = R::expert(j);
    g[j] = loss_grad && e < experts ? (float)counts[e] * up : 0.0f;
  }
  uint32_t bad = 0;
  for (uint32_t t = blockIdx.x * kWaves * kRows + part; t < tokens; t += gridDim.x * kWaves * kRows) {
    const float* const s = scores + (uint64_t)t * experts;
    R row;
    row.load(s, experts, vec);
    // lane r of the row holds routes r, r + LANES, ..: id, upstream gradient, score
    uint32_t id[kRoutes];
    float dw[kRoutes], chosen[kRoutes];
    if (weights_grad) {
#pragma unroll
      for (uint32_t r = 0; r < kRoutes; ++r) {
        const uint32_t k = r * LANES + i;
        id[r] = k < topk ? ids[(uint64_t)t * topk + k] : kNoId;
        dw[r] = k < topk ? weights_grad[(uint64_t)t * topk + k] : 0.0f;
        if (id[r] >= experts) {
          if (k < topk) bad |= 2u;
          id[r] = kNoId;
          dw[r] = 0.0f;
        }
      }
#pragma unroll
      for (uint32_t r = 0; r < kRoutes; ++r) chosen[r] = id[r] != kNoId ? s[id[r]] : 0.0f;
    } else {
      for (uint32_t k = i; k < topk; k += LANES)
        if (ids[(uint64_t)t * topk + k] >= experts) bad |= 2u;
    }
    row.work(s, experts);
    bad |= row.wrong;
    const float inv = 1.0f / row.sum;
    float dot = 0.0f;
#pragma unroll
    for (int j = 0; j < R::N; ++j) dot += g[j] * (row.b[j] * inv);
    dot = row_sum<LANES>(dot);
    float d[R::N];
#pragma unroll
    for (int j = 0; j < R::N; ++j) d[j] = row.slope[j] * inv * (g[j] - dot);
    if (weights_grad) {
      float cb[kRoutes], cs[kRoutes], sum = 0.0f, back = 0.0f;
#pragma unroll
      for (uint32_t r = 0; r < kRoutes; ++r) {
        affinity<MODE>(chosen[r], row.top, cb[r], cs[r]);
        if (row.far && chosen[r] < kFarScore) far_affinity(chosen[r], cb[r], cs[r]);
        if (id[r] == kNoId || row.wrong) cb[r] = cs[r] = 0.0f;
        sum += cb[r];
        back += dw[r] * cb[r];
      }
      sum = row_sum<LANES>(sum);
      back = row_sum<LANES>(back);
      // (below the normal numbers 1 / sum could be infinite)
      const bool none = sum < 0x1p-126f;
      if (none && !row.wrong) {
#pragma unroll
        for (uint32_t r = 0; r < kRoutes; ++r) bad |= id[r] != kNoId ? 4u : 0u;
      }
      const float per = none ? 0.0f : 1.0f / sum, mean = back * per;
#pragma unroll
      for (int q = 0; q < Q; ++q) *reinterpret_cast<v4f*>(mine + R::expert(4 * q)) = v4f{0.f, 0.f, 0.f, 0.f};
      wave_lds_order();
#pragma unroll
      for (uint32_t r = 0; r < kRoutes; ++r)
        if (id[r] != kNoId) atomicAdd(mine + id[r], cs[r] * per * (scale * (dw[r] - mean)));
      wave_lds_order();
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const v4f v = *reinterpret_cast<const v4f*>(mine + R::expert(4 * q));
#pragma unroll
        for (int c = 0; c < 4; ++c) d[4 * q + c] += v[c];
      }
    }
    // (0 times an upstream gradient that is not finite)
    if (row.wrong) {
#pragma unroll
      for (int j = 0; j < R::N; ++j) d[j] = 0.0f;
    }
    float* const out = scores_grad + (uint64_t)t * experts;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const uint32_t e = R::expert(4 * q);
      if (vec) {
        if (e < experts) *reinterpret_cast<v4f*>(out + e) = v4f{d[4 * q], d[4 * q + 1], d[4 * q + 2], d[4 * q + 3]};
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (e + c < experts) out[e + c] = d[4 * q + c];
      }
    }
  }
  if (bad) atomicOr(err, bad);
}

bool shape_ok(uint32_t tokens, uint32_t topk, uint32_t experts) {
  return tokens && tokens <= kMaxTokens && experts && experts <= kMaxExperts && topk && topk <= kMaxTopk && topk <= experts;
}

// lanes of a row and float4s a lane holds
template <typename F>
void with_row(uint32_t experts, F&& f) {
  if (experts <= 64) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 1>{});
  else if (experts <= 128) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
  else if (experts <= 256) f(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
  else if (experts <= 512) f(std::integral_constant<int, 32>{}, std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{});
}
uint32_t row_lanes(uint32_t experts) { return experts <= 256 ? 16 : experts <= 512 ? 32 : 64; }
uint32_t balance_blocks(uint32_t tokens, uint32_t experts) {
  const uint32_t rows = kBalanceWaves * 64 / row_lanes(experts);
  return std::min(kBlocks, (tokens + rows - 1) / rows);
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
template <typename... P>
bool aligned4(P... p) {
  return ((reinterpret_cast<uintptr_t>(p) % 4 == 0) && ...);
}

}  // namespace

uint64_t RouterBalanceWorkspaceBytes(uint32_t tokens, uint32_t topk, uint32_t experts) {
  if (!shape_ok(tokens, topk, experts)) return 0;
  return (uint64_t)balance_blocks(tokens, experts) * experts * 8;
}

St LaunchRouterBalance(const RouterBalanceArgs& a) {
  if (!a.scores || !a.ids || !a.loss || !a.counts || !a.mean || !a.workspace || !a.error_flag || !a.stream)
    return Invalid("router_balance_null_argument");
  if (!shape_ok(a.tokens, a.topk, a.experts)) return Invalid("router_balance_shape_invalid");
  if (a.mode != kRouterSoftmax && a.mode != kRouterSqrtSoftplus) return Invalid("router_balance_mode_invalid");
  if (!__builtin_isfinite(a.coefficient)) return Invalid("router_balance_coefficient_invalid");
  if (!aligned4(a.scores, a.ids, a.loss, a.counts, a.mean, a.error_flag))
    return Invalid("router_balance_alignment_invalid");
  if (a.workspace_bytes < RouterBalanceWorkspaceBytes(a.tokens, a.topk, a.experts) ||
      !aligned16(a.workspace))
    return Invalid("router_balance_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  const uint32_t blocks = balance_blocks(a.tokens, a.experts);
  const bool vec = a.experts % 4 == 0 && aligned16(a.scores);
  float* sums = static_cast<float*>(a.workspace);
  uint32_t* counts = reinterpret_cast<uint32_t*>(sums + (uint64_t)blocks * a.experts);
  const Balance to{a.loss, a.counts, a.mean, (float)((double)a.coefficient * a.experts / ((double)a.tokens * a.topk))};
  with_row(a.experts, [&](auto lanes, auto quads) {
    constexpr int L = decltype(lanes)::value, Q = decltype(quads)::value;
    auto kernel = a.mode == kRouterSoftmax ? router_balance_kernel<kRouterSoftmax, L, Q>
                                           : router_balance_kernel<kRouterSqrtSoftplus, L, Q>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kBalanceWaves), 0, a.stream, a.scores, a.ids, sums, counts,
                       to, a.error_flag, a.tokens, a.experts, a.topk, vec);
  });
  if (blocks > 1) {
    auto finish = a.experts % 4 == 0 ? router_balance_finish_kernel<4> : router_balance_finish_kernel<1>;
    hipLaunchKernelGGL(finish, dim3(1), dim3(1024), 0, a.stream, sums, counts, to, blocks, a.tokens, a.experts);
  }
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
  if (!aligned4(a.scores, a.ids, a.counts, a.loss_grad, a.weights_grad, a.scores_grad, a.error_flag))
    return Invalid("router_backward_alignment_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  // of a score's own term: the loss's weight over T
  const float weight = (float)((double)a.coefficient * a.experts / ((double)a.tokens * a.tokens * a.topk));
  const uint32_t rows = kWaves * 64 / row_lanes(a.experts), blocks = std::min<uint32_t>(1024, (a.tokens + rows - 1) / rows);
  const bool vec = a.experts % 4 == 0 && aligned16(a.scores) && aligned16(a.scores_grad);
  with_row(a.experts, [&](auto lanes, auto quads) {
    constexpr int L = decltype(lanes)::value, Q = decltype(quads)::value;
    auto kernel = a.mode == kRouterSoftmax ? router_backward_kernel<kRouterSoftmax, L, Q>
                                           : router_backward_kernel<kRouterSqrtSoftplus, L, Q>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(64 * kWaves), 0, a.stream, a.scores, a.ids, a.counts, a.loss_grad,
                       a.weights_grad, a.scores_grad, a.error_flag, a.tokens, a.experts, a.topk, weight, a.scale, vec);
  });
  return AfterLaunch("router_backward_launch_failed");
}

}  // namespace pih_amd
