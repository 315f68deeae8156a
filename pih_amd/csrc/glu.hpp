// The gated feed-forward block's activation and its gradient, element by element.
#pragma once

#include "device_common.hpp"

namespace pih_amd {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// With s the logistic function of g = min(gate, limit) and u the clamped up:
// silu(g) = g s, silu'(g) = s + g s (1 - s).
__device__ __forceinline__ float logistic(float g) {
  // (g -> -inf: exp -> inf, 1 / inf = 0)
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));
}
// (not fminf, which drops a NaN)
__device__ __forceinline__ float at_most(float v, float limit) { return v > limit ? limit : v; }
__device__ __forceinline__ float within(float v, float limit) { return v > limit ? limit : v < -limit ? -limit : v; }
__device__ __forceinline__ float activated(float gate, float up, float limit) {
  const float g = at_most(gate, limit);
  return g * logistic(g) * within(up, limit);
}
// from dh, gate and up: dgate, dup and h
struct GluGrad {
  float dgate, dup, h;
};
__device__ __forceinline__ GluGrad glu_grad(float dh, float gate, float up, float limit) {
  const float g = at_most(gate, limit), u = within(up, limit), s = logistic(g), silu = g * s;
  return {gate > limit ? 0.0f : dh * u * (s + silu * (1.0f - s)), up > limit || up < -limit ? 0.0f : dh * silu, silu * u};
}
// four bf16 values of a uint2
__device__ __forceinline__ v4f bf16x4_to_f32(uint2 v) {
  return v4f{bf16_bits_to_f32(v.x & 0xffffu), bf16_bits_to_f32(v.x >> 16), bf16_bits_to_f32(v.y & 0xffffu),
             bf16_bits_to_f32(v.y >> 16)};
}
__device__ __forceinline__ uint2 bf16x4(v4f v) { return uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])}; }

}  // namespace
}  // namespace pih_amd
