// Gated feed-forward block and its gradients for gfx950:
//   gate = x Wg^T,  up = x Wu^T,  h = silu(gate) up,  y = h Wd^T
//   dh = dy Wd,  dup = dh silu(gate),  dgate = dh up silu'(gate),
//   dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dWd = dy^T h
// with gate clamped from above and up from both sides where there is a limit
// (no gradient beyond it).
//
// h, dgate and dup are rounded to bf16 for the matrix cores: 2^-9 of each
// element at most, independent from element to element, in sums that are
// rounded to bf16 once themselves.  gate, up and dh stay in fp32 between
// their product and the activation.
#include <algorithm>

#include "kernels.hpp"
#include "tile64.hpp"

namespace pih_amd {
namespace {

// With s the logistic function of g = min(gate, limit) and u the clamped up:
// silu(g) = g s, silu'(g) = s + g s (1 - s).
__device__ __forceinline__ float logistic(float g) {
  // (g -> -inf: exp -> inf, 1 / inf = 0)
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896340736f * g));
}
// (not fminf, which drops a NaN)
__device__ __forceinline__ float at_most(float v, float limit) { return v > limit ? limit : v; }
__device__ __forceinline__ float within(float v, float limit) { return v > limit ? limit : v < -limit ? -limit : v; }

__device__ __forceinline__ float activated(float gate, float up, float limit) {
  const float g = at_most(gate, limit);
  return g * logistic(g) * within(up, limit);
}

struct MlpArgs {
  const uint16_t* a;
  const uint16_t* b;
  const uint16_t* b2;
  uint32_t m, n, k;
  uint16_t* out;
  uint16_t* gate;
  uint16_t* up;
  uint16_t* dgate;
  uint16_t* dup;
  float limit;
};

// h of a 64 x 64 tile
__global__ __launch_bounds__(256) void mlp_up64_kernel(MlpArgs p) {
  __shared__ __align__(16) Plane64 sa, sb;
  const uint32_t m0 = blockIdx.y * kT64, n0 = blockIdx.x * kT64;
  v4f gate[2][2] = {}, up[2][2] = {};
  multiply64<false, false>(sa, sb, gate, {p.a, p.k, p.m}, {p.b, p.k, p.n}, m0, n0, p.k);
  multiply64<false, false>(sa, sb, up, {p.a, p.k, p.m}, {p.b2, p.k, p.n}, m0, n0, p.k);
  each64(m0, n0, [&](uint32_t r, uint32_t c, int i, int j) {
    if (r >= p.m || c >= p.n) return;
    const uint64_t at = (uint64_t)r * p.n + c;
    v4f h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = activated(gate[i][j][e], up[i][j][e], p.limit);
    *reinterpret_cast<uint2*>(p.out + at) = bf16x4(h);
    if (p.gate) {
      *reinterpret_cast<uint2*>(p.gate + at) = bf16x4(gate[i][j]);
      *reinterpret_cast<uint2*>(p.up + at) = bf16x4(up[i][j]);
    }
  });
}

// out = A . B^T of a 64 x 64 tile, with A2 . B2^T of the same k added where
// there is a second pair; AK, BK: stored [k][row]
template <bool AK, bool BK>
__global__ __launch_bounds__(256) void mlp_product64_kernel(MlpArgs p, const uint16_t* a2) {
  __shared__ __align__(16) Plane64 sa, sb;
  const uint32_t m0 = blockIdx.y * kT64, n0 = blockIdx.x * kT64, lda = AK ? p.m : p.k, ldb = BK ? p.n : p.k;
  v4f acc[2][2] = {};
  multiply64<AK, BK>(sa, sb, acc, {p.a, lda, p.m}, {p.b, ldb, p.n}, m0, n0, p.k);
  if (a2) multiply64<AK, BK>(sa, sb, acc, {a2, lda, p.m}, {p.b2, ldb, p.n}, m0, n0, p.k);
  each64(m0, n0, [&](uint32_t r, uint32_t c, int i, int j) {
    if (r < p.m && c < p.n) *reinterpret_cast<uint2*>(p.out + (uint64_t)r * p.n + c) = bf16x4(acc[i][j]);
  });
}

// dh of a 64 x 64 tile, and what follows of it: dgate, dup and h
__global__ __launch_bounds__(256) void mlp_dh64_kernel(MlpArgs p) {
  __shared__ __align__(16) Plane64 sa, sb;
  const uint32_t m0 = blockIdx.y * kT64, n0 = blockIdx.x * kT64;
  v4f dh[2][2] = {};
  multiply64<false, true>(sa, sb, dh, {p.a, p.k, p.m}, {p.b, p.n, p.n}, m0, n0, p.k);
  each64(m0, n0, [&](uint32_t r, uint32_t c, int i, int j) {
    if (r >= p.m || c >= p.n) return;
    const uint64_t at = (uint64_t)r * p.n + c;
    const uint2 gw = *reinterpret_cast<const uint2*>(p.gate + at), uw = *reinterpret_cast<const uint2*>(p.up + at);
    v4f dg, du, h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float gate = bf16_bits_to_f32(((e < 2 ? gw.x : gw.y) >> (16 * (e & 1))) & 0xffffu);
      const float up = bf16_bits_to_f32(((e < 2 ? uw.x : uw.y) >> (16 * (e & 1))) & 0xffffu);
      const float g = at_most(gate, p.limit), u = within(up, p.limit), s = logistic(g), silu = g * s, d = dh[i][j][e];
      dg[e] = gate > p.limit ? 0.0f : d * u * (s + silu * (1.0f - s));
      du[e] = up > p.limit || up < -p.limit ? 0.0f : d * silu;
      h[e] = silu * u;
    }
    *reinterpret_cast<uint2*>(p.dgate + at) = bf16x4(dg);
    *reinterpret_cast<uint2*>(p.dup + at) = bf16x4(du);
    *reinterpret_cast<uint2*>(p.out + at) = bf16x4(h);
  });
}

bool shape_ok(uint32_t rows, uint32_t inter, uint32_t hidden) {
  return rows && rows <= (1u << 20) && inter && hidden && inter % 8 == 0 && hidden % 8 == 0 && inter <= (1u << 17) &&
         hidden <= (1u << 17);
}
bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }
dim3 tiles64(uint32_t m, uint32_t n) { return dim3((n + kT64 - 1) / kT64, (m + kT64 - 1) / kT64); }
// (a clamp that nothing passes; infinities stay what they are)
float limit_of(const GatedMlpArgs& a) { return a.limit > 0.0f ? a.limit : INFINITY; }

}  // namespace

uint64_t GatedMlpWorkspaceBytes(uint32_t rows, uint32_t inter, uint32_t hidden) {
  if (!shape_ok(rows, inter, hidden)) return 0;
  return padded((uint64_t)rows * inter * 2);
}

uint64_t GatedMlpBackwardWorkspaceBytes(uint32_t rows, uint32_t inter, uint32_t hidden) {
  if (!shape_ok(rows, inter, hidden)) return 0;
  return 3 * padded((uint64_t)rows * inter * 2);
}

St LaunchGatedMlp(const GatedMlpArgs& a) {
  if (!a.x || !a.wg || !a.wu || !a.wd || !a.y || !a.workspace || !a.stream || !a.gate != !a.up)
    return Invalid("gated_mlp_null_argument");
  if (!shape_ok(a.rows, a.inter, a.hidden)) return Invalid("gated_mlp_shape_invalid");
  if (!__builtin_isfinite(a.limit)) return Invalid("gated_mlp_limit_invalid");
  if (!aligned(a.x) || !aligned(a.wg) || !aligned(a.wu) || !aligned(a.wd) || !aligned(a.y) || !aligned(a.gate) ||
      !aligned(a.up))
    return Invalid("gated_mlp_alignment_invalid");
  if (a.workspace_bytes < GatedMlpWorkspaceBytes(a.rows, a.inter, a.hidden) || !aligned(a.workspace))
    return Invalid("gated_mlp_workspace_invalid");
  if (a.y == a.x || (a.gate && (a.gate == a.x || a.up == a.x || a.gate == a.up || a.gate == a.y || a.up == a.y)))
    return Invalid("gated_mlp_alias_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  MlpArgs p{};
  p.a = a.x;
  p.b = a.wg;
  p.b2 = a.wu;
  p.m = a.rows;
  p.n = a.inter;
  p.k = a.hidden;
  p.out = static_cast<uint16_t*>(a.workspace);
  p.gate = a.gate;
  p.up = a.up;
  p.limit = limit_of(a);
  hipLaunchKernelGGL(mlp_up64_kernel, tiles64(a.rows, a.inter), dim3(256), 0, a.stream, p);
  MlpArgs q{};
  q.a = p.out;
  q.b = a.wd;
  q.m = a.rows;
  q.n = a.hidden;
  q.k = a.inter;
  q.out = a.y;
  hipLaunchKernelGGL((mlp_product64_kernel<false, false>), tiles64(q.m, q.n), dim3(256), 0, a.stream, q, nullptr);
  return AfterLaunch("gated_mlp_launch_failed");
}

St LaunchGatedMlpBackward(const GatedMlpArgs& a) {
  if (!a.dy || !a.x || !a.wg || !a.wu || !a.wd || !a.gate || !a.up || !a.workspace || !a.stream ||
      (!a.dx && !a.dwg && !a.dwu && !a.dwd))
    return Invalid("gated_mlp_backward_null_argument");
  if (!shape_ok(a.rows, a.inter, a.hidden)) return Invalid("gated_mlp_backward_shape_invalid");
  if (!__builtin_isfinite(a.limit)) return Invalid("gated_mlp_backward_limit_invalid");
  const void* const inputs[] = {a.dy, a.x, a.wg, a.wu, a.wd, a.gate, a.up};
  const void* const results[] = {a.dx, a.dwg, a.dwu, a.dwd};
  for (const void* i : inputs)
    if (!aligned(i)) return Invalid("gated_mlp_backward_alignment_invalid");
  for (int r = 0; r < 4; ++r) {
    if (!aligned(results[r])) return Invalid("gated_mlp_backward_alignment_invalid");
    for (const void* i : inputs)
      if (results[r] == i) return Invalid("gated_mlp_backward_alias_invalid");
    for (int s = 0; s < r; ++s)
      if (results[r] && results[r] == results[s]) return Invalid("gated_mlp_backward_alias_invalid");
  }
  if (a.workspace_bytes < GatedMlpBackwardWorkspaceBytes(a.rows, a.inter, a.hidden) || !aligned(a.workspace))
    return Invalid("gated_mlp_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  const uint64_t plane = padded((uint64_t)a.rows * a.inter * 2);
  uint16_t* const dgate = reinterpret_cast<uint16_t*>(ws);
  uint16_t* const dup = reinterpret_cast<uint16_t*>(ws + plane);
  uint16_t* const h = reinterpret_cast<uint16_t*>(ws + 2 * plane);
  MlpArgs p{};
  p.a = a.dy;
  p.b = a.wd;
  p.m = a.rows;
  p.n = a.inter;
  p.k = a.hidden;
  p.out = h;
  p.gate = a.gate;
  p.up = a.up;
  p.dgate = dgate;
  p.dup = dup;
  p.limit = limit_of(a);
  hipLaunchKernelGGL(mlp_dh64_kernel, tiles64(p.m, p.n), dim3(256), 0, a.stream, p);
  if (a.dx) {
    MlpArgs q{};
    q.a = dgate;
    q.b = a.wg;
    q.b2 = a.wu;
    q.m = a.rows;
    q.n = a.hidden;
    q.k = a.inter;
    q.out = a.dx;
    hipLaunchKernelGGL((mlp_product64_kernel<false, true>), tiles64(q.m, q.n), dim3(256), 0, a.stream, q, dup);
  }
  auto weight = [&](const uint16_t* rows, const uint16_t* cols, uint32_t m, uint32_t n, uint16_t* out) {
    if (!out) return;
    MlpArgs q{};
    q.a = rows;
    q.b = cols;
    q.m = m;
    q.n = n;
    q.k = a.rows;
    q.out = out;
    hipLaunchKernelGGL((mlp_product64_kernel<true, true>), tiles64(m, n), dim3(256), 0, a.stream, q, nullptr);
  };
  weight(dgate, a.x, a.inter, a.hidden, a.dwg);
  weight(dup, a.x, a.inter, a.hidden, a.dwu);
  weight(a.dy, h, a.hidden, a.inter, a.dwd);
  return AfterLaunch("gated_mlp_backward_launch_failed");
}

}  // namespace pih_amd
