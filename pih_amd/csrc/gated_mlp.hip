// Gated feed-forward block and its gradients for gfx950:
//   gate = x Wg^T,  up = x Wu^T,  h = silu(gate) up,  y = h Wd^T
//   dh = dy Wd,  dup = dh silu(gate),  dgate = dh up silu'(gate),
//   dx = dgate Wg + dup Wu,  dWg = dgate^T x,  dWu = dup^T x,  dWd = dy^T h
// with gate clamped from above and up from both sides where there is a limit
// (no gradient beyond it).
//
// h, dgate and dup are rounded to bf16 for the matrix cores: 2^-8 of each
// element at most, independent from element to element, in sums that are
// rounded to bf16 once themselves (y, dx and the weights' gradients 0.23 % of
// their norm off 64 bits, 0.17 % of it their own rounding).  gate, up and dh stay
// in fp32 between their product and the activation.
//
// Forward two products, backward four, of which a product with too few tiles for
// the CUs has k in parts, joined by a launch of its own.  Gate and up are one
// product whose tile holds 16 columns of each in turn, so that a wave has both of
// an element and leaves h; dh's tile reads gate and up and leaves dgate and dup
// side by side, so that dx is one product over both weights and their gradients
// one over both halves, and h for dWd.
//
// Measured: 1 row of 4096 x 2048 15 us (50 MB; the host's time of a call), 57 rows
// of 4096 x 12288 69 us (302 MB at 4.4 TB/s: gate and up 5.4, down 4.6), 4099 rows
// with gate and up kept 0.92-0.94 ms (1.33 PFLOP/s); gradients of 4096 rows 1.93-2.01 ms
// (1.25 PFLOP/s), of 509 rows of 7168 x 2048 142-145 us (0.62 PFLOP/s).  Many rows: the matrix
// pipe at the clock that power leaves (1.9 GHz; a library product of 4096 x 24576 x
// 4096 takes 650-750 us over and over, 550 with pauses), and in the gradients what the
// tiles of a round write at once (dh's 165 MB, ~50 us of a round) and the transposing
// reads of the weights' gradients (12 % more cycles).
// Few rows: the weights' bytes; 509 rows: 64-row tiles, bound by what a CU takes in.
#include "dense_route.hpp"
#include "dma_tile.hpp"
#include "tile64.hpp"

namespace pih_amd {
namespace {

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
    const v4f gate = bf16x4_to_f32(*reinterpret_cast<const uint2*>(p.gate + at));
    const v4f up = bf16x4_to_f32(*reinterpret_cast<const uint2*>(p.up + at));
    v4f dg, du, h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const GluGrad d = glu_grad(dh[i][j][e], gate[e], up[e], p.limit);
      dg[e] = d.dgate;
      du[e] = d.dup;
      h[e] = d.h;
    }
    *reinterpret_cast<uint2*>(p.dgate + at) = bf16x4(dg);
    *reinterpret_cast<uint2*>(p.dup + at) = bf16x4(du);
    *reinterpret_cast<uint2*>(p.out + at) = bf16x4(h);
  });
}

// ------------------------------------------- products split over k
// A product with too few tiles for the CUs leaves fp32 sums, a plane per split,
// which these join in order.

// h, and gate and up where they are kept: the sums' columns are 16 of gate and 16
// of up in turn
__global__ __launch_bounds__(256) void mlp_join_glu_kernel(const float* sums, uint32_t splits, uint64_t plane,
                                                           uint16_t* h, uint16_t* gate, uint16_t* up, uint64_t count,
                                                           uint32_t inter, float limit) {
  for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += (uint64_t)gridDim.x * 1024) {
    const uint32_t c = (uint32_t)(i % inter);
    const float* const from = sums + i / inter * (2 * (uint64_t)inter) + c / 16 * 32 + c % 16;
    v4f g = *reinterpret_cast<const v4f*>(from), u = *reinterpret_cast<const v4f*>(from + 16);
#pragma unroll 4
    for (uint32_t s = 1; s < splits; ++s) {
      g += *reinterpret_cast<const v4f*>(from + s * plane);
      u += *reinterpret_cast<const v4f*>(from + s * plane + 16);
    }
    v4f v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = activated(g[e], u[e], limit);
    *reinterpret_cast<uint2*>(h + i) = bf16x4(v);
    if (gate) {
      *reinterpret_cast<uint2*>(gate + i) = bf16x4(g);
      *reinterpret_cast<uint2*>(up + i) = bf16x4(u);
    }
  }
}

// dgate, dup (side by side, rows 2 inter long) and h of dh; zeros for the rows
// from count / inter up to a multiple of 64
__global__ __launch_bounds__(256) void mlp_join_dh_kernel(const float* sums, uint32_t splits, uint64_t plane,
                                                          const uint16_t* gate, const uint16_t* up, uint16_t* dgu,
                                                          uint16_t* h, uint64_t count, uint64_t padded, uint32_t inter,
                                                          float limit) {
  for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < padded; i += (uint64_t)gridDim.x * 1024) {
    v4f dg{0.f, 0.f, 0.f, 0.f}, du = dg, v = dg;
    if (i < count) {
      v4f dh = *reinterpret_cast<const v4f*>(sums + i);
#pragma unroll 4
      for (uint32_t s = 1; s < splits; ++s) dh += *reinterpret_cast<const v4f*>(sums + s * plane + i);
      const v4f g = bf16x4_to_f32(*reinterpret_cast<const uint2*>(gate + i));
      const v4f u = bf16x4_to_f32(*reinterpret_cast<const uint2*>(up + i));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const GluGrad d = glu_grad(dh[e], g[e], u[e], limit);
        dg[e] = d.dgate;
        du[e] = d.dup;
        v[e] = d.h;
      }
    }
    uint16_t* const row = dgu + i / inter * (2 * (uint64_t)inter) + i % inter;
    *reinterpret_cast<uint2*>(row) = bf16x4(dg);
    *reinterpret_cast<uint2*>(row + inter) = bf16x4(du);
    *reinterpret_cast<uint2*>(h + i) = bf16x4(v);
  }
}

__global__ __launch_bounds__(256) void mlp_join_kernel(const float* sums, uint32_t splits, uint64_t plane, uint16_t* out,
                                                       uint64_t count) {
  for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += (uint64_t)gridDim.x * 1024) {
    v4f v = *reinterpret_cast<const v4f*>(sums + i);
#pragma unroll 4
    for (uint32_t s = 1; s < splits; ++s) v += *reinterpret_cast<const v4f*>(sums + s * plane + i);
    *reinterpret_cast<uint2*>(out + i) = bf16x4(v);
  }
}
dim3 join_grid(uint64_t count) { return dim3((uint32_t)std::min<uint64_t>((count + 1023) / 1024, 1u << 16)); }

// EPI for the rows in one part, SUM and join(sums, first row, rows, splits,
// elements of a plane) for those in several; rest(first row, rows) does the rows
// behind the whole 256 where rest_apart
template <bool BT, int EPI, int SUM, typename A, typename J, typename R>
St run_route(const Route& r, BigArgs p, float* sums, hipStream_t s, A&& advance, J&& join, bool rest_apart, R&& rest) {
  const uint32_t m = p.m;
  p.splits = 1;
  if (r.whole) {
    p.m = r.whole;
    launch_rows<256, false, BT, EPI>(p, s);
    if (r.whole == m) return Ok();
    if (rest_apart) return rest(r.whole, m - r.whole);
    advance(p, r.whole);
    p.m = m - r.whole;
  }
  if (r.rest.splits > 1) {
    p.splits = r.rest.splits;
    p.split_stride = (uint64_t)p.m * p.n;
    p.out = sums;
    p.ldo = p.n;
    if (r.rest.rows == 64) launch_rows<64, false, BT, SUM>(p, s);
    else if (r.rest.rows == 128) launch_rows<128, false, BT, SUM>(p, s);
    else launch_rows<256, false, BT, SUM>(p, s);
    join(r.whole, p.m, p.splits, p.split_stride);
  } else {
    if (r.rest.rows == 64) launch_rows<64, false, BT, EPI>(p, s);
    else if (r.rest.rows == 128) launch_rows<128, false, BT, EPI>(p, s);
    else launch_rows<256, false, BT, EPI>(p, s);
  }
  return Ok();
}

bool shape_ok(uint32_t rows, uint32_t inter, uint32_t hidden) {
  return rows && rows <= (1u << 20) && inter && hidden && inter % 8 == 0 && hidden % 8 == 0 && inter <= (1u << 17) &&
         hidden <= (1u << 17);
}
bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }
dim3 tiles64(uint32_t m, uint32_t n) { return dim3((n + kT64 - 1) / kT64, (m + kT64 - 1) / kT64); }
// The tiles fed by DMA take 64-deep steps of every product; other sizes run on 64 x 64
// tiles, us at 1024 rows of 1024 x 4096 -> of 1000 x 4008: forward 41 -> 178, gradients
// 131 -> 507; at 1 row 13 -> 116 and 42 -> 224
bool dma_takes(uint32_t inter, uint32_t hidden) { return inter % KB == 0 && hidden % KB == 0; }
// Few rows: the tiles of gemm_tile.hip, chosen per shape for all CUs without
// splits, against the route here, by both estimates (what those tiles take, in pairs
// or walked by a block per CU, is underestimated by 15 % against these: 4096 x 12288,
// down on them in spite of it at 180 rows 106 -> 97 us, at 257 147 -> 139, but walked
// at 2049 552 -> 585, and gate and up at 180 rows 106 -> 114).  Forward pass, us, route -> tiles for
// gate and up -> for down too: 1 row of 4096 x 2048 23.8 -> 19.1 -> 15.9, of 4096
// x 12288 64.9 -> 57.1 -> 52.0; 57 rows 35.0 -> 25.0 -> 19.1 and 78.9 -> 67.4 ->
// 58.7; 512 rows 59.2 -> 51.6 -> 43.0, but 157.9 -> 209.4 -> 223.8.  The same
// choice for the rows behind the whole 256 of a route: 1030 rows of 4096 x 12288
// 334 -> 321, 4099 rows 964 -> 943.
bool tiles_faster(uint32_t m, uint32_t n, uint32_t k, bool pair, float route_us) {
  const TilePick t = PickTile(true, m, n, 2 * k, 1, pair);
  return (pair || t.grid ? 1.15 : 1.0) * t.us < route_us;
}
struct ForwardPlan {
  Route up, down;
  bool up_tiles, down_tiles;            // all rows
  bool up_rest_tiles, down_rest_tiles;  // the rows behind the whole 256 of the route
  uint64_t sums, bytes;
};
ForwardPlan forward_plan(uint32_t rows, uint32_t inter, uint32_t hidden) {
  ForwardPlan p{};
  p.sums = padded((uint64_t)rows * inter * 2);
  p.bytes = p.sums;
  if (!dma_takes(inter, hidden)) return p;
  p.up = route_of(rows, 2 * inter, hidden);
  p.down = route_of(rows, hidden, inter);
  auto up_tiles = [&](uint32_t m, float us) {
    TileGluArgs t;
    t.m = m;
    t.inter = inter;
    t.k = hidden;
    return TileGluTakes(t) && tiles_faster(m, 2 * inter, hidden, true, us);
  };
  // LaunchBf16Gemm, where it runs those tiles, or up to 64 rows the GEMV, which takes
  // the intermediate sizes that those do not (inter % 128 == 64).  Forward pass, us,
  // route -> GEMV for down at 8, 17, 33 and 64 rows: 12352 -> 4096 53.6 -> 51.8, 55.6 ->
  // 59.8, 59.8 -> 71.0, 64.3 -> 91; 4160 -> 1024 16.5 -> 14.8, 17.5 -> 17.8, 19.0 -> 22.4,
  // 21.5 -> 30.7; 2112 -> 4096 20.5 -> 15.7, 22.5 -> 18.0, 25.4 -> 22.3, 30.9 -> 29.0.  Above
  // 64 rows it would run them on the 128 x 256 tiles without splits: 12352 -> 4096
  // at 192 rows 104 on the route, 152 there, 5696 -> 2048 at 65 rows 32 and 68.
  auto down_tiles = [&](uint32_t m, float us) {
    if (Bf16EstimateHolds(m, hidden, inter)) return tiles_faster(m, hidden, inter, false, us);
    return m <= 64 && Bf16GemvUs(m, hidden, inter) < us;
  };
  p.up_tiles = up_tiles(rows, p.up.us);
  p.down_tiles = down_tiles(rows, p.down.us);
  p.up_rest_tiles = p.up.whole && p.up.whole < rows && up_tiles(rows - p.up.whole, p.up.rest.us);
  p.down_rest_tiles = p.down.whole && p.down.whole < rows && down_tiles(rows - p.down.whole, p.down.rest.us);
  p.bytes += padded(std::max(p.up_tiles || p.up_rest_tiles ? 0 : p.up.sums,
                             p.down_tiles || p.down_rest_tiles ? 0 : p.down.sums) * 4);
  return p;
}
struct BackwardPlan {
  Route dh, dx;
  uint64_t h, sums, bytes;
};
BackwardPlan backward_plan(uint32_t rows, uint32_t inter, uint32_t hidden) {
  BackwardPlan p{};
  const uint64_t plane = (uint64_t)(rows + 63) / 64 * 64 * inter * 2;
  p.h = padded(2 * plane);
  p.bytes = p.sums = p.h + padded(plane);
  if (!dma_takes(inter, hidden)) return p;
  p.dh = route_of(rows, inter, hidden);
  p.dx = route_of(rows, hidden, 2 * inter);
  p.bytes += padded(std::max(p.dh.sums, p.dx.sums) * 4);
  return p;
}
// (a clamp that nothing passes; infinities stay what they are)
float limit_of(const GatedMlpArgs& a) { return a.limit > 0.0f ? a.limit : INFINITY; }

}  // namespace

uint64_t GatedMlpWorkspaceBytes(uint32_t rows, uint32_t inter, uint32_t hidden) {
  if (!shape_ok(rows, inter, hidden)) return 0;
  return forward_plan(rows, inter, hidden).bytes;
}

uint64_t GatedMlpBackwardWorkspaceBytes(uint32_t rows, uint32_t inter, uint32_t hidden) {
  if (!shape_ok(rows, inter, hidden)) return 0;
  return backward_plan(rows, inter, hidden).bytes;
}

St LaunchGatedMlp(const GatedMlpArgs& a) {
  if (!a.x || !a.wg || !a.wu || !a.wd || !a.y || !a.workspace || !a.stream || !a.gate != !a.up)
    return Invalid("gated_mlp_null_argument");
  if (!shape_ok(a.rows, a.inter, a.hidden)) return Invalid("gated_mlp_shape_invalid");
  if (!__builtin_isfinite(a.limit)) return Invalid("gated_mlp_limit_invalid");
  if (!aligned(a.x) || !aligned(a.wg) || !aligned(a.wu) || !aligned(a.wd) || !aligned(a.y) || !aligned(a.gate) ||
      !aligned(a.up))
    return Invalid("gated_mlp_alignment_invalid");
  const ForwardPlan plan = forward_plan(a.rows, a.inter, a.hidden);
  if (a.workspace_bytes < plan.bytes || !aligned(a.workspace)) return Invalid("gated_mlp_workspace_invalid");
  const uint64_t of_rows = (uint64_t)a.rows * a.hidden * 2, of_inter = (uint64_t)a.rows * a.inter * 2,
                 of_weight = (uint64_t)a.inter * a.hidden * 2;
  const Span results[] = {{a.y, of_rows}, {a.gate, of_inter}, {a.up, of_inter}};
  const Span inputs[] = {{a.x, of_rows}, {a.wg, of_weight}, {a.wu, of_weight}, {a.wd, of_weight}};
  if (ResultsOverlap(results, inputs)) return Invalid("gated_mlp_alias_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint16_t* const h = static_cast<uint16_t*>(a.workspace);
  if (dma_takes(a.inter, a.hidden)) {
    float* const sums = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + plan.sums);
    auto up_on_tiles = [&](uint32_t first, uint32_t rows) {
      const uint64_t from = (uint64_t)first * a.inter;
      TileGluArgs t;
      t.x = a.x + (uint64_t)first * a.hidden;
      t.wg = a.wg;
      t.wu = a.wu;
      t.h = h + from;
      t.gate = a.gate ? a.gate + from : nullptr;
      t.up = a.up ? a.up + from : nullptr;
      t.stream = a.stream;
      t.m = rows;
      t.inter = a.inter;
      t.k = a.hidden;
      t.limit = limit_of(a);
      return LaunchTileGlu(t);
    };
    auto down_on_tiles = [&](uint32_t first, uint32_t rows) {
      Bf16GemmArgs g;
      g.a = h + (uint64_t)first * a.inter;
      g.w = a.wd;
      g.out = a.y + (uint64_t)first * a.hidden;
      g.stream = a.stream;
      g.m = rows;
      g.n = a.hidden;
      g.k = a.inter;
      return LaunchBf16Gemm(g);
    };
    St up = Ok();
    if (plan.up_tiles) {
      up = up_on_tiles(0, a.rows);
    } else {
      BigArgs p{};
      p.a = a.x;
      p.b = a.wg;
      p.b2 = a.wu;
      p.m = a.rows;
      p.n = 2 * a.inter;
      p.k = p.k_valid = a.hidden;
      p.lda = p.ldb = a.hidden;
      p.out = h;
      p.ldo = a.inter;
      p.gate = a.gate;
      p.up = a.up;
      p.limit = limit_of(a);
      up = run_route<false, kEpiGlu, kEpiGluSum>(
          plan.up, p, sums, a.stream,
          [&](BigArgs& q, uint32_t rows) {
            q.a += (uint64_t)rows * a.hidden;
            q.out = h + (uint64_t)rows * a.inter;
            if (a.gate) {
              q.gate += (uint64_t)rows * a.inter;
              q.up += (uint64_t)rows * a.inter;
            }
          },
          [&](uint32_t first, uint32_t rows, uint32_t splits, uint64_t plane) {
            const uint64_t from = (uint64_t)first * a.inter, count = (uint64_t)rows * a.inter;
            hipLaunchKernelGGL(mlp_join_glu_kernel, join_grid(count), dim3(256), 0, a.stream, sums, splits, plane, h + from,
                               a.gate ? a.gate + from : nullptr, a.up ? a.up + from : nullptr, count, a.inter, p.limit);
          },
          plan.up_rest_tiles, up_on_tiles);
    }
    if (!up.ok()) return up;
    if (plan.down_tiles) return down_on_tiles(0, a.rows);
    BigArgs q{};
    q.a = h;
    q.b = a.wd;
    q.m = a.rows;
    q.n = a.hidden;
    q.out_rows = a.rows;
    q.k = q.k_valid = a.inter;
    q.lda = q.ldb = a.inter;
    q.out = a.y;
    q.ldo = a.hidden;
    q.b_steps = 0xffffffffu;
    const St down = run_route<false, kEpiStore, kEpiSum>(
        plan.down, q, sums, a.stream,
        [&](BigArgs& r, uint32_t rows) {
          r.a += (uint64_t)rows * a.inter;
          r.out = a.y + (uint64_t)rows * a.hidden;
        },
        [&](uint32_t first, uint32_t rows, uint32_t splits, uint64_t plane) {
          const uint64_t count = (uint64_t)rows * a.hidden;
          hipLaunchKernelGGL(mlp_join_kernel, join_grid(count), dim3(256), 0, a.stream, sums, splits, plane,
                             a.y + (uint64_t)first * a.hidden, count);
        },
        plan.down_rest_tiles, down_on_tiles);
    return down.ok() ? AfterLaunch("gated_mlp_launch_failed") : down;
  }
  MlpArgs p{};
  p.a = a.x;
  p.b = a.wg;
  p.b2 = a.wu;
  p.m = a.rows;
  p.n = a.inter;
  p.k = a.hidden;
  p.out = h;
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
  const uint64_t of_rows = (uint64_t)a.rows * a.hidden * 2, of_inter = (uint64_t)a.rows * a.inter * 2,
                 of_weight = (uint64_t)a.inter * a.hidden * 2;
  const Span inputs[] = {{a.dy, of_rows},   {a.x, of_rows},     {a.wg, of_weight}, {a.wu, of_weight},
                         {a.wd, of_weight}, {a.gate, of_inter}, {a.up, of_inter}};
  const Span results[] = {{a.dx, of_rows}, {a.dwg, of_weight}, {a.dwu, of_weight}, {a.dwd, of_weight}};
  for (const Span& i : inputs)
    if (!aligned(i.p)) return Invalid("gated_mlp_backward_alignment_invalid");
  for (const Span& r : results)
    if (!aligned(r.p)) return Invalid("gated_mlp_backward_alignment_invalid");
  if (ResultsOverlap(results, inputs)) return Invalid("gated_mlp_backward_alias_invalid");
  const BackwardPlan plan = backward_plan(a.rows, a.inter, a.hidden);
  if (a.workspace_bytes < plan.bytes || !aligned(a.workspace)) return Invalid("gated_mlp_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  uint16_t* const h = reinterpret_cast<uint16_t*>(ws + plan.h);
  if (dma_takes(a.inter, a.hidden)) {
    uint16_t* const dgu = reinterpret_cast<uint16_t*>(ws);  // [rows up to a multiple of 64][dgate, dup]
    float* const sums = reinterpret_cast<float*>(ws + plan.sums);
    const uint32_t row_up = (a.rows + 63) / 64 * 64;
    BigArgs p{};
    p.a = a.dy;
    p.b = a.wd;
    p.m = a.rows;
    p.n = a.inter;
    p.k = p.k_valid = a.hidden;
    p.lda = a.hidden;
    p.ldb = a.inter;
    p.out = dgu;
    p.ldo = 2 * a.inter;
    p.h = h;
    p.ldh = a.inter;
    p.gate = a.gate;
    p.up = a.up;
    p.b_steps = 0xffffffffu;
    p.limit = limit_of(a);
    run_route<true, kEpiGluGrad, kEpiSum>(
        plan.dh, p, sums, a.stream,
        [&](BigArgs& q, uint32_t rows) {
          q.a += (uint64_t)rows * a.hidden;
          q.out = dgu + (uint64_t)rows * 2 * a.inter;
          q.h += (uint64_t)rows * a.inter;
          q.gate += (uint64_t)rows * a.inter;
          q.up += (uint64_t)rows * a.inter;
        },
        [&](uint32_t first, uint32_t rows, uint32_t splits, uint64_t plane) {
          const uint64_t from = (uint64_t)first * a.inter, count = (uint64_t)rows * a.inter;
          const uint64_t up_to = (uint64_t)(row_up - first) * a.inter;
          hipLaunchKernelGGL(mlp_join_dh_kernel, join_grid(up_to), dim3(256), 0, a.stream, sums, splits, plane,
                             a.gate + from, a.up + from, dgu + 2 * from, h + from, count, up_to, a.inter, p.limit);
        },
        false, [](uint32_t, uint32_t) { return Ok(); });
    if (a.dx) {
      BigArgs q{};
      q.a = dgu;
      q.b = a.wg;
      q.b2 = a.wu;
      q.b_steps = a.inter / KB;
      q.m = q.out_rows = a.rows;
      q.n = a.hidden;
      q.k = q.k_valid = 2 * a.inter;
      q.lda = 2 * a.inter;
      q.ldb = a.hidden;
      q.out = a.dx;
      q.ldo = a.hidden;
      run_route<true, kEpiStore, kEpiSum>(
          plan.dx, q, sums, a.stream,
          [&](BigArgs& r, uint32_t rows) {
            r.a += (uint64_t)rows * 2 * a.inter;
            r.out = a.dx + (uint64_t)rows * a.hidden;
          },
          [&](uint32_t first, uint32_t rows, uint32_t splits, uint64_t plane) {
            const uint64_t count = (uint64_t)rows * a.hidden;
            hipLaunchKernelGGL(mlp_join_kernel, join_grid(count), dim3(256), 0, a.stream, sums, splits, plane,
                               a.dx + (uint64_t)first * a.hidden, count);
          },
          false, [](uint32_t, uint32_t) { return Ok(); });
    }
    // the weights' gradients, columns of A against columns of B over the rows
    auto weight = [&](const uint16_t* from, uint32_t ld, uint32_t from_valid, uint32_t m, const uint16_t* with,
                      uint32_t with_valid, uint32_t n, uint16_t* out, uint16_t* out2, uint32_t out_rows) {
      BigArgs q{};
      q.a = from;
      q.b = with;
      q.m = m;
      q.n = n;
      q.k = row_up;
      q.a_valid = from_valid;
      q.k_valid = with_valid;
      q.lda = ld;
      q.ldb = q.ldo = n;
      q.out = out;
      q.out2 = out2;
      q.out_rows = out_rows;
      q.b_steps = 0xffffffffu;
      launch_rows<256, true, true, kEpiStore>(q, a.stream);
    };
    if (a.dwg && a.dwu) weight(dgu, 2 * a.inter, row_up, 2 * a.inter, a.x, a.rows, a.hidden, a.dwg, a.dwu, a.inter);
    else if (a.dwg) weight(dgu, 2 * a.inter, row_up, a.inter, a.x, a.rows, a.hidden, a.dwg, nullptr, a.inter);
    else if (a.dwu) weight(dgu + a.inter, 2 * a.inter, row_up, a.inter, a.x, a.rows, a.hidden, a.dwu, nullptr, a.inter);
    if (a.dwd) weight(a.dy, a.hidden, a.rows, a.hidden, h, row_up, a.inter, a.dwd, nullptr, a.hidden);
    return AfterLaunch("gated_mlp_backward_launch_failed");
  }
  uint16_t* const dgate = reinterpret_cast<uint16_t*>(ws);
  uint16_t* const dup = dgate + (uint64_t)a.rows * a.inter;
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
