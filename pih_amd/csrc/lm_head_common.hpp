// What the LM head's losses share beside the DMA tiles (dma_tile.hpp): the
// products of hidden sizes that those do not take, the rows' upstream factors
// and the plan of a backward pass over pieces of the vocabulary.
#pragma once

#include "dma_tile.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kErrTarget = 1u, kErrLoss = 4u;
constexpr uint32_t TS = 64, KS = 64, kPitch = KS + 8;

typedef uint16_t Tile16[TS][kPitch];

// C [m][n] = A . B^T over k.  A: [m][k] with row stride lda, B: [n][k].
struct GemmArgs {
  const uint16_t* a;
  const uint16_t* b;
  uint32_t m, n, k;
  uint64_t lda, ldb;
  void* out;            // kEpiGrad: bf16
  uint64_t ldo;
  // rows of the result are x rows, columns vocabulary entries from v0 on
  const uint32_t* target;
  const float* lse;
  const float* mantissa;  // kEpiGrad: [m]
  float2* stats;        // [m][stat_tiles]
  float* target_logit;  // [m]
  uint32_t v0, vocab, stat_tiles;
  float inverse;        // kEpiTeacher*: 1 / temperature
  const float* most;    // kEpiTeacherGrad: what a row's exponentials sum to
};

// 64 x 64 elements of an operand into LDS, zeros outside
__device__ __forceinline__ void stage(Tile16& s, const uint16_t* p, uint64_t ld, uint32_t r0, uint32_t rows, uint32_t k0,
                                      uint32_t k) {
  for (uint32_t i = threadIdx.x; i < TS * KS / 8; i += 256) {
    const uint32_t r = i / 8, c = i % 8 * 8;
    v4i v{0, 0, 0, 0};
    if (r0 + r < rows && k0 + c < k) v = *reinterpret_cast<const v4i*>(p + (uint64_t)(r0 + r) * ld + k0 + c);
    *reinterpret_cast<v4i*>(&s[r][c]) = v;
  }
}

// The logits' product for hidden sizes that are no multiple of 64.  Tile of
// 64 x 64: four waves of 32 x 32.  The MFMA's first operand is B, so that a
// lane's four results are consecutive columns of one row.  1024 rows, 32768
// entries: 267 us at hidden 1000 (251 TFLOP/s), the tiles below 70 us at 1024.
template <int EPI>
__global__ __launch_bounds__(256) void loss_gemm_kernel(GemmArgs p) {
  __shared__ __align__(16) Tile16 sa, sb;
  __shared__ float tile[TS][TS + 1];
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const uint32_t m0 = blockIdx.x * TS, n0 = blockIdx.y * TS, wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  v4f acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i / 2][i % 2] = v4f{0.f, 0.f, 0.f, 0.f};
  for (uint32_t k0 = 0; k0 < p.k; k0 += KS) {
    stage(sa, p.a, p.lda, m0, p.m, k0, p.k);
    stage(sb, p.b, p.ldb, n0, p.n, k0, p.k);
    __syncthreads();
#pragma unroll
    for (uint32_t q = 0; q < KS; q += 32) {
      v4i a[2], b[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = *reinterpret_cast<const v4i*>(&sa[wm + 16 * i + lr][q + 8 * lg]);
        b[i] = *reinterpret_cast<const v4i*>(&sb[wn + 16 * i + lr][q + 8 * lg]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b[j]),
                                                              __builtin_bit_cast(v8bf, a[i]), acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) tile[wm + 16 * i + lr][wn + 16 * j + 4 * lg + e] = acc[i][j][e];
  __syncthreads();
  if constexpr (has_stats(EPI)) {
    // four threads a row, 16 columns each
    const uint32_t r = tid / 4, c0 = tid % 4 * 16;
    float top = -INFINITY;
    for (uint32_t c = c0; c < c0 + 16; ++c)
      if (n0 + c < p.n) top = fmaxf(top, tile[r][c]);
    top = reduce_max_xor<4>(top);
    // a row of -inf (or of NaN) alone: exponents against 0
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    for (uint32_t c = c0; c < c0 + 16; ++c)
      if (n0 + c < p.n) sum += expf(EPI == kEpiStats ? tile[r][c] - from : (tile[r][c] - from) * p.inverse);
    sum = reduce_sum_xor<4>(sum);
    if (m0 + r < p.m) {
      if (tid % 4 == 0) p.stats[(uint64_t)(m0 + r) * p.stat_tiles + blockIdx.y] = float2{top, sum};
      if constexpr (EPI == kEpiStats) {
        const uint32_t target = p.target[m0 + r];
        if (target >= n0 + c0 && target < n0 + c0 + 16 && target < p.n) p.target_logit[m0 + r] = tile[r][target - n0];
      }
    }
  } else {
    for (uint32_t i = tid; i < TS * TS; i += 256) {
      const uint32_t r = i / TS, c = i % TS, row = m0 + r, col = n0 + c;
      float v = tile[r][c];
      // (rows and columns past the last up to the tile's end are read as zeros
      // by the products with g)
      float g = 0.0f;
      if (row < p.m && col < p.n) {
        const uint32_t target = p.target[row], at = p.v0 + col;
        if (target < p.vocab) {
          if constexpr (EPI == kEpiGrad) g = p.mantissa[row] * (expf(v - p.lse[row]) - (target == at ? 1.0f : 0.0f));
          else g = p.mantissa[row] * at_most(expf(v * p.inverse - p.lse[row]), p.most[row]);
        }
      }
      static_cast<uint16_t*>(p.out)[(uint64_t)row * p.ldo + col] = (uint16_t)f32_to_bf16_bits(g);
    }
  }
}

// the largest upstream factor of the rows with a target, by one block; a NaN
// among them is one
__global__ __launch_bounds__(1024) void loss_factor_kernel(const float* up, const uint32_t* target, float* out,
                                                           uint32_t rows, uint32_t vocab) {
  __shared__ float tops[16];
  float top = 0.0f;
  bool nan = false;
  for (uint32_t i = threadIdx.x; i < rows; i += 1024)
    if (target[i] < vocab) {
      const float v = fabsf(up[i]);
      top = fmaxf(top, v);
      nan |= v != v;
    }
  top = reduce_max_xor<64>(top);
  if (__builtin_amdgcn_ballot_w64(nan)) top = __builtin_nanf("");
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w)
      if (!(top >= tops[w]) && top == top) top = tops[w];
    *out = top;
  }
}

// up = factor 2^e m: m of every row, and for dw's product 2^e x with zeros for
// the rows without a target, [rows up to a multiple of 64] (out null: without
// dw).  Where up / factor is not a normal number (0, NaN, or of no weight in dw)
// 2^e is that number and m is 1.
__global__ __launch_bounds__(256) void loss_live_rows_kernel(const uint16_t* x, const uint32_t* target,
                                                             const float* up, const float* factor, uint16_t* out,
                                                             float* mantissa, uint32_t* err, uint32_t rows,
                                                             uint32_t vocab, uint32_t hidden) {
  const uint32_t row = blockIdx.x;
  const uint32_t y = row < rows ? target[row] : kNoTarget;
  float power = 0.0f, m = 1.0f;
  if (y < vocab) {
    power = *factor != 0.0f ? up[row] / *factor : 0.0f;
    const uint32_t bits = __float_as_uint(power), exponent = bits & 0x7f800000u;
    if (exponent != 0 && exponent != 0x7f800000u) {
      m = __uint_as_float((bits & 0x807fffffu) | 0x3f800000u);
      power = __uint_as_float(exponent);
    }
  }
  if (threadIdx.x == 0) {
    if (row < rows) mantissa[row] = m;
    if (y >= vocab && y != kNoTarget) atomicOr(err, kErrTarget);
  }
  if (!out) return;
  for (uint32_t c = threadIdx.x * 8; c < hidden; c += 2048) {
    v4i v{0, 0, 0, 0};
    if (y < vocab) {
      v = *reinterpret_cast<const v4i*>(x + (uint64_t)row * hidden + c);
      if (power != 1.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t bits = (uint32_t)v[i];
          v[i] = (int)f32x2_to_bf16x2(power * bf16_bits_to_f32(bits & 0xffffu), power * bf16_bits_to_f32(bits >> 16));
        }
      }
    }
    *reinterpret_cast<v4i*>(out + (uint64_t)row * hidden + c) = v;
  }
}

// dx: bf16 of up / m times the fp32 sums, the splits' added in order
__global__ __launch_bounds__(256) void loss_round_kernel(const float* sums, const uint32_t* target, const float* up,
                                                         const float* mantissa, uint16_t* out, uint32_t hidden, uint32_t vocab,
                                                         uint64_t count, uint32_t splits) {
  for (uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += (uint64_t)gridDim.x * 1024) {
    const uint32_t row = (uint32_t)(i / hidden);
    const bool live = target[row] < vocab;
    const float f = live ? up[row] / mantissa[row] : 0.0f;
    v4f v = *reinterpret_cast<const v4f*>(sums + i);
#pragma unroll 8
    for (uint32_t s = 1; s < splits; ++s) v += *reinterpret_cast<const v4f*>(sums + s * count + i);
    // (a row without a target: 0, whatever the weights' infinities made of it)
    if (!live) v = v4f{0.f, 0.f, 0.f, 0.f};
    *reinterpret_cast<uint2*>(out + i) =
        uint2{f32x2_to_bf16x2(v[0] * f, v[1] * f), f32x2_to_bf16x2(v[2] * f, v[3] * f)};
  }
}

template <int EPI>
void launch_gemm(const GemmArgs& g, hipStream_t s) {
  hipLaunchKernelGGL((loss_gemm_kernel<EPI>), dim3((g.m + TS - 1) / TS, (g.n + TS - 1) / TS), dim3(256), 0, s,
                     g);
}

bool shape_ok(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  return rows && vocab && hidden && hidden % 8 == 0 && rows <= (1u << 20) && vocab <= (1u << 20) && hidden <= (1u << 20);
}
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

// Columns of a piece, in whole tiles: 2/3 to 4/3 of 2^26 elements of g (of 4096
// columns at least, or all columns), by the rounds of tiles that a piece's logits
// and weights' gradient take and 25 us of its own (three launches, and dx's sums
// read and written once more).  1021 rows over 151936 x 1024: two pieces, 990 us,
// three of 2^26 elements 1031; 4096 rows: pieces of whole rounds 3476 us, nine
// even ones 4284.
uint32_t piece_columns(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  const uint32_t all = (vocab + TB - 1) / TB, tall = (rows + 255) / 256, wide = (hidden + TB - 1) / TB;
  const uint32_t fit = (uint32_t)std::max<uint64_t>((1ull << 26) / rows, 4096) / TB;
  const uint32_t most = std::max(1u, fit + fit / 3);
  if (all <= most) return all * TB;
  auto time = [&](uint64_t tiles, uint32_t k) {
    return (float)((tiles + kCus - 1) / kCus) * (9.0f + 1.45f * (float)k / KB);
  };
  auto piece = [&](uint64_t c) { return c ? time(tall * c, hidden) + time(wide * c, rows) + 25.0f : 0.0f; };
  uint32_t best = most;
  float least = INFINITY;
  for (uint32_t c = most; c >= std::max(1u, fit - fit / 3); --c) {
    const float cost = (float)(all / c) * piece(c) + piece(all % c);
    if (cost < least) {
      least = cost;
      best = c;
    }
  }
  return best * TB;
}

// the tiles fed by DMA take 64-deep steps
bool big_takes(uint32_t hidden) { return hidden % KB == 0; }
// a row's pairs of the forward pass: one per column tile
uint32_t stat_tiles(uint32_t vocab, uint32_t hidden) {
  const uint32_t columns = big_takes(hidden) ? TB : TS;
  return (vocab + columns - 1) / columns;
}

struct BackwardPlan {
  uint32_t piece, splits;
  uint64_t g, live, sums, factor, mantissa, bytes;
};
BackwardPlan backward_plan(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  BackwardPlan p{};
  p.piece = piece_columns(rows, vocab, hidden);
  const uint64_t row_up = (rows + 63) / 64 * 64;
  p.g = 0;
  p.live = p.g + padded(row_up * p.piece * 2);
  p.sums = p.live + padded(row_up * hidden * 2);
  // dx has few tiles: its contraction, a piece's columns, is split until
  // there is a tile for every CU, at 1024 columns a split or more
  const uint32_t tiles = ((rows + TB - 1) / TB) * ((hidden + TB - 1) / TB);
  p.splits = std::max<uint32_t>(1, std::min<uint32_t>(kCus / tiles, p.piece / 1024));
  p.factor = p.sums + padded((uint64_t)p.splits * rows * hidden * 4);
  p.mantissa = p.factor + padded(4);
  p.bytes = p.mantissa + padded((uint64_t)rows * 4);
  return p;
}

// The launches of a backward pass.  target: kNoTarget (or past the vocabulary)
// for the rows whose g is 0; up: their upstream factors.
struct BackwardCall {
  const uint16_t* x;
  const uint16_t* w;
  const uint32_t* target;
  const float* lse;
  const float* up;
  uint16_t* dx;
  uint16_t* dw;
  uint32_t* error_flag;
  hipStream_t stream;
  uint32_t rows, vocab, hidden;
  float temperature = 1.0f;  // kEpiTeacherGrad
  const float* most = nullptr;  // the same: what a row's exponentials sum to
};

// dx of a piece on a route of its own: the rows in whole tiles of 256 and the
// rest each with the splits that suit them, whose sums lie behind one another
struct DxRoute {
  Tiling whole, rest;
  uint32_t whole_rows;
  uint64_t sums;  // fp32 elements
};
DxRoute dx_route(uint32_t rows, uint32_t hidden, uint32_t columns) {
  const Tiling all = tiling_of(rows, hidden, columns);
  DxRoute r{all, {}, rows, (uint64_t)all.splits * rows * hidden};
  const uint32_t whole = rows / 256 * 256;
  if (whole && whole < rows) {
    const Tiling first = tiling_of(whole, hidden, columns), last = tiling_of(rows - whole, hidden, columns);
    if (first.us + last.us + 3.0f < all.us)
      r = {first, last, whole, ((uint64_t)first.splits * whole + (uint64_t)last.splits * (rows - whole)) * hidden};
  }
  return r;
}
inline void launch_dx(const Tiling& t, BigArgs b, hipStream_t s) {
  b.splits = t.splits;
  b.split_stride = (uint64_t)b.m * b.n;
  if (t.rows == 64) launch_rows<64, false, true, kEpiAdd>(b, s);
  else if (t.rows == 128) launch_rows<128, false, true, kEpiAdd>(b, s);
  else launch_rows<256, false, true, kEpiAdd>(b, s);
}

// after_logits(v0, cols): enqueues what g of a piece still needs.  route: dx's
// (null: all rows alike, in plan.splits parts).  The cross entropy keeps the even
// parts: neither way is the faster one everywhere, and the estimate does not tell
// where.  Its gradients of dx, us, even -> routed: 2053 rows over 129280 x 4096 4305 ->
// 3525, 4096 over 151936 x 2560 5700 -> 5300, but 1 row there 279 -> 325, 257 748 -> 810,
// 33 298 -> 349, 512 over 32768 x 2048 148 -> 162; 800 and 1021 rows within 2 %.
template <int EPI, typename F>
void launch_backward(const BackwardCall& a, const BackwardPlan& plan, const DxRoute* route, uint8_t* ws,
                     F&& after_logits) {
  uint16_t* const grad = reinterpret_cast<uint16_t*>(ws + plan.g);
  uint16_t* const live = reinterpret_cast<uint16_t*>(ws + plan.live);
  float* const sums = reinterpret_cast<float*>(ws + plan.sums);
  const uint32_t row_up = (a.rows + 63) / 64 * 64;
  float* const factor = reinterpret_cast<float*>(ws + plan.factor);
  float* const mantissa = reinterpret_cast<float*>(ws + plan.mantissa);
  hipLaunchKernelGGL(loss_factor_kernel, dim3(1), dim3(1024), 0, a.stream, a.up, a.target, factor, a.rows, a.vocab);
  hipLaunchKernelGGL(loss_live_rows_kernel, dim3(row_up), dim3(256), 0, a.stream, a.x, a.target, a.up, factor,
                     a.dw ? live : nullptr, mantissa, a.error_flag, a.rows, a.vocab, a.hidden);
  for (uint32_t v0 = 0; v0 < a.vocab; v0 += plan.piece) {
    const uint32_t cols = std::min(plan.piece, a.vocab - v0);
    const uint16_t* const w = a.w + (uint64_t)v0 * a.hidden;
    if (big_takes(a.hidden)) {
      BigArgs b{};
      b.a = a.x;
      b.b = w;
      b.m = a.rows;
      b.n = cols;
      b.k = a.hidden;
      b.lda = b.ldb = a.hidden;
      b.out = grad;
      b.ldo = plan.piece;
      b.target = a.target;
      b.lse = a.lse;
      b.mantissa = mantissa;
      b.v0 = v0;
      b.vocab = a.vocab;
      b.exponent = kLog2e / a.temperature;
      b.most = a.most;
      launch_big<false, false, EPI>(b, a.stream);
    } else {
      GemmArgs g{};
      g.a = a.x;
      g.b = w;
      g.m = a.rows;
      g.n = cols;
      g.k = a.hidden;
      g.lda = g.ldb = a.hidden;
      g.out = grad;
      g.ldo = plan.piece;
      g.target = a.target;
      g.lse = a.lse;
      g.mantissa = mantissa;
      g.v0 = v0;
      g.vocab = a.vocab;
      g.inverse = 1.0f / a.temperature;
      g.most = a.most;
      launch_gemm<has_teacher_grad(EPI) ? kEpiTeacherGrad : EPI>(g, a.stream);
    }
    after_logits(v0, cols);
    if (a.dw) {
      BigArgs b{};
      b.a = grad;
      b.b = live;
      b.m = cols;
      b.n = a.hidden;
      b.k = b.k_valid = row_up;
      b.lda = plan.piece;
      b.ldb = a.hidden;
      b.out = a.dw + (uint64_t)v0 * a.hidden;
      b.scale = factor;
      b.ldo = a.hidden;
      launch_big<true, true, kEpiBf16>(b, a.stream);
    }
    BigArgs b{};
    b.a = grad;
    b.b = w;
    b.m = a.rows;
    b.n = a.hidden;
    b.k = (cols + KB - 1) / KB * KB;
    b.k_valid = cols;
    b.lda = plan.piece;
    b.ldb = a.hidden;
    b.out = sums;
    b.ldo = a.hidden;
    b.first = v0 == 0;
    if (route) {
      b.m = route->whole_rows;
      launch_dx(route->whole, b, a.stream);
      if (route->whole_rows < a.rows) {
        b.m = a.rows - route->whole_rows;
        b.a += (uint64_t)route->whole_rows * plan.piece;
        b.out = sums + (uint64_t)route->whole.splits * route->whole_rows * a.hidden;
        launch_dx(route->rest, b, a.stream);
      }
    } else {
      b.splits = plan.splits;
      b.split_stride = (uint64_t)a.rows * a.hidden;
      launch_big<false, true, kEpiAdd>(b, a.stream);
    }
  }
  auto round = [&](const float* from, uint32_t first, uint32_t rows, uint32_t splits) {
    const uint64_t count = (uint64_t)rows * a.hidden;
    hipLaunchKernelGGL(loss_round_kernel, dim3((uint32_t)std::min<uint64_t>((count + 1023) / 1024, 1u << 20)), dim3(256),
                       0, a.stream, from, a.target + first, a.up + first, mantissa + first,
                       a.dx + (uint64_t)first * a.hidden, a.hidden, a.vocab, count, splits);
  };
  if (!route) {
    round(sums, 0, a.rows, plan.splits);
  } else {
    round(sums, 0, route->whole_rows, route->whole.splits);
    if (route->whole_rows < a.rows)
      round(sums + (uint64_t)route->whole.splits * route->whole_rows * a.hidden, route->whole_rows,
            a.rows - route->whole_rows, route->rest.splits);
  }
}

}  // namespace
}  // namespace pih_amd
