// Softmax cross entropy of an LM head and its gradients for gfx950, without
// the logits in memory:
//   lse_t = log sum_v exp(x_t . w_v),  loss_t = lse_t - x_t . w_target,
//   g_tv  = up_t (exp(x_t . w_v - lse_t) - [v == target_t]),
//   dx = g W,  dw = g^T x.
//
// Forward: one GEMM whose tiles leave, in place of logits, the maximum m and
// the sum of exp(l - m) of every row over their columns, 8 bytes per row and
// tile, and the target's logit where they hold it; a second launch joins a
// row's pairs.  Backward: pieces of the vocabulary.  For a piece the logits
// are computed again and leave as g, bf16 [rows][piece] in the workspace
// (128 MB at most, so that it stays in the memory-side cache between its
// writer and its two readers), then dw of the piece is g^T x, and dx grows by
// g W_piece in fp32.  g is rounded to bf16 for the matrix cores: 2^-9 of each
// element at most, independent over the sums of rows or vocabulary that the
// results are, which are themselves rounded to bf16 once.
//
// Rows without a target take no part in the gradients: their g is 0, and the
// x of dw's product is a copy with those rows as zeros, so that nothing an
// unused row holds (infinities, NaN) reaches dw.
#include <algorithm>

#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kNoTarget = 0xffffffffu;
constexpr uint32_t kErrTarget = 1u, kErrLoss = 4u;
constexpr uint32_t TS = 64, KS = 64, kPitch = KS + 8;

typedef uint16_t Tile16[TS][kPitch];

enum : int { kEpiStats = 0, kEpiGrad = 1, kEpiBf16 = 2, kEpiAdd = 3 };

// C [m][n] = A . B^T over k.  A: [m][k] with row stride lda, or (AT) [k][m];
// B: [n][k], or (BT) [k][n].
struct GemmArgs {
  const uint16_t* a;
  const uint16_t* b;
  uint32_t m, n, k;
  uint64_t lda, ldb;
  void* out;            // kEpiBf16: bf16, kEpiAdd: f32, kEpiGrad: bf16
  uint64_t ldo;
  // kEpiStats, kEpiGrad: rows of the result are x rows, columns vocabulary
  // entries from v0 on
  const uint32_t* target;
  const float* lse;
  const float* up;
  float2* stats;        // [m][stat_tiles]
  float* target_logit;  // [m]
  uint32_t v0, vocab, stat_tiles, first;
};

// 64 x 64 elements of an operand into LDS as [row][k], zeros outside
template <bool kT>
__device__ __forceinline__ void stage(Tile16& s, const uint16_t* p, uint64_t ld, uint32_t r0, uint32_t rows, uint32_t k0,
                                      uint32_t k) {
  for (uint32_t i = threadIdx.x; i < TS * KS / 8; i += 256) {
    const uint32_t r = i / 8, c = i % 8 * 8;
    v4i v{0, 0, 0, 0};
    if constexpr (kT) {
      // source row k0 + r, columns r0 + c ..
      if (k0 + r < k && r0 + c < rows) {
        const uint16_t* src = p + (uint64_t)(k0 + r) * ld + r0 + c;
        if (r0 + c + 8 <= rows) {
          v = *reinterpret_cast<const v4i*>(src);
        } else {
          for (uint32_t q = 0; q < rows - r0 - c; ++q) v[q / 2] |= (int)((uint32_t)src[q] << (16 * (q & 1)));
        }
      }
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q) s[c + q][r] = (uint16_t)((uint32_t)v[q / 2] >> (16 * (q & 1)));
    } else {
      if (r0 + r < rows && k0 + c < k) v = *reinterpret_cast<const v4i*>(p + (uint64_t)(r0 + r) * ld + k0 + c);
      *reinterpret_cast<v4i*>(&s[r][c]) = v;
    }
  }
}

// Tile of 64 x 64: four waves of 32 x 32.  The MFMA's first operand is B, so
// that a lane's four results are consecutive columns of one row.
template <bool AT, bool BT, int EPI>
__global__ __launch_bounds__(256) void loss_gemm_kernel(GemmArgs p) {
  __shared__ __align__(16) Tile16 sa, sb;
  __shared__ float tile[TS][TS + 1];
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const uint32_t m0 = blockIdx.x * TS, n0 = blockIdx.y * TS, wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  v4f acc[2][2];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i / 2][i % 2] = v4f{0.f, 0.f, 0.f, 0.f};
  for (uint32_t k0 = 0; k0 < p.k; k0 += KS) {
    stage<AT>(sa, p.a, p.lda, m0, p.m, k0, p.k);
    stage<BT>(sb, p.b, p.ldb, n0, p.n, k0, p.k);
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
  if constexpr (EPI == kEpiStats) {
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
      if (n0 + c < p.n) sum += expf(tile[r][c] - from);
    sum = reduce_sum_xor<4>(sum);
    if (m0 + r < p.m) {
      const uint32_t target = p.target[m0 + r];
      if (tid % 4 == 0) p.stats[(uint64_t)(m0 + r) * p.stat_tiles + blockIdx.y] = float2{top, sum};
      if (target >= n0 + c0 && target < n0 + c0 + 16 && target < p.n) p.target_logit[m0 + r] = tile[r][target - n0];
    }
  } else {
    for (uint32_t i = tid; i < TS * TS; i += 256) {
      const uint32_t r = i / TS, c = i % TS, row = m0 + r, col = n0 + c;
      float v = tile[r][c];
      if constexpr (EPI == kEpiGrad) {
        if (row >= p.m) continue;
        const uint32_t target = p.target[row], at = p.v0 + col;
        float g = 0.0f;
        if (target < p.vocab && col < p.n) g = p.up[row] * (expf(v - p.lse[row]) - (target == at ? 1.0f : 0.0f));
        static_cast<uint16_t*>(p.out)[(uint64_t)row * p.ldo + col] = (uint16_t)f32_to_bf16_bits(g);
      } else if (row < p.m && col < p.n) {
        const uint64_t o = (uint64_t)row * p.ldo + col;
        if constexpr (EPI == kEpiBf16) static_cast<uint16_t*>(p.out)[o] = (uint16_t)f32_to_bf16_bits(v);
        else static_cast<float*>(p.out)[o] = p.first ? v : static_cast<float*>(p.out)[o] + v;
      }
    }
  }
}

// A row's pairs joined, by a wave: lse = M + log(sum of s exp(m - M))
__global__ __launch_bounds__(256) void loss_join_kernel(const float2* stats, const float* target_logit,
                                                        const uint32_t* target, float* loss, float* lse, uint32_t* err,
                                                        uint32_t rows, uint32_t vocab, uint32_t tiles) {
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const float2* s = stats + (uint64_t)row * tiles;
  float top = -INFINITY, sum = 0.0f;
  for (uint32_t i = lane; i < tiles; i += 64) top = fmaxf(top, s[i].x);
  top = reduce_max_xor<64>(top);
  // (a tile of -inf or NaN alone has the sum 0 or NaN, whatever the factor)
  for (uint32_t i = lane; i < tiles; i += 64) sum += s[i].x == -INFINITY ? s[i].y : s[i].y * expf(s[i].x - top);
  sum = reduce_sum_xor<64>(sum);
  if (lane) return;
  const float l = top + logf(sum);
  const uint32_t y = target[row];
  float out = 0.0f;
  uint32_t bad = 0;
  if (y < vocab) {
    out = l - target_logit[row];
    if (!__builtin_isfinite(out)) bad = kErrLoss;
  } else if (y != kNoTarget) {
    bad = kErrTarget;
  }
  lse[row] = l;
  loss[row] = out;
  if (bad) atomicOr(err, bad);
}

// x with zeros for the rows without a target, [rows up to a multiple of 64]
__global__ __launch_bounds__(256) void loss_live_rows_kernel(const uint16_t* x, const uint32_t* target, uint16_t* out,
                                                             uint32_t* err, uint32_t rows, uint32_t vocab,
                                                             uint32_t hidden) {
  const uint32_t row = blockIdx.x;
  const uint32_t y = row < rows ? target[row] : kNoTarget;
  if (threadIdx.x == 0 && y >= vocab && y != kNoTarget) atomicOr(err, kErrTarget);
  for (uint32_t c = threadIdx.x * 8; c < hidden; c += 2048) {
    v4i v{0, 0, 0, 0};
    if (y < vocab) v = *reinterpret_cast<const v4i*>(x + (uint64_t)row * hidden + c);
    *reinterpret_cast<v4i*>(out + (uint64_t)row * hidden + c) = v;
  }
}

// dx: bf16 of the fp32 sums
__global__ __launch_bounds__(256) void loss_round_kernel(const float* sums, uint16_t* out, uint64_t count) {
  const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  const v4f v = *reinterpret_cast<const v4f*>(sums + i);
  *reinterpret_cast<uint2*>(out + i) = uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
}

template <bool AT, bool BT, int EPI>
void launch_gemm(const GemmArgs& g, hipStream_t s) {
  hipLaunchKernelGGL((loss_gemm_kernel<AT, BT, EPI>), dim3((g.m + TS - 1) / TS, (g.n + TS - 1) / TS), dim3(256), 0, s,
                     g);
}

bool shape_ok(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  return rows && vocab && hidden && hidden % 8 == 0 && rows <= (1u << 20) && vocab <= (1u << 20) && hidden <= (1u << 20);
}
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }

// columns of a piece: 2^26 elements of g, in whole tiles
uint32_t piece_columns(uint32_t rows, uint32_t vocab) {
  const uint32_t all = (vocab + 255) / 256 * 256;
  const uint32_t fit = (uint32_t)std::min<uint64_t>((1ull << 26) / rows / 256 * 256, 32768);
  return std::min(all, std::max(fit, 4096u));
}

struct BackwardPlan {
  uint32_t piece;
  uint64_t g, live, sums, bytes;
};
BackwardPlan backward_plan(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  BackwardPlan p{};
  p.piece = piece_columns(rows, vocab);
  const uint64_t row_up = (rows + 63) / 64 * 64;
  p.g = 0;
  p.live = p.g + padded(row_up * p.piece * 2);
  p.sums = p.live + padded(row_up * hidden * 2);
  p.bytes = p.sums + padded((uint64_t)rows * hidden * 4);
  return p;
}

}  // namespace

uint64_t LmHeadLossWorkspaceBytes(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  if (!shape_ok(rows, vocab, hidden)) return 0;
  return padded((uint64_t)rows * ((vocab + TS - 1) / TS) * 8) + padded((uint64_t)rows * 4);
}

uint64_t LmHeadLossBackwardWorkspaceBytes(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  return shape_ok(rows, vocab, hidden) ? backward_plan(rows, vocab, hidden).bytes : 0;
}

St LaunchLmHeadLoss(const LmHeadLossArgs& a) {
  if (!a.x || !a.w || !a.target || !a.loss || !a.lse || !a.workspace || !a.error_flag || !a.stream)
    return Invalid("lm_head_loss_null_argument");
  if (!shape_ok(a.rows, a.vocab, a.hidden)) return Invalid("lm_head_loss_shape_invalid");
  if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.target, 4) || !aligned(a.loss, 4) || !aligned(a.lse, 4) ||
      !aligned(a.error_flag, 4))
    return Invalid("lm_head_loss_alignment_invalid");
  if (a.workspace_bytes < LmHeadLossWorkspaceBytes(a.rows, a.vocab, a.hidden) || !aligned(a.workspace, 16))
    return Invalid("lm_head_loss_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  GemmArgs g{};
  g.a = a.x;
  g.b = a.w;
  g.m = a.rows;
  g.n = g.vocab = a.vocab;
  g.k = a.hidden;
  g.lda = g.ldb = a.hidden;
  g.target = a.target;
  g.stat_tiles = (a.vocab + TS - 1) / TS;
  g.stats = static_cast<float2*>(a.workspace);
  g.target_logit = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) +
                                            padded((uint64_t)a.rows * g.stat_tiles * 8));
  launch_gemm<false, false, kEpiStats>(g, a.stream);
  hipLaunchKernelGGL(loss_join_kernel, dim3((a.rows + 3) / 4), dim3(256), 0, a.stream, g.stats, g.target_logit,
                     a.target, a.loss, a.lse, a.error_flag, a.rows, a.vocab, g.stat_tiles);
  return AfterLaunch("lm_head_loss_launch_failed");
}

St LaunchLmHeadLossBackward(const LmHeadLossArgs& a) {
  if (!a.x || !a.w || !a.target || !a.lse || !a.loss_grad || !a.dx || !a.workspace || !a.error_flag || !a.stream)
    return Invalid("lm_head_loss_backward_null_argument");
  if (!shape_ok(a.rows, a.vocab, a.hidden)) return Invalid("lm_head_loss_backward_shape_invalid");
  if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.dx, 16) || !aligned(a.dw, 16) || !aligned(a.target, 4) ||
      !aligned(a.lse, 4) || !aligned(a.loss_grad, 4) || !aligned(a.error_flag, 4))
    return Invalid("lm_head_loss_backward_alignment_invalid");
  const BackwardPlan plan = backward_plan(a.rows, a.vocab, a.hidden);
  if (a.workspace_bytes < plan.bytes || !aligned(a.workspace, 16))
    return Invalid("lm_head_loss_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  uint16_t* const grad = reinterpret_cast<uint16_t*>(ws + plan.g);
  uint16_t* const live = reinterpret_cast<uint16_t*>(ws + plan.live);
  float* const sums = reinterpret_cast<float*>(ws + plan.sums);
  const uint32_t row_up = (a.rows + 63) / 64 * 64;
  hipLaunchKernelGGL(loss_live_rows_kernel, dim3(row_up), dim3(256), 0, a.stream, a.x, a.target, live, a.error_flag,
                     a.rows, a.vocab, a.hidden);
  for (uint32_t v0 = 0; v0 < a.vocab; v0 += plan.piece) {
    const uint32_t cols = std::min(plan.piece, a.vocab - v0);
    const uint16_t* const w = a.w + (uint64_t)v0 * a.hidden;
    GemmArgs g{};
    g.a = live;
    g.b = w;
    g.m = a.rows;
    g.n = cols;
    g.k = a.hidden;
    g.lda = g.ldb = a.hidden;
    g.out = grad;
    g.ldo = plan.piece;
    g.target = a.target;
    g.lse = a.lse;
    g.up = a.loss_grad;
    g.v0 = v0;
    g.vocab = a.vocab;
    launch_gemm<false, false, kEpiGrad>(g, a.stream);
    if (a.dw) {
      GemmArgs d{};
      d.a = grad;
      d.b = live;
      d.m = cols;
      d.n = a.hidden;
      d.k = a.rows;
      d.lda = plan.piece;
      d.ldb = a.hidden;
      d.out = a.dw + (uint64_t)v0 * a.hidden;
      d.ldo = a.hidden;
      launch_gemm<true, true, kEpiBf16>(d, a.stream);
    }
    GemmArgs d{};
    d.a = grad;
    d.b = w;
    d.m = a.rows;
    d.n = a.hidden;
    d.k = cols;
    d.lda = plan.piece;
    d.ldb = a.hidden;
    d.out = sums;
    d.ldo = a.hidden;
    d.first = v0 == 0;
    launch_gemm<false, true, kEpiAdd>(d, a.stream);
  }
  const uint64_t count = (uint64_t)a.rows * a.hidden;
  hipLaunchKernelGGL(loss_round_kernel, dim3((uint32_t)((count / 4 + 255) / 256)), dim3(256), 0, a.stream, sums, a.dx,
                     count);
  return AfterLaunch("lm_head_loss_backward_launch_failed");
}

}  // namespace pih_amd
