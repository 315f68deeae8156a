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
// (128 MB or so, so that it stays in the memory-side cache between its writer and
// its two readers; 4096 columns or so, which is more, above 16384 rows), then dw of the piece is g^T x, and dx
// grows by g W_piece in fp32.
//
// g is rounded to bf16 for the matrix cores, which costs half the MFMAs of two
// parts: 2^-8 of each element at most, independent from element to element, in
// sums that are rounded to bf16 once themselves (4096 rows over 129280 x 4096:
// dx and dw 0.20 % of their norm off 64 bits, 0.17 % of it their own rounding).
// Of the upstream factors up_t = s 2^e m, with s the largest and
// 1 <= |m| < 2, g holds m alone; 2^e goes into the x of dw's product, exactly,
// s into dw in fp32, and up_t / m into dx in fp32.  So a mean's equal factors
// (1 / rows, whose rounding would be the same error in every element) are
// exact (all of up_t rounded inside g: 0.34 %).
//
// Measured: 4096 rows, 129280 x 4096 2.95-3.04 ms (1.45 PFLOP/s; a library
// product of that shape alone 3.25 ms) and 9.3-9.5 ms for the gradients, bound
// by the matrix pipe, 70 % busy, and the power it takes (1.9 GHz); 33 rows, 151936
// x 1024 64.4 us, of which the weights' 311 MB take 61 at 5.1 TB/s; the gradients
// of 1021 rows there 0.93 ms (1.02 PFLOP/s: of a 256 x 256 tile's 31 us 9 are the
// exponentials and the stores).  dx alone, for a frozen head: 33 rows 136 us over
// 151936 x 1024 and 374 over 129280 x 4096 (the weights twice from HBM), 4096 rows
// 6.2 ms over 129280 x 4096 (1.41 PFLOP/s).
//
// Rows without a target take no part in the gradients: their g is 0, and the
// x of dw's product is a copy with those rows as zeros, so that nothing an
// unused row holds (infinities, NaN) reaches dw.
#include "lm_head_common.hpp"

namespace pih_amd {
namespace {

// A row's pairs joined, by a wave: lse = M + log(sum of s exp(m - M)).  33 rows
// of 594 pairs 4.5 us, 4096 rows of 505 9 us.
__global__ __launch_bounds__(256) void loss_join_kernel(const float2* stats, const float* target_logit,
                                                        const uint32_t* target, float* loss, float* lse, uint32_t* err,
                                                        uint32_t rows, uint32_t vocab, uint32_t tiles) {
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  const float2* s = stats + (uint64_t)row * tiles;
  float top = -INFINITY, sum = 0.0f;
#pragma unroll 8
  for (uint32_t i = lane; i < tiles; i += 64) top = fmaxf(top, s[i].x);
  top = reduce_max_xor<64>(top);
  // (a tile of -inf or NaN alone has the sum 0 or NaN, whatever the factor)
#pragma unroll 8
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

}  // namespace

uint64_t LmHeadLossWorkspaceBytes(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  if (!shape_ok(rows, vocab, hidden)) return 0;
  return padded((uint64_t)rows * stat_tiles(vocab, hidden) * 8) + padded((uint64_t)rows * 4);
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
  g.stat_tiles = stat_tiles(a.vocab, a.hidden);
  g.stats = static_cast<float2*>(a.workspace);
  g.target_logit = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) +
                                            padded((uint64_t)a.rows * g.stat_tiles * 8));
  if (big_takes(a.hidden)) {
    BigArgs b{};
    b.a = a.x;
    b.b = a.w;
    b.m = a.rows;
    b.n = b.vocab = a.vocab;
    b.k = a.hidden;
    b.lda = b.ldb = a.hidden;
    b.target = a.target;
    b.stats = g.stats;
    b.target_logit = g.target_logit;
    launch_big<false, false, kEpiStats>(b, a.stream);
  } else {
    launch_gemm<kEpiStats>(g, a.stream);
  }
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
  // (the weights' gradient of a piece is written before dx reads its weights)
  if (a.dw == a.w) return Invalid("lm_head_loss_backward_alias_invalid");
  const BackwardPlan plan = backward_plan(a.rows, a.vocab, a.hidden);
  if (a.workspace_bytes < plan.bytes || !aligned(a.workspace, 16))
    return Invalid("lm_head_loss_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  BackwardCall call{};
  call.x = a.x;
  call.w = a.w;
  call.target = a.target;
  call.lse = a.lse;
  call.up = a.loss_grad;
  call.dx = a.dx;
  call.dw = a.dw;
  call.error_flag = a.error_flag;
  call.stream = a.stream;
  call.rows = a.rows;
  call.vocab = a.vocab;
  call.hidden = a.hidden;
  launch_backward<kEpiGrad>(call, plan, nullptr, static_cast<uint8_t*>(a.workspace), [](uint32_t, uint32_t) {});
  return AfterLaunch("lm_head_loss_backward_launch_failed");
}

}  // namespace pih_amd
