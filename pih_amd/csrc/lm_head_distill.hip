// Divergence of an LM head from a teacher's top logits and its gradients for
// gfx950, without the head's own logits in memory.  With z_tv = x_t . w_v, the
// temperature T and a row's teacher entries k of id i_k and probability q_k:
//   lse_t = log sum_v exp(z_tv / T),
//   loss_t = T^2 sum_k q_k (log q_k - z_{t i_k} / T + lse_t),
//   g_tv = up_t T (Q_t exp(z_tv / T - lse_t) - sum of q_k over i_k = v),
//   dx = g W,  dw = g^T x,  Q_t = sum_k q_k.
//
// Measured: 33 rows over 151936 x 1024, 20 entries, 65 us (the weights' 311 MB in 59,
// 5.3 TB/s), 4096 rows over 129280 x 4096, 64 entries, 3.09-3.16 ms (1.38 PFLOP/s: the
// matrix pipe at the clock that power leaves); gradients of 1021 rows over 151936 x 1024
// 0.95-0.97 ms (0.99 PFLOP/s: of a tile's 31 us 9 are exponentials and stores), of 2053
// over 129280 x 4096 5.26-5.40 ms (1.22 PFLOP/s), of 33 over 151936 x 1024 228 us.
//
// The products are those of the cross entropy (lm_head_loss.hip) without a
// target.  The teacher's entries are few against the vocabulary: forward their
// logits are dot products of their own, or where that is much (listed()) every row's
// entries come in order, with how many lie before each tile, and the tile that
// has an entry's logit writes it out; backward the elements of g at them, which
// the tiles have written without their q, are written once more.
#include "lm_head_common.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kTopMax = 256;

// Teacher entries of a row, by a wave: lane l holds entries l, l + 64, ..
struct Entries {
  uint32_t id[kTopMax / 64];  // kNoTarget: none
  float s[kTopMax / 64];      // logit over the temperature, -inf: none
};
__device__ __forceinline__ bool load_entries(Entries& e, const uint32_t* ids, const float* teacher, uint64_t at,
                                             uint32_t top_k, uint32_t vocab, float inverse) {
  const uint32_t lane = threadIdx.x & 63;
  bool bad = false;
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    const uint32_t k = lane + 64 * i;
    e.id[i] = k < top_k ? ids[at + k] : kNoTarget;
    bad |= e.id[i] >= vocab && e.id[i] != kNoTarget;
    if (e.id[i] >= vocab) e.id[i] = kNoTarget;
    e.s[i] = e.id[i] != kNoTarget ? teacher[at + k] * inverse : -INFINITY;
  }
  return bad;
}
// log of what exp(s) is divided by, of a row; -inf where no entry has a
// probability (its q are then 0 by probability())
__device__ __forceinline__ float normalizer(const Entries& e, const float* teacher_lse, uint32_t row) {
  if (teacher_lse) return teacher_lse[row];
  float top = -INFINITY, sum = 0.0f;
  bool nan = false;
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    top = fmaxf(top, e.s[i]);
    nan |= e.s[i] != e.s[i];
  }
  top = reduce_max_xor<64>(top);
  if (__builtin_amdgcn_ballot_w64(nan)) return __builtin_nanf("");
  if (top == -INFINITY) return top;
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) sum += expf(e.s[i] - top);
  return top + logf(reduce_sum_xor<64>(sum));
}
__device__ __forceinline__ float probability(float s, float normalizer) {
  return s == -INFINITY ? 0.0f : expf(s - normalizer);
}

// The entries of a row in order of their ids, by a wave (an entry's place is how
// many are less; no two are equal), how many lie before each tile of the
// vocabulary, and 0 for the logits of those that are not there
__global__ __launch_bounds__(256) void distill_sort_kernel(const uint32_t* ids, uint32_t* sorted, uint16_t* before,
                                                           float* logits, uint32_t rows, uint32_t vocab, uint32_t tiles,
                                                           uint32_t top_k) {
  __shared__ uint32_t all[4][kTopMax], ordered[4][kTopMax];
  const uint32_t wave = threadIdx.x >> 6, row = blockIdx.x * 4 + wave, lane = threadIdx.x & 63;
  if (row >= rows) return;
  const uint64_t at = (uint64_t)row * top_k;
  uint32_t key[kTopMax / 64], there = 0;
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    const uint32_t k = lane + 64 * i, id = k < top_k ? ids[at + k] : kNoTarget;
    // (those that are not there last, in order of their places too)
    key[i] = (id < vocab ? id << 8 : 1u << 28) | k;
    there += __popcll(__builtin_amdgcn_ballot_w64(id < vocab));
    if (k < top_k) {
      all[wave][k] = key[i];
      if (id >= vocab) logits[at + k] = 0.0f;
    }
  }
  wave_lds_order();
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    if (64 * i >= top_k) break;
    uint32_t less = 0;
    for (uint32_t k = 0; k < top_k; ++k) less += all[wave][k] < key[i];
    if (lane + 64 * i < top_k) {
      ordered[wave][less] = key[i];
      sorted[at + less] = key[i];
    }
  }
  wave_lds_order();
  uint16_t* const out = before + (uint64_t)row * (tiles + 1);
  for (uint32_t t = lane; t <= tiles; t += 64) {
    uint32_t low = 0, high = there;
    while (low < high) {
      const uint32_t mid = (low + high) / 2;
      if (ordered[wave][mid] >> 8 < t * TB) low = mid + 1;
      else high = mid;
    }
    out[t] = (uint16_t)low;
  }
}

// z of an entry, by a wave: a dot product over the hidden size; 0 for none
__device__ __forceinline__ float entry_logit(const uint16_t* a, const uint16_t* w, uint32_t id, uint32_t vocab,
                                             uint32_t hidden) {
  if (id >= vocab) return 0.0f;
  const uint16_t* const b = w + (uint64_t)id * hidden;
  float sum = 0.0f;
  for (uint32_t c = (threadIdx.x & 63) * 8; c < hidden; c += 512) {
    const v4i u = *reinterpret_cast<const v4i*>(a + c), v = *reinterpret_cast<const v4i*>(b + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t p = (uint32_t)u[i], q = (uint32_t)v[i];
      sum = __builtin_fmaf(bf16_bits_to_f32(p & 0xffffu), bf16_bits_to_f32(q & 0xffffu), sum);
      sum = __builtin_fmaf(bf16_bits_to_f32(p >> 16), bf16_bits_to_f32(q >> 16), sum);
    }
  }
  return reduce_sum_xor<64>(sum);
}

__global__ __launch_bounds__(256) void distill_gather_kernel(const uint16_t* x, const uint16_t* w, const uint32_t* ids,
                                                             float* logits, uint64_t entries, uint32_t top_k,
                                                             uint32_t vocab, uint32_t hidden) {
  for (uint64_t at = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6); at < entries; at += (uint64_t)gridDim.x * 4) {
    const float v = entry_logit(x + at / top_k * hidden, w, ids[at], vocab, hidden);
    if ((threadIdx.x & 63) == 0) logits[at] = v;
  }
}

// A row's pairs joined to its log-sum-exp, by a wave
__device__ __forceinline__ float joined(const float2* s, uint32_t tiles, float inverse) {
  const uint32_t lane = threadIdx.x & 63;
  float top = -INFINITY, sum = 0.0f;
#pragma unroll 8
  for (uint32_t i = lane; i < tiles; i += 64) top = fmaxf(top, s[i].x);
  top = reduce_max_xor<64>(top);
  // (a tile of -inf or NaN alone has the sum 0 or NaN, whatever the factor)
#pragma unroll 8
  for (uint32_t i = lane; i < tiles; i += 64) sum += s[i].x == -INFINITY ? s[i].y : s[i].y * expf((s[i].x - top) * inverse);
  return top * inverse + logf(reduce_sum_xor<64>(sum));
}
// A row's loss, by a wave; z: its entries' logits
__device__ __forceinline__ void row_loss(const Entries& e, bool bad, const float* teacher_lse, const float* z, float l,
                                         float* loss, float* lse, uint32_t* err, uint32_t row, float temperature) {
  const uint32_t lane = threadIdx.x & 63;
  const float inverse = 1.0f / temperature, norm = normalizer(e, teacher_lse, row);
  float total = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    const float q = probability(e.s[i], norm);
    // (an entry of probability 0 adds nothing, whatever its logit)
    if (q != 0.0f) total += q * ((e.s[i] - norm) - (z[lane + 64 * i] * inverse - l));
  }
  total = reduce_sum_xor<64>(total) * temperature * temperature;
  uint32_t bits = __builtin_amdgcn_ballot_w64(bad) ? kErrTarget : 0;
  if (!__builtin_isfinite(total)) bits |= kErrLoss;
  if (lane) return;
  lse[row] = l;
  loss[row] = total;
  if (bits) atomicOr(err, bits);
}

// Rows whose entries' logits are there, a wave each
__global__ __launch_bounds__(256) void distill_join_kernel(const float2* stats, const uint32_t* ids,
                                                           const float* teacher, const float* teacher_lse,
                                                           const float* logits, float* loss, float* lse, uint32_t* err,
                                                           uint32_t rows, uint32_t vocab, uint32_t tiles, uint32_t top_k,
                                                           float temperature) {
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const uint64_t at = (uint64_t)row * top_k;
  const float l = joined(stats + (uint64_t)row * tiles, tiles, 1.0f / temperature);
  Entries e;
  const bool bad = load_entries(e, ids, teacher, at, top_k, vocab, 1.0f / temperature);
  row_loss(e, bad, teacher_lse, logits + at, l, loss, lse, err, row, temperature);
}

// A row by eight waves: one joins its pairs while the others work out its entries'
// logits
__global__ __launch_bounds__(512) void distill_row_kernel(const uint16_t* x, const uint16_t* w, const float2* stats,
                                                          const uint32_t* ids, const float* teacher,
                                                          const float* teacher_lse, float* logits, float* loss, float* lse,
                                                          uint32_t* err, uint32_t vocab, uint32_t hidden, uint32_t tiles,
                                                          uint32_t top_k, float temperature) {
  __shared__ float z[kTopMax];
  const uint32_t row = blockIdx.x, wave = threadIdx.x >> 6;
  const uint64_t at = (uint64_t)row * top_k;
  float l = 0.0f;
  bool bad = false;
  Entries e;
  if (wave == 0) {
    l = joined(stats + (uint64_t)row * tiles, tiles, 1.0f / temperature);
    bad = load_entries(e, ids, teacher, at, top_k, vocab, 1.0f / temperature);
  } else {
    for (uint32_t k = wave - 1; k < top_k; k += 7) {
      const float v = entry_logit(x + (uint64_t)row * hidden, w, ids[at + k], vocab, hidden);
      if ((threadIdx.x & 63) == 0) z[k] = logits[at + k] = v;
    }
  }
  __syncthreads();
  if (wave == 0) row_loss(e, bad, teacher_lse, z, l, loss, lse, err, row, temperature);
}

// What the backward pass needs of a row's teacher, by a wave: live 0
// (kNoTarget where no entry has a probability), the normalizer, Q, lse - log Q
// and the upstream factor up T
struct TeacherRows {
  uint32_t* live;
  float *norm, *total, *shift, *up;
};
__global__ __launch_bounds__(256) void distill_teacher_kernel(const uint32_t* ids, const float* teacher,
                                                              const float* teacher_lse, const float* lse,
                                                              const float* loss_grad, TeacherRows out, uint32_t* err,
                                                              uint32_t rows, uint32_t vocab, uint32_t top_k,
                                                              float temperature) {
  const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (row >= rows) return;
  Entries e;
  const bool bad = load_entries(e, ids, teacher, (uint64_t)row * top_k, top_k, vocab, 1.0f / temperature);
  const float norm = normalizer(e, teacher_lse, row);
  float total = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) total += probability(e.s[i], norm);
  total = reduce_sum_xor<64>(total);
  const bool any_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
  if (lane) return;
  out.live[row] = total == 0.0f ? kNoTarget : 0;
  out.norm[row] = norm;
  out.total[row] = total;
  out.shift[row] = lse[row] - logf(total);
  out.up[row] = loss_grad[row] * temperature;
  if (any_bad) atomicOr(err, kErrTarget);
}

// g at the teacher's entries whose id lies in the piece [v0, v0 + cols), a
// wave a row; an id twice in a row gets the sum of its entries twice, the same
__global__ __launch_bounds__(256) void distill_entries_kernel(const uint32_t* ids, const float* teacher,
                                                              const float* logits, const float* lse, TeacherRows in,
                                                              const float* mantissa, uint16_t* g, uint64_t ldg,
                                                              uint32_t rows, uint32_t vocab, uint32_t top_k, uint32_t v0,
                                                              uint32_t cols, float temperature) {
  __shared__ uint32_t all_id[4][kTopMax];
  __shared__ float all_q[4][kTopMax];
  const uint32_t wave = threadIdx.x >> 6, row = blockIdx.x * 4 + wave, lane = threadIdx.x & 63;
  if (row >= rows || in.live[row] == kNoTarget) return;
  Entries e;
  const float inverse = 1.0f / temperature;
  const uint64_t at = (uint64_t)row * top_k;
  load_entries(e, ids, teacher, at, top_k, vocab, inverse);
  const float norm = in.norm[row];
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    all_id[wave][lane + 64 * i] = e.id[i];
    all_q[wave][lane + 64 * i] = probability(e.s[i], norm);
  }
  wave_lds_order();
#pragma unroll
  for (uint32_t i = 0; i < kTopMax / 64; ++i) {
    const uint32_t id = e.id[i], place = id - v0;
    if (id == kNoTarget || place >= cols) continue;
    float q = 0.0f;
    for (uint32_t k = 0; k < top_k; ++k) q += all_id[wave][k] == id ? all_q[wave][k] : 0.0f;
    const float p = in.total[row] * at_most(expf(logits[at + lane + 64 * i] * inverse - lse[row]), 1.0f);
    g[row * ldg + place] = (uint16_t)f32_to_bf16_bits(mantissa[row] * (p - q));
  }
}

bool distill_ok(const LmHeadDistillArgs& a) {
  return shape_ok(a.rows, a.vocab, a.hidden) && a.top_k && a.top_k <= kTopMax;
}
// (log2(e) / t multiplies the logits' differences, 0 among them)
bool temperature_ok(float t) { return t > 0.0f && __builtin_isfinite(t) && __builtin_isfinite(kLog2e / t); }

// Whether the tiles write the entries' logits: 4 us a round of tiles and 6 for the
// sort, against the dot products' bytes at 8 TB/s.  64 entries, 4096 rows over
// 129280 x 4096: 3499 us with dot products, 3330 so; 20 entries, 33 rows over
// 151936 x 1024: 68 and 74.
bool listed(uint32_t rows, uint32_t vocab, uint32_t hidden, uint32_t top_k) {
  const float rounds = (float)rows * vocab / (65536.0f * kCus);
  return big_takes(hidden) && (float)rows * top_k * hidden * (2.0f / 8.0e6f) > 6.0f + 4.0f * rounds;
}
// Whether a row's entries are few enough for the waves beside the one that joins it,
// us, two launches -> one: 33 rows over 151936 x 1024, 20 entries 68.5 -> 65.1, 64
// 69.2 -> 71.9; over 129280 x 4096, 1 entry 200 -> 196, 20 199 -> 201.5
bool by_row(uint32_t hidden, uint32_t top_k) { return top_k * hidden <= 1u << 15; }
// the forward pass's workspace: the rows' pairs, and for the tiles fed by DMA the
// entries in order and how many lie before each tile
struct DistillForward {
  uint64_t sorted, before, bytes;
};
DistillForward distill_forward(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  DistillForward f{};
  f.bytes = f.sorted = padded((uint64_t)rows * stat_tiles(vocab, hidden) * 8);
  if (!big_takes(hidden)) return f;
  f.before = f.sorted + padded((uint64_t)rows * kTopMax * 4);
  f.bytes = f.before + padded((uint64_t)rows * (stat_tiles(vocab, hidden) + 1) * 2);
  return f;
}

struct DistillPlan {
  BackwardPlan loss;
  DxRoute dx;
  uint64_t live, norm, total, shift, up, bytes;
};
DistillPlan distill_plan(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  DistillPlan p{};
  p.loss = backward_plan(rows, vocab, hidden);
  // (dx has its own sums)
  p.dx = dx_route(rows, hidden, (std::min(p.loss.piece, vocab) + KB - 1) / KB * KB);
  const uint64_t each = padded((uint64_t)rows * 4);
  p.loss.factor = p.loss.sums + padded(p.dx.sums * 4);
  p.loss.mantissa = p.loss.factor + padded(4);
  p.live = p.loss.mantissa + each;
  p.norm = p.live + each;
  p.total = p.norm + each;
  p.shift = p.total + each;
  p.up = p.shift + each;
  p.bytes = p.up + each;
  return p;
}

}  // namespace

uint64_t LmHeadDistillWorkspaceBytes(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  if (!shape_ok(rows, vocab, hidden)) return 0;
  return distill_forward(rows, vocab, hidden).bytes;
}

uint64_t LmHeadDistillBackwardWorkspaceBytes(uint32_t rows, uint32_t vocab, uint32_t hidden) {
  return shape_ok(rows, vocab, hidden) ? distill_plan(rows, vocab, hidden).bytes : 0;
}

St LaunchLmHeadDistill(const LmHeadDistillArgs& a) {
  if (!a.x || !a.w || !a.ids || !a.teacher || !a.loss || !a.lse || !a.logits || !a.workspace || !a.error_flag ||
      !a.stream)
    return Invalid("lm_head_distill_null_argument");
  if (!distill_ok(a)) return Invalid("lm_head_distill_shape_invalid");
  if (!temperature_ok(a.temperature)) return Invalid("lm_head_distill_temperature_invalid");
  if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.ids, 4) || !aligned(a.teacher, 4) ||
      !aligned(a.teacher_lse, 4) || !aligned(a.loss, 4) || !aligned(a.lse, 4) || !aligned(a.logits, 4) ||
      !aligned(a.error_flag, 4))
    return Invalid("lm_head_distill_alignment_invalid");
  const uint64_t each = (uint64_t)a.rows * 4, entries = each * a.top_k;
  const Span x{a.x, (uint64_t)a.rows * a.hidden * 2}, w{a.w, (uint64_t)a.vocab * a.hidden * 2};
  const Span results[] = {{a.loss, each}, {a.lse, each}, {a.logits, entries}};
  const Span inputs[] = {x, w, {a.ids, entries}, {a.teacher, entries}};
  const Span teacher_lse{a.teacher_lse, each};
  bool alias = ResultsOverlap(results, inputs) || Overlap(results[2], teacher_lse);
  // (a row's own place in it is read before its loss and lse are written)
  for (int r = 0; r < 2; ++r) alias |= results[r].p != teacher_lse.p && Overlap(results[r], teacher_lse);
  if (alias) return Invalid("lm_head_distill_alias_invalid");
  if (a.workspace_bytes < LmHeadDistillWorkspaceBytes(a.rows, a.vocab, a.hidden) || !aligned(a.workspace, 16))
    return Invalid("lm_head_distill_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  const uint32_t tiles = stat_tiles(a.vocab, a.hidden);
  float2* const stats = static_cast<float2*>(a.workspace);
  const bool in_tiles = listed(a.rows, a.vocab, a.hidden, a.top_k);
  if (big_takes(a.hidden)) {
    const DistillForward plan = distill_forward(a.rows, a.vocab, a.hidden);
    uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
    uint32_t* const sorted = reinterpret_cast<uint32_t*>(ws + plan.sorted);
    uint16_t* const before = reinterpret_cast<uint16_t*>(ws + plan.before);
    if (in_tiles)
      hipLaunchKernelGGL(distill_sort_kernel, dim3((a.rows + 3) / 4), dim3(256), 0, a.stream, a.ids, sorted, before, a.logits,
                         a.rows, a.vocab, tiles, a.top_k);
    BigArgs b{};
    b.a = a.x;
    b.b = a.w;
    b.m = a.rows;
    b.n = b.vocab = a.vocab;
    b.k = a.hidden;
    b.lda = b.ldb = a.hidden;
    b.stats = stats;
    b.exponent = kLog2e / a.temperature;
    b.sorted = sorted;
    b.before = in_tiles ? before : nullptr;
    b.logits = a.logits;
    b.top_k = a.top_k;
    launch_big<false, false, kEpiTeacherStats>(b, a.stream);
  } else {
    GemmArgs g{};
    g.a = a.x;
    g.b = a.w;
    g.m = a.rows;
    g.n = g.vocab = a.vocab;
    g.k = a.hidden;
    g.lda = g.ldb = a.hidden;
    g.stat_tiles = tiles;
    g.stats = stats;
    g.inverse = 1.0f / a.temperature;
    launch_gemm<kEpiTeacherStats>(g, a.stream);
  }
  if (!in_tiles && by_row(a.hidden, a.top_k)) {
    hipLaunchKernelGGL(distill_row_kernel, dim3(a.rows), dim3(512), 0, a.stream, a.x, a.w, stats, a.ids, a.teacher,
                       a.teacher_lse, a.logits, a.loss, a.lse, a.error_flag, a.vocab, a.hidden, tiles, a.top_k,
                       a.temperature);
    return AfterLaunch("lm_head_distill_launch_failed");
  }
  if (!in_tiles) {
    const uint64_t entries = (uint64_t)a.rows * a.top_k;
    hipLaunchKernelGGL(distill_gather_kernel, dim3((uint32_t)std::min<uint64_t>((entries + 3) / 4, 1u << 20)), dim3(256), 0,
                       a.stream, a.x, a.w, a.ids, a.logits, entries, a.top_k, a.vocab, a.hidden);
  }
  hipLaunchKernelGGL(distill_join_kernel, dim3((a.rows + 3) / 4), dim3(256), 0, a.stream, stats, a.ids, a.teacher,
                     a.teacher_lse, a.logits, a.loss, a.lse, a.error_flag, a.rows, a.vocab, tiles, a.top_k,
                     a.temperature);
  return AfterLaunch("lm_head_distill_launch_failed");
}

St LaunchLmHeadDistillBackward(const LmHeadDistillArgs& a) {
  if (!a.x || !a.w || !a.ids || !a.teacher || !a.lse || !a.logits || !a.loss_grad || !a.dx || !a.workspace ||
      !a.error_flag || !a.stream)
    return Invalid("lm_head_distill_backward_null_argument");
  if (!distill_ok(a)) return Invalid("lm_head_distill_backward_shape_invalid");
  if (!temperature_ok(a.temperature)) return Invalid("lm_head_distill_backward_temperature_invalid");
  if (!aligned(a.x, 16) || !aligned(a.w, 16) || !aligned(a.dx, 16) || !aligned(a.dw, 16) || !aligned(a.ids, 4) ||
      !aligned(a.teacher, 4) || !aligned(a.teacher_lse, 4) || !aligned(a.lse, 4) || !aligned(a.logits, 4) ||
      !aligned(a.loss_grad, 4) || !aligned(a.error_flag, 4))
    return Invalid("lm_head_distill_backward_alignment_invalid");
  // (a piece's weights' gradient is written before dx reads its weights, and before
  // the other pieces read the rest)
  const uint64_t each = (uint64_t)a.rows * 4, entries = each * a.top_k;
  const uint64_t of_rows = (uint64_t)a.rows * a.hidden * 2, of_weight = (uint64_t)a.vocab * a.hidden * 2;
  const Span results[] = {{a.dx, of_rows}, {a.dw, of_weight}};
  const Span inputs[] = {{a.x, of_rows},          {a.w, of_weight}, {a.ids, entries},    {a.teacher, entries},
                         {a.teacher_lse, each}, {a.lse, each},    {a.logits, entries}, {a.loss_grad, each}};
  if (ResultsOverlap(results, inputs)) return Invalid("lm_head_distill_backward_alias_invalid");
  const DistillPlan plan = distill_plan(a.rows, a.vocab, a.hidden);
  if (a.workspace_bytes < plan.bytes || !aligned(a.workspace, 16))
    return Invalid("lm_head_distill_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  uint16_t* const grad = reinterpret_cast<uint16_t*>(ws + plan.loss.g);
  float* const mantissa = reinterpret_cast<float*>(ws + plan.loss.mantissa);
  const TeacherRows rows{reinterpret_cast<uint32_t*>(ws + plan.live), reinterpret_cast<float*>(ws + plan.norm),
                         reinterpret_cast<float*>(ws + plan.total), reinterpret_cast<float*>(ws + plan.shift),
                         reinterpret_cast<float*>(ws + plan.up)};
  const dim3 row_grid((a.rows + 3) / 4);
  hipLaunchKernelGGL(distill_teacher_kernel, row_grid, dim3(256), 0, a.stream, a.ids, a.teacher, a.teacher_lse, a.lse,
                     a.loss_grad, rows, a.error_flag, a.rows, a.vocab, a.top_k, a.temperature);
  BackwardCall call{};
  call.x = a.x;
  call.w = a.w;
  call.target = rows.live;
  call.lse = rows.shift;
  call.up = rows.up;
  call.dx = a.dx;
  call.dw = a.dw;
  call.error_flag = a.error_flag;
  call.stream = a.stream;
  call.rows = a.rows;
  call.vocab = a.vocab;
  call.hidden = a.hidden;
  call.temperature = a.temperature;
  call.most = rows.total;
  auto entries_of = [&](uint32_t v0, uint32_t cols) {
    hipLaunchKernelGGL(distill_entries_kernel, row_grid, dim3(256), 0, a.stream, a.ids, a.teacher, a.logits, a.lse, rows,
                       mantissa, grad, (uint64_t)plan.loss.piece, a.rows, a.vocab, a.top_k, v0, cols, a.temperature);
  };
  // Below, a log-sum-exp of logits of some hundred, rounded, makes exponentials that
  // pass 1, by e^88 where it is 7e8; the limit on each costs 1021 rows over 151936 x
  // 1024 2 to 6 %, also where rows without need of one skip it
  if (a.temperature < 0x1p-10f) launch_backward<kEpiTeacherGradLow>(call, plan.loss, &plan.dx, ws, entries_of);
  else launch_backward<kEpiTeacherGrad>(call, plan.loss, &plan.dx, ws, entries_of);
  return AfterLaunch("lm_head_distill_backward_launch_failed");
}

}  // namespace pih_amd
