// Verification of drafted tokens against a target model's logits for gfx950.
// With p and q the softmax of a target and a draft row over the sequence's
// temperature T, u and r given uniform numbers: drafted token d is accepted
// while u q(d) < p(d); behind the accepted ones comes the smallest v with
//   sum over v' <= v of w(v') > r sum of w,   w = max(0, p - q) at the rejected
// place, w = p behind the last one.  (The tokens so put out are distributed as
// the target's own.)
//
// Which token passes the threshold is decided among sums over the whole
// vocabulary, whose neighbours may differ by 1e-8 and less; exponentials and
// sums are therefore in 64 bits (of which the vector units do as many a clock
// as of 32), so that the order of the sums moves no token.
//
// Launches: the largest logit and the sum of exponentials of every row and chunk
// of the vocabulary; then for few sequences one launch, a block per sequence and
// chunk, that does the three others' work: a block per sequence that joins the
// rows and walks the drafts; the chunks' sums of w at the rejected places; a block
// per sequence that finds the chunk and in it the token.  (The last two in one for
// many, the token found by the last of a sequence's blocks: 57 sequences 21 -> 24
// us, 256 46 -> 58.)
//
// Measured: 1 sequence of 5 drafts over 151936 columns of fp32 23 us (two launches of
// 5 and 18, dependent loads), 57 of up to 7 over 129280 of bf16, looked up, 52-54, 256
// of up to 4 over 151936 of fp32 205-220.  The statistics are bound by the 64-bit
// arithmetic of their exponentials: 1.0 G logits a ms in bf16 (33 M in 34 us, 2.0 TB/s)
// as in fp32 (194 M in 185-202, 3.9-4.2 TB/s, the vector units busy in 85 % of the cycles).
#include "dense_route.hpp"
#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kChunk = 4096, kPer = kChunk / 256;  // a block's columns, a thread's
constexpr uint32_t kMaxVocab = 1u << 20, kMaxSequences = 1u << 14, kMostDrafts = 255;
constexpr uint32_t kNone = 0xffffffffu;
constexpr uint32_t kErrToken = 1u, kErrOffsets = 2u, kErrRow = 4u;
static_assert(kMaxVocab / kChunk <= 256, "a thread per chunk");

struct Stat {
  double sum;      // of exp((logit - top) / T)
  float top;       // largest logit
  uint32_t index;  // greedy: its first place
};
// What the walk over a sequence's drafts leaves to be drawn
struct Plan {
  double p_inverse, q_inverse, k;  // 1 / sums of the rows, log2(e) / T
  float p_top, q_top;
  uint32_t place;       // in the sequence, kNone: nothing to draw
  uint32_t rejected;    // the draft row or token `without` is taken off
  uint32_t without;     // looked-up drafts: the rejected token
  uint32_t target_row, draft_row;
  uint32_t pad;
};

struct VerifyArgs {
  const void* target;
  const void* draft;
  const uint32_t* tokens;
  const uint32_t* offsets;
  const float* accept;
  const float* sample;
  const float* temperature;
  uint32_t* out;
  uint32_t* accepted;
  uint32_t* err;
  Stat* stats;   // [sequences][rows][chunks]
  Plan* plans;   // [sequences]
  double* rest;  // [sequences][chunks]
  uint32_t* done;  // [sequences]: blocks that have written theirs
  uint64_t target_stride, draft_stride;
  uint32_t sequences, drafts, most, vocab, chunks, rows;
};

// 2^y for y <= 0, 2^-1021 for all below that (and -inf): 2^f of |f| <= 1/2 by the
// polynomial of degree 9 whose largest relative error, 1.4e-14, is least (Remez
// exchange), times 2^n by an addition to the exponent; n = rint(y) by adding and
// taking off 1.5 * 2^52, whose sum's lower word is n.  So all of it but the
// conversion of y's float issues at the full rate, which rounding and ldexp do
// not (16 exponentials a thread with those and degree 11: 194e6 logits in 202 us).
// `lead`: lead_coefficient(), once for many
__device__ __forceinline__ double lead_coefficient() {
  double e = 0x1.b3f4221448a2ap-24;
  asm("" : "+v"(e));  // (in registers: an FMA takes one constant from elsewhere)
  return e;
}
__device__ __forceinline__ double exp2_64(double y, double lead) {
  constexpr double kRound = 6755399441055744.0;
  y = __builtin_fmax(y, -1021.0);
  const double n = y + kRound, f = y - (n - kRound);
  double e = __builtin_fma(lead, f, 0x1.63edf10ad3737p-20);
  e = __builtin_fma(e, f, 0x1.ffce246029cbcp-17);
  e = __builtin_fma(e, f, 0x1.43088fca94b5ep-13);
  e = __builtin_fma(e, f, 0x1.5d87fd9012504p-10);
  e = __builtin_fma(e, f, 0x1.3b2ab72a109c3p-7);
  e = __builtin_fma(e, f, 0x1.c6b08d70d1fffp-5);
  e = __builtin_fma(e, f, 0x1.ebfbdff81570dp-3);
  e = __builtin_fma(e, f, 0x1.62e42fefa3752p-1);
  e = __builtin_fma(e, f, 0x1.0000000000039p+0);
  uint2 v = __builtin_bit_cast(uint2, e);
  asm("v_lshl_add_u32 %0, %1, 20, %0" : "+v"(v.y) : "v"(__builtin_bit_cast(uint2, n).x));
  return __builtin_bit_cast(double, v);
}
// the same, and 0 below 2^-1021
__device__ __forceinline__ double exp2_or_0(double y, double lead) { return y < -1021.0 ? 0.0 : exp2_64(y, lead); }
__device__ __forceinline__ double exp2_or_0(double y) { return exp2_or_0(y, lead_coefficient()); }

// A thread's logits from column c on, -inf past the vocabulary
template <bool BF16, bool WIDE>
__device__ __forceinline__ void load_logits(float (&v)[kPer], const void* row, uint32_t c, uint32_t vocab) {
  if (WIDE && c + kPer <= vocab) {
    if constexpr (BF16) {
      const uint4* const p = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c);
      const uint4 x = p[0], y = p[1];
      const uint32_t w[kPer / 2] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
      for (uint32_t e = 0; e < kPer; ++e) v[e] = bf16_bits_to_f32((w[e / 2] >> (16 * (e & 1))) & 0xffffu);
    } else {
      const v4f* const p = reinterpret_cast<const v4f*>(static_cast<const float*>(row) + c);
#pragma unroll
      for (uint32_t i = 0; i < kPer / 4; ++i) {
        const v4f x = p[i];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) v[4 * i + e] = x[e];
      }
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
      v[i] = -INFINITY;
      if (c + i < vocab)
        v[i] = BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(row)[c + i]) : static_cast<const float*>(row)[c + i];
    }
  }
}

template <bool BF16>
__device__ __forceinline__ const void* row_of(const void* base, uint64_t stride, uint64_t row) {
  return static_cast<const uint8_t*>(base) + row * stride * (BF16 ? 2 : 4);
}
template <bool BF16>
__device__ __forceinline__ float logit_at(const void* row, uint32_t c) {
  return BF16 ? bf16_bits_to_f32(static_cast<const uint16_t*>(row)[c]) : static_cast<const float*>(row)[c];
}

// Running sums and largest values over a wave by lane moves: within 16 lanes, then
// from the last lane of one 16 to the next, then from the 32nd to the upper half;
// lane 63 has all.  (~25 cycles a step of a 64-bit sum; through LDS ~130.)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v, uint32_t other) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)other, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double plus_moved(double v) {
  const uint2 x = __builtin_bit_cast(uint2, v);
  return v + __builtin_bit_cast(double, uint2{moved<CTRL, ROWS>(x.x, 0u), moved<CTRL, ROWS>(x.y, 0u)});
}
__device__ __forceinline__ double wave_running_sum(double v) {
  v = plus_moved<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v = plus_moved<0x112, 0xf>(v);
  v = plus_moved<0x114, 0xf>(v);
  v = plus_moved<0x118, 0xf>(v);
  v = plus_moved<0x142, 0xa>(v);  // row_bcast 15
  return plus_moved<0x143, 0xc>(v);  // row_bcast 31
}
__device__ __forceinline__ double wave_sum(double v) {
  const uint2 x = __builtin_bit_cast(uint2, wave_running_sum(v));
  return __builtin_bit_cast(double, uint2{(uint32_t)__builtin_amdgcn_readlane((int)x.x, 63),
                                          (uint32_t)__builtin_amdgcn_readlane((int)x.y, 63)});
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_moved(float v) {
  return fmaxf(v, __uint_as_float(moved<CTRL, ROWS>(__float_as_uint(v), 0xff800000u)));
}
__device__ __forceinline__ float wave_max(float v) {
  v = max_moved<0x111, 0xf>(v);
  v = max_moved<0x112, 0xf>(v);
  v = max_moved<0x114, 0xf>(v);
  v = max_moved<0x118, 0xf>(v);
  v = max_moved<0x142, 0xa>(v);
  v = max_moved<0x143, 0xc>(v);
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

struct Sequence {
  uint32_t first, count;
  float temperature;
  bool offsets_ok;
};
__device__ __forceinline__ Sequence sequence_of(const VerifyArgs& p, uint32_t s) {
  const uint32_t lo = p.offsets[s], hi = p.offsets[s + 1];
  const float t = p.temperature ? p.temperature[s] : 1.0f;
  return {lo, hi - lo, t, lo <= hi && hi <= p.drafts && hi - lo <= p.most};
}
// (what is left of these stops the sequence at its first place)
__device__ __forceinline__ bool temperature_ok(float t) { return t >= 0.0f && t < INFINITY; }

template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs p) {
  __shared__ double sums[4];
  __shared__ float tops[4];
  __shared__ uint32_t indexes[4];
  const uint32_t chunk = blockIdx.x % p.chunks, at = blockIdx.x / p.chunks, y = at % p.rows, s = at / p.rows;
  const Sequence q = sequence_of(p, s);
  if (y == 0 && chunk == 0 && threadIdx.x == 0) p.done[s] = 0;
  const bool greedy = q.temperature == 0.0f, of_draft = y > p.most;
  const uint32_t place = of_draft ? y - p.most - 1 : y;
  if (!q.offsets_ok || !temperature_ok(q.temperature) || place > q.count || (of_draft && (greedy || place == q.count)))
    return;
  const void* const row = of_draft ? row_of<BF16>(p.draft, p.draft_stride, (uint64_t)q.first + place)
                                   : row_of<BF16>(p.target, p.target_stride, (uint64_t)q.first + s + place);
  const uint32_t c = chunk * kChunk + threadIdx.x * kPer, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float v[kPer];
  load_logits<BF16, WIDE>(v, row, c, p.vocab);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < (int)kPer; ++i) top = fmaxf(top, v[i]);
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  double sum = 0.0;
  uint32_t index = kNone;
  bool bad = false;
  if (greedy) {
#pragma unroll
    for (int i = (int)kPer - 1; i >= 0; --i) {
      if (v[i] == top) index = c + i;
      bad |= v[i] != v[i];
    }
    if (index >= p.vocab) index = kNone;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) index = min(index, (uint32_t)__shfl_xor((int)index, off, 64));
  } else {
    const double k = 1.44269504088896340736 / (double)q.temperature, shift = -(double)top * k;
    const double lead = lead_coefficient();
    // the argument in one FMA where -top k, whose rounding puts all of the chunk off
    // by one factor, is at most 2^10 and that within 1e-13 of 1 (otherwise the logits
    // are read again one by one: both unrolled took 76 registers and 2 % more time)
    if (__builtin_fabs(shift) <= 1024.0) {
#pragma unroll
      for (int i = 0; i < (int)kPer; ++i) sum += exp2_64(__builtin_fma((double)v[i], k, shift), lead);
    } else {
#pragma unroll 1
      for (uint32_t i = c; i < min(c + kPer, p.vocab); ++i)
        sum += exp2_64(((double)logit_at<BF16>(row, i) - (double)top) * k, lead);
    }
#pragma unroll
    for (int i = 0; i < (int)kPer; ++i) bad |= !(v[i] < INFINITY);  // +inf or NaN
    if (top == -INFINITY) sum = 0.0;
  }
  if (bad) sum = __builtin_nan("");
  sum = wave_sum(sum);
  if (lane == 0) {
    sums[wave] = sum;
    indexes[wave] = index;
  }
  __syncthreads();
  if (threadIdx.x == 0)
    p.stats[(uint64_t)at * p.chunks + chunk] = Stat{sums[0] + sums[1] + sums[2] + sums[3], top,
                                                    min(min(indexes[0], indexes[1]), min(indexes[2], indexes[3]))};
}

struct WalkRows {
  double sum[2 * kMostDrafts + 1];
  float top[2 * kMostDrafts + 1];
  uint32_t index[kMostDrafts + 1];
  uint32_t stop, why;
};
// The walk over a sequence's drafts by a block: what is left to be drawn into
// `plan` (in LDS too; to be read behind a barrier), the tokens and the count written
// by the one block that `writes`
template <bool BF16>
__device__ __forceinline__ void walk(const VerifyArgs& p, uint32_t s, bool writes, WalkRows& row, Plan& plan) {
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Sequence q = sequence_of(p, s);
  uint32_t* const out = p.out + (uint64_t)s * (p.most + 1);
  const bool usable = q.offsets_ok && temperature_ok(q.temperature), greedy = q.temperature == 0.0f;
  if (!usable) {
    for (uint32_t i = tid; writes && i <= p.most; i += 256) out[i] = kNone;
    if (tid == 0) {
      plan.place = kNone;
      if (writes) {
        p.accepted[s] = 0;
        atomicOr(p.err, q.offsets_ok ? kErrRow : kErrOffsets);
      }
    }
    return;
  }
  const double k = 1.44269504088896340736 / (double)(greedy ? 1.0f : q.temperature);
  const bool soft = p.draft && !greedy;
  // rows 0 .. count of the target, then the draft's; four of a wave's at a time
  const uint32_t rows = q.count + 1 + (soft ? q.count : 0);
  auto stats_of = [&](uint32_t r) {
    const uint32_t y = r <= q.count ? r : p.most + 1 + r - (q.count + 1);
    return p.stats + ((uint64_t)s * p.rows + y) * p.chunks;
  };
  Stat ahead[4];
  auto load_rows = [&](uint32_t r0) {
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
      ahead[b] = Stat{0.0, -INFINITY, kNone};
      if (r0 + 4 * b < rows && lane < p.chunks) ahead[b] = stats_of(r0 + 4 * b)[lane];
    }
  };
  load_rows(wave);
  // (a draft's own logits, on their way while the rows are joined)
  uint32_t token = kNone;
  float target_logit = 0.0f, draft_logit = 0.0f, number = 0.0f;
  if (tid < q.count) {
    token = p.tokens[q.first + tid];
    number = p.accept[q.first + tid];
    if (token < p.vocab) {
      target_logit = logit_at<BF16>(row_of<BF16>(p.target, p.target_stride, (uint64_t)q.first + s + tid), token);
      if (soft) draft_logit = logit_at<BF16>(row_of<BF16>(p.draft, p.draft_stride, (uint64_t)q.first + tid), token);
    }
  }
  for (uint32_t r0 = wave; r0 < rows; r0 += 16) {
    if (r0 != wave) load_rows(r0);
    float top[4];
    double sum[4];
    // (the four in step, for the waits in between)
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
      top[b] = ahead[b].top;
      for (uint32_t i = lane + 64; r0 + 4 * b < rows && i < p.chunks; i += 64)
        top[b] = fmaxf(top[b], stats_of(r0 + 4 * b)[i].top);
    }
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) top[b] = wave_max(top[b]);
    // (a chunk of -inf alone has the sum 0, or NaN)
    auto part = [&](const Stat& x, float largest) {
      if (greedy || x.top == -INFINITY) return x.sum;
      return x.sum * exp2_or_0(((double)x.top - (double)largest) * k);
    };
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
      sum[b] = part(ahead[b], top[b]);
      for (uint32_t i = lane + 64; r0 + 4 * b < rows && i < p.chunks; i += 64)
        sum[b] += part(stats_of(r0 + 4 * b)[i], top[b]);
    }
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
      sum[b] = wave_sum(sum[b]);
      // greedy: a sum of 1 stands for a row that has a largest logit
      if (greedy && sum[b] == 0.0) sum[b] = top[b] == -INFINITY ? 0.0 : 1.0;
    }
#pragma unroll
    for (uint32_t b = 0; b < 4; ++b) {
      const uint32_t r = r0 + 4 * b;
      if (r >= rows) break;
      if (lane == 0) {
        row.sum[r] = sum[b];
        row.top[r] = top[b];
      }
      if (!greedy) continue;
      uint32_t index = ahead[b].top == top[b] ? ahead[b].index : kNone;
      for (uint32_t i = lane + 64; i < p.chunks; i += 64) {
        const Stat x = stats_of(r)[i];
        if (x.top == top[b]) index = min(index, x.index);
      }
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) index = min(index, (uint32_t)__shfl_xor((int)index, off, 64));
      if (lane == 0) row.index[r] = index;
    }
  }
  if (tid == 0) row.stop = q.count;
  __syncthreads();
  // a row's sum is above 0 and finite, or the row has no probabilities
  auto usable_row = [&](uint32_t r) { return row.sum[r] > 0.0 && row.sum[r] < (double)INFINITY; };
  bool ok = true, bad_token = false, bad_row = false;
  if (tid <= q.count) bad_row = !usable_row(tid) || (soft && tid < q.count && !usable_row(q.count + 1 + tid));
  if (tid < q.count) {
    bad_token = token >= p.vocab;
    if (greedy) {
      ok = token == row.index[tid];
    } else if (bad_token) {
      ok = false;
    } else {
      const double pd = exp2_or_0(((double)target_logit - (double)row.top[tid]) * k) / row.sum[tid];
      const uint32_t r = q.count + 1 + tid;
      const double qd = soft ? exp2_or_0(((double)draft_logit - (double)row.top[r]) * k) / row.sum[r] : 1.0;
      ok = (double)number * qd < pd;
    }
    if (!ok || bad_row) atomicMin(&row.stop, tid);
  }
  __syncthreads();
  const uint32_t j = row.stop;
  // the thread of the place has its token at hand
  if (tid == j) {
    const uint32_t bits = (bad_row ? kErrRow : 0) | (bad_token ? kErrToken : 0);
    row.why = bits;
    plan.place = greedy || (bits & kErrRow) ? kNone : j;
    plan.k = k;
    plan.p_top = row.top[j];
    plan.p_inverse = 1.0 / row.sum[j];
    plan.rejected = j < q.count;
    plan.target_row = q.first + s + j;
    plan.draft_row = q.first + j;
    plan.without = token;
    const bool with_draft = soft && j < q.count;
    plan.q_top = with_draft ? row.top[q.count + 1 + j] : 0.0f;
    plan.q_inverse = with_draft ? 1.0 / row.sum[q.count + 1 + j] : 0.0;
    if (writes) {
      p.accepted[s] = j;
      if (bits) atomicOr(p.err, bits);
    }
  }
  if (!writes) return;
  __syncthreads();
  const uint32_t bits = row.why;
  for (uint32_t i = tid; i <= p.most; i += 256) {
    uint32_t t = kNone;
    if (i < j) t = token;  // (i is tid: j <= count < 256)
    else if (i == j && greedy && !(bits & kErrRow)) t = row.index[j];
    // (the place to be drawn is written by who draws it, in another block perhaps)
    if (i != j || plan.place == kNone) out[i] = t;
  }
}

template <bool BF16>
__global__ __launch_bounds__(256) void verify_walk_kernel(VerifyArgs p) {
  __shared__ WalkRows rows;
  __shared__ Plan plan;
  walk<BF16>(p, blockIdx.x, true, rows, plan);
  __syncthreads();
  if (threadIdx.x == 0) p.plans[blockIdx.x] = plan;
}

// w of a thread's columns of a chunk; `whole`: p alone
template <bool BF16, bool WIDE>
__device__ __forceinline__ void weights(double (&w)[kPer], const VerifyArgs& p, const Plan& plan, uint32_t c, bool whole) {
  float v[kPer], d[kPer];
  const double lead = lead_coefficient();
  load_logits<BF16, WIDE>(v, row_of<BF16>(p.target, p.target_stride, plan.target_row), c, p.vocab);
  const bool soft = p.draft && !whole;
  if (soft) load_logits<BF16, WIDE>(d, row_of<BF16>(p.draft, p.draft_stride, plan.draft_row), c, p.vocab);
#pragma unroll
  for (int i = 0; i < (int)kPer; ++i) {
    w[i] = exp2_or_0(((double)v[i] - (double)plan.p_top) * plan.k, lead) * plan.p_inverse;
    if (!whole && !p.draft && c + i == plan.without) w[i] = 0.0;
  }
  if (!soft) return;
#pragma unroll
  for (int i = 0; i < (int)kPer; ++i) {
    const double e = w[i] - exp2_or_0(((double)d[i] - (double)plan.q_top) * plan.k, lead) * plan.q_inverse;
    w[i] = e > 0.0 ? e : 0.0;
  }
}

// Sum of w over a chunk, in thread 0
template <bool BF16, bool WIDE>
__device__ __forceinline__ double chunk_rest(const VerifyArgs& p, const Plan& plan, uint32_t chunk, double (&sums)[4]) {
  double w[kPer];
  weights<BF16, WIDE>(w, p, plan, chunk * kChunk + threadIdx.x * kPer, false);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < (int)kPer; ++i) sum += w[i];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  return sums[0] + sums[1] + sums[2] + sums[3];
}

// Sums of w over the chunks, at the rejected places
template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void verify_rest_kernel(VerifyArgs p) {
  __shared__ double sums[4];
  const uint32_t chunk = blockIdx.x % p.chunks, s = blockIdx.x / p.chunks;
  const Plan plan = p.plans[s];
  if (plan.place == kNone || !plan.rejected) return;
  const double sum = chunk_rest<BF16, WIDE>(p, plan, chunk, sums);
  if (threadIdx.x == 0) p.rest[(uint64_t)s * p.chunks + chunk] = sum;
}

// Running sum over the block's threads, in order; `parts`: one per wave
__device__ __forceinline__ double running_sum(double v, double (&parts)[4]) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_running_sum(v);
  if (lane == 63) parts[wave] = v;
  __syncthreads();
  for (uint32_t i = 0; i < wave; ++i) v += parts[i];
  return v;
}

// The token behind the accepted ones, by a block
struct PickRows {
  double parts[3][4];
  double all, before;
  uint32_t found, last;
};
// the sum of p over chunk threadIdx.x
__device__ __forceinline__ double chunk_of_p(const VerifyArgs& p, uint32_t s, const Plan& plan) {
  if (threadIdx.x >= p.chunks) return 0.0;
  const Stat st = p.stats[((uint64_t)s * p.rows + plan.place) * p.chunks + threadIdx.x];
  if (st.top == -INFINITY) return 0.0;
  return st.sum * exp2_or_0(((double)st.top - (double)plan.p_top) * plan.k) * plan.p_inverse;
}
// own: the sum of w over it
template <bool BF16, bool WIDE>
__device__ __forceinline__ void pick(const VerifyArgs& p, uint32_t s, const Plan& plan, PickRows& lds, float number,
                                     double of_p, double own) {
  const uint32_t tid = threadIdx.x;
  if (tid == 0) {
    lds.found = kNone;
    lds.last = 0;
  }
  // where the sums of w are 0 throughout, of p
  bool whole = !plan.rejected;
  double run = running_sum(whole ? of_p : own, lds.parts[0]);
  if (tid == 255) lds.all = run;
  __syncthreads();
  if (!whole && !(lds.all > 0.0)) {
    whole = true;
    run = running_sum(of_p, lds.parts[1]);
    if (tid == 255) lds.all = run;
    __syncthreads();
  }
  if (whole) own = of_p;
  const double threshold = (double)number * lds.all;
  // (where rounding leaves none above the threshold, the last that has a sum)
  if (own > 0.0) {
    if (run > threshold) atomicMin(&lds.found, tid);
    atomicMax(&lds.last, tid);
  }
  __syncthreads();
  const uint32_t chunk = lds.found != kNone ? lds.found : lds.last;
  if (tid == chunk) lds.before = run - own;
  __syncthreads();
  if (tid == 0) {
    lds.found = kNone;
    lds.last = 0;
  }
  const double left = threshold - lds.before;
  const uint32_t first = chunk * kChunk + tid * kPer;
  double w[kPer];
  weights<BF16, WIDE>(w, p, plan, first, whole);
  own = 0.0;
#pragma unroll
  for (int i = 0; i < (int)kPer; ++i) own += w[i];
  run = running_sum(own, lds.parts[2]);
  if (own > 0.0) {
    if (run > left) atomicMin(&lds.found, tid);
    atomicMax(&lds.last, tid);
  }
  __syncthreads();
  if (tid != (lds.found != kNone ? lds.found : lds.last)) return;
  double sum = run - own;
  uint32_t token = 0;
  bool done = false;
#pragma unroll
  for (int i = 0; i < (int)kPer; ++i) {
    if (done || !(w[i] > 0.0)) continue;
    sum += w[i];
    token = first + i;
    done = sum > left;
  }
  p.out[(uint64_t)s * (p.most + 1) + plan.place] = token;
}

// (1024 threads of 4 columns each: 10.4 -> 11.7 us for one sequence)
template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs p) {
  __shared__ PickRows lds;
  const uint32_t s = blockIdx.x;
  const Plan plan = p.plans[s];
  if (plan.place == kNone) return;
  const float number = p.sample[s];
  const double own = plan.rejected && threadIdx.x < p.chunks ? p.rest[(uint64_t)s * p.chunks + threadIdx.x] : 0.0;
  pick<BF16, WIDE>(p, s, plan, lds, number, chunk_of_p(p, s, plan), own);
}

// The three in one: every block of a sequence walks its drafts, the last that has
// its chunk's sum written finds the token
template <bool BF16, bool WIDE>
__global__ __launch_bounds__(256) void verify_draw_kernel(VerifyArgs p) {
  __shared__ WalkRows rows;
  __shared__ Plan plan;
  __shared__ PickRows lds;
  __shared__ double sums[4];
  __shared__ uint32_t order;
  const uint32_t chunk = blockIdx.x % p.chunks, s = blockIdx.x / p.chunks;
  const float number = p.sample[s];
  walk<BF16>(p, s, chunk == 0, rows, plan);
  __syncthreads();
  if (plan.place == kNone || (!plan.rejected && chunk)) return;
  double* const rest = p.rest + (uint64_t)s * p.chunks;
  // (on its way before the chunk's sum is worked out)
  const double of_p = chunk_of_p(p, s, plan);
  double own = 0.0;
  if (plan.rejected) {
    const double sum = chunk_rest<BF16, WIDE>(p, plan, chunk, sums);
    if (threadIdx.x == 0) {
      __hip_atomic_store(rest + chunk, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      order = __hip_atomic_fetch_add(p.done + s, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (order != p.chunks - 1) return;
    if (threadIdx.x < p.chunks) own = __hip_atomic_load(rest + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  pick<BF16, WIDE>(p, s, plan, lds, number, of_p, own);
}

bool sizes_ok(uint32_t sequences, uint32_t most, uint32_t vocab) {
  return sequences && sequences <= kMaxSequences && most <= kMostDrafts && vocab && vocab <= kMaxVocab;
}
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
uint64_t padded(uint64_t bytes) { return (bytes + 255) / 256 * 256; }
uint32_t chunks_of(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }

// whether a result overlaps one of the logits' rows (what lies between them is the
// caller's)
bool overlaps_rows(Span result, const void* base, uint64_t rows, uint64_t bytes, uint64_t stride) {
  if (!rows || !Overlap(result, {base, (rows - 1) * stride + bytes})) return false;
  const uintptr_t from = reinterpret_cast<uintptr_t>(result.p), first = reinterpret_cast<uintptr_t>(base);
  if (from < first) return true;
  const uint64_t row = (from - first) / stride, within = (from - first) % stride;
  return within < bytes || (row + 1 < rows && within + result.bytes > stride);
}

struct VerifyPlan {
  uint64_t plans, rest, done, bytes;
};
VerifyPlan verify_plan(uint32_t sequences, uint32_t most, uint32_t vocab) {
  VerifyPlan v{};
  v.plans = padded((uint64_t)sequences * (2 * most + 1) * chunks_of(vocab) * sizeof(Stat));
  v.rest = v.plans + padded((uint64_t)sequences * sizeof(Plan));
  v.done = v.rest + padded((uint64_t)sequences * chunks_of(vocab) * 8);
  v.bytes = v.done + padded((uint64_t)sequences * 4);
  return v;
}

template <bool BF16, bool WIDE>
void launch(const VerifyArgs& p, hipStream_t s) {
  hipLaunchKernelGGL((verify_stats_kernel<BF16, WIDE>), dim3(p.sequences * p.rows * p.chunks), dim3(256), 0, s, p);
  // One launch behind the first where its blocks, which repeat the walk, are at most
  // three for two CUs; us, three -> one: 151936 columns of fp32 with a draft
  // model's, 1 sequence (38 blocks) 25.5 -> 23.0, 4 27.2 -> 23.9, 32 (1216) 53.5 ->
  // 56.3; 129280 of bf16, 8 (256) 28.3 -> 27.4, 12 (384) 30.5 -> 30.9, 16 31.9 -> 33.6;
  // 32000, 1 (8) 23.7 -> 20.1, 32 (256) 30.9 -> 27.6
  if (p.sequences * p.chunks <= kCus * 3 / 2) {
    hipLaunchKernelGGL((verify_draw_kernel<BF16, WIDE>), dim3(p.sequences * p.chunks), dim3(256), 0, s, p);
    return;
  }
  hipLaunchKernelGGL((verify_walk_kernel<BF16>), dim3(p.sequences), dim3(256), 0, s, p);
  if (p.drafts) hipLaunchKernelGGL((verify_rest_kernel<BF16, WIDE>), dim3(p.sequences * p.chunks), dim3(256), 0, s, p);
  hipLaunchKernelGGL((verify_pick_kernel<BF16, WIDE>), dim3(p.sequences), dim3(256), 0, s, p);
}

}  // namespace

uint64_t DraftVerifyWorkspaceBytes(uint32_t sequences, uint32_t max_drafts, uint32_t vocab) {
  return sizes_ok(sequences, max_drafts, vocab) ? verify_plan(sequences, max_drafts, vocab).bytes : 0;
}

St LaunchDraftVerify(const DraftVerifyArgs& a) {
  if (!a.target || !a.offsets || !a.sample || !a.out || !a.accepted || !a.workspace || !a.error_flag || !a.stream ||
      (a.drafts && (!a.tokens || !a.accept)))
    return Invalid("draft_verify_null_argument");
  if (!sizes_ok(a.sequences, a.max_drafts, a.vocab) || a.drafts > (1u << 20) || a.target_stride < a.vocab ||
      (a.draft && a.draft_stride < a.vocab))
    return Invalid("draft_verify_shape_invalid");
  const uint32_t size = a.kind == kOutBf16 ? 2 : 4;
  if (!aligned(a.target, size) || !aligned(a.draft, size) || !aligned(a.tokens, 4) || !aligned(a.offsets, 4) ||
      !aligned(a.accept, 4) || !aligned(a.sample, 4) || !aligned(a.temperature, 4) || !aligned(a.out, 4) ||
      !aligned(a.accepted, 4) || !aligned(a.error_flag, 4))
    return Invalid("draft_verify_alignment_invalid");
  const uint64_t of_drafts = (uint64_t)a.drafts * 4, of_sequences = (uint64_t)a.sequences * 4;
  const Span results[] = {{a.out, of_sequences * (a.max_drafts + 1)}, {a.accepted, of_sequences}};
  const Span inputs[] = {{a.tokens, of_drafts},    {a.offsets, of_sequences + 4},   {a.accept, of_drafts},
                         {a.sample, of_sequences}, {a.temperature, of_sequences}};
  bool alias = ResultsOverlap(results, inputs);
  for (const Span& r : results)
    alias |= overlaps_rows(r, a.target, (uint64_t)a.drafts + a.sequences, (uint64_t)a.vocab * size,
                           (uint64_t)a.target_stride * size) ||
             overlaps_rows(r, a.draft, a.drafts, (uint64_t)a.vocab * size, (uint64_t)a.draft_stride * size);
  if (alias) return Invalid("draft_verify_alias_invalid");
  const VerifyPlan plan = verify_plan(a.sequences, a.max_drafts, a.vocab);
  const uint32_t chunks = chunks_of(a.vocab), rows = a.max_drafts + 1 + (a.draft ? a.max_drafts : 0);
  if (a.workspace_bytes < plan.bytes || !aligned(a.workspace, 16)) return Invalid("draft_verify_workspace_invalid");
  if ((uint64_t)a.sequences * rows * chunks > (1u << 24) - 1) return Invalid("draft_verify_shape_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  VerifyArgs p{};
  p.target = a.target;
  p.draft = a.draft;
  p.tokens = a.tokens;
  p.offsets = a.offsets;
  p.accept = a.accept;
  p.sample = a.sample;
  p.temperature = a.temperature;
  p.out = a.out;
  p.accepted = a.accepted;
  p.err = a.error_flag;
  p.stats = reinterpret_cast<Stat*>(ws);
  p.plans = reinterpret_cast<Plan*>(ws + plan.plans);
  p.rest = reinterpret_cast<double*>(ws + plan.rest);
  p.done = reinterpret_cast<uint32_t*>(ws + plan.done);
  p.target_stride = a.target_stride;
  p.draft_stride = a.draft_stride;
  p.sequences = a.sequences;
  p.drafts = a.drafts;
  p.most = a.max_drafts;
  p.vocab = a.vocab;
  p.chunks = chunks;
  p.rows = rows;
  // 16-byte reads of whole rows
  const bool wide = aligned(a.target, 16) && a.target_stride * size % 16 == 0 &&
                    (!a.draft || (aligned(a.draft, 16) && a.draft_stride * size % 16 == 0));
  if (a.kind == kOutBf16) {
    if (wide) launch<true, true>(p, a.stream);
    else launch<true, false>(p, a.stream);
  } else {
    if (wide) launch<false, true>(p, a.stream);
    else launch<false, false>(p, a.stream);
  }
  return AfterLaunch("draft_verify_launch_failed");
}

}  // namespace pih_amd
