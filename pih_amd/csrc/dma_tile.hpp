// Product tiles of bf16 operands fed by DMA, shared by the LM head's losses and
// the feed-forward block: C [m][n] = A . B^T on the MFMAs, summed in fp32, with
// what becomes of C chosen by EPI.
#pragma once

#include <algorithm>
#include <type_traits>

#include "dma_route.hpp"
#include "glu.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

// an entry of a list of vocabulary ids that is none
constexpr uint32_t kNoTarget = 0xffffffffu;

// kEpiStats: maximum and sum of exponentials of every row's columns, and the
// target's logit; kEpiGrad: the logits' gradient in bf16; kEpiBf16: a scaled
// result in bf16; kEpiAdd: added to fp32 sums; kEpiTeacherStats, kEpiTeacherGrad: the
// first two of logits over a temperature, without a target, the first with the
// logits at a list of columns that every row has; kEpiTeacherGradLow: the second at
// low temperatures.  The feed-forward block's: kEpiStore: bf16; kEpiSum: fp32, a plane
// per split; kEpiGlu: two products side by side, gate and up, joined to h;
// kEpiGluSum: the same two as kEpiSum; kEpiGluGrad: dh, joined with gate and up
enum : int {
  kEpiStats = 0, kEpiGrad = 1, kEpiBf16 = 2, kEpiAdd = 3, kEpiTeacherStats = 4, kEpiTeacherGrad = 5,
  kEpiStore = 6, kEpiSum = 7, kEpiGlu = 8, kEpiGluSum = 9, kEpiGluGrad = 10, kEpiTeacherGradLow = 11
};
constexpr bool has_pair(int epi) { return epi == kEpiGlu || epi == kEpiGluSum; }
constexpr bool has_stats(int epi) { return epi == kEpiStats || epi == kEpiTeacherStats; }
constexpr bool has_teacher_grad(int epi) { return epi == kEpiTeacherGrad || epi == kEpiTeacherGradLow; }
constexpr bool has_grad(int epi) { return epi == kEpiGrad || has_teacher_grad(epi); }

// ------------------------------------------------ tiles fed by DMA
// C [m][n] = A . B^T in tiles of 256 columns and 256, 128 or 64 rows.  Four
// waves: 2 x 2 quarters of 128 x 128 (64 x 128), one wave per SIMD with 256
// accumulator registers, or 1 x 4 of 64 x 64.  A K step is 64 deep and moved
// into LDS by DMA, two (128 and 64 rows: three) steps resident.  Two layouts
// of an operand:
//   rows     [row][k] in memory: LDS rows of 128 bytes, 16-byte chunk c of row
//            r in slot c ^ ((r >> 1) & 7); a fragment is one ds_read_b128
//            (16 rows, one chunk each: all 64 banks once);
//   columns  [k][row] in memory: LDS rows of 512 bytes (one k each), chunk c
//            of k row r in slot c ^ 2 f(r), f(r) = (r & 3) + 4 (r >> 3 & 1); a
//            fragment is two transposing reads (ds_read_b64_tr_b16: lane l of
//            16 gives the address of 4 values of k row l / 4 and receives
//            column l of the four rows), whose 8 k rows per half wave lie in
//            different 32-byte slots.
// The step's two 32-deep halves: while the MFMAs of the first run, the second
// half's fragments are read; then one wait and one barrier (every wave has
// read the step, and the next one has arrived), and while the MFMAs of the
// second run, the next step's first fragments are read and another step is
// sent for, into the buffer just freed.  With two steps resident the wait for
// the next one stands, with a barrier of its own, in the middle of the second
// half, and its fragments are read in the rest.  Reads and DMAs are issued one
// by one between MFMAs, which run for four issues each: in front of a group's
// eight the matrix pipe ran dry.  (Both together: the block's forward pass of 4099
// rows of 4096 x 12288 958 -> 920 us, its gradients of 4096 2046 -> 1964; the loss of
// 4096 rows over 129280 x 4096 3100 -> 2960, its gradients 9706 -> 9335; a half of it
// from the order of issue, a half from the wait.  The wait three, five or six eighths
// into the half: no better; DMAs all at its start: 4-8 % slower.)  A block per CU walks its tiles; the
// next tile's first steps are sent for before the results of this one are
// worked on.
// (Eight waves, two to a SIMD, that take turns on 32-deep halves, so that one's
// LDS reads run under the other's MFMAs: fewer cycles, but 5-10 % more time over
// and over, with more LDS traffic: power sets the clock, 1.9 GHz of 2.4.)

// 16 bytes of a row that is not there
__device__ const v4i kNoRow{0, 0, 0, 0};

struct BigArgs {
  const uint16_t* a;
  const uint16_t* b;
  uint32_t m, n, k;        // k a multiple of 64
  uint32_t k_valid;        // columns layout of B: k rows that exist (kEpiAdd, kEpiStore; the others are zeros)
  uint64_t lda, ldb;
  void* out;
  uint64_t ldo;
  uint32_t m_tiles, n_tiles, splits;
  uint64_t split_stride;   // kEpiAdd: elements between the splits' sums
  const uint32_t* target;
  const float* lse;
  const float* mantissa;   // kEpiGrad: [m]
  const float* scale;      // kEpiBf16: factor of the result
  float2* stats;
  float* target_logit;
  uint32_t v0, vocab, first;
  float exponent;          // kEpiTeacher*: log2(e) / temperature
  const float* most;       // kEpiTeacherGradLow: what a row's exponentials sum to
  // kEpiTeacherStats: a row's columns in order, id << 8 | place in its list
  // ([m][top_k]), how many of them lie before each tile ([m][n_tiles + 1]; null: no
  // lists), and where their logits go ([m][top_k])
  const uint32_t* sorted;
  const uint16_t* before;
  float* logits;
  uint32_t top_k;
  // the feed-forward block's products
  const uint16_t* b2;      // kEpiGlu*: up's weights; kEpiStore, kEpiSum: B behind step b_steps
  uint16_t* out2;          // kEpiStore: rows of the result from out_rows on
  uint32_t a_valid;        // kEpiStore, columns layout of A: as k_valid
  uint32_t b_steps, out_rows;
  uint16_t* gate;          // kEpiGlu: written where not null; kEpiGluGrad: read; [m][n or n / 2]
  uint16_t* up;
  uint16_t* h;             // kEpiGluGrad: beside out, which has dgate and n columns on dup
  uint64_t ldh;
  float limit;
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

__device__ __forceinline__ v4i join(v4s x, v4s y) {
  const uint2 a = __builtin_bit_cast(uint2, x), b = __builtin_bit_cast(uint2, y);
  return v4i{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
}

// Accumulators held in their registers: with all 256 in use the compiler
// otherwise moved them about, 518 moves beside 128 MFMAs (now none).
template <int NB>
__device__ __forceinline__ void pin(v4f (&c)[NB]) {
  static_assert(NB == 4 || NB == 8, "blocks");
  if constexpr (NB == 8)
    asm volatile("" : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]), "+a"(c[4]), "+a"(c[5]), "+a"(c[6]), "+a"(c[7]));
  else
    asm volatile("" : "+a"(c[0]), "+a"(c[1]), "+a"(c[2]), "+a"(c[3]));
}

template <int ROWS>
struct BigShape {
  static constexpr int WM = ROWS >= 128 ? 2 : 1, WN = 4 / WM;        // waves
  static constexpr int MB = ROWS / 16 / WM, NB = TB / 16 / WN;       // a wave's 16 x 16 blocks
  static constexpr int ST = ROWS == 256 ? 2 : 3;                     // steps resident
  static constexpr uint32_t kA = ROWS * KB * 2, kB = TB * KB * 2, kStage = kA + kB;
  static constexpr int LA = ROWS / 32, LB = 8, NL = LA + LB;         // DMAs per wave and step
  static constexpr uint32_t kOutRow = 16 * NB * 2 + 16;              // a wave's staged output row
  static constexpr uint32_t kOutRows = ROWS == 128 ? 8 : 16;         // staged at a time
  static constexpr uint32_t kOut = ST * kStage;                      // kOutRows of them per wave
  static constexpr uint32_t kMeta = kOut + 4 * kOutRows * kOutRow;   // per row: two tiles' targets, lse, mantissas
  static constexpr uint32_t kLds = kMeta + 2 * ROWS * 12;
  static_assert(kLds <= 160 * 1024, "LDS");
};

template <int ROWS, bool AT, bool BT, int EPI>
__global__ __launch_bounds__(256, 1) void loss_big_kernel(BigArgs p) {
  using S = BigShape<ROWS>;
  constexpr int MB = S::MB, NB = S::NB, ST = S::ST, LA = S::LA, LB = S::LB, NL = S::NL;
  // (kEpiTeacherStats: the waves' parts of a row beside the staged logits)
  constexpr uint32_t kParts = EPI == kEpiTeacherStats ? S::kLds : S::kOut;
  __shared__ __align__(16) uint8_t smem[S::kLds + (EPI == kEpiTeacherStats ? S::WN * ROWS * 8 : 0)];
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / S::WN, wn = wave % S::WN;
  const uint32_t lds0 = lds_addr(smem);

  // tiles: strips of 8 M tiles, M fastest, so that the 32 tiles an XCD works
  // on are 8 x 4 (each operand tile is shared by several of them in its L2);
  // the splits of a tile side by side
  const uint32_t total = p.m_tiles * p.n_tiles * p.splits, per = (total + 7) / 8, stride = gridDim.x >> 3;
  const uint32_t end = min(((blockIdx.x & 7) + 1) * per, total);
  const uint32_t all_steps = p.k / KB, per_split = (all_steps + p.splits - 1) / p.splits;
  uint32_t t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  uint32_t m0, n0, split, s0, steps;

  // ---- DMA: instruction i of a wave moves 1 KB: rows 32 i + 8 wave + (l >> 3)
  // of a rows layout, k rows 8 i + 2 wave + (l >> 5) of a columns layout
  uint32_t off_a[LA], off_b[LB];
  const uint8_t* base_a;
  const uint8_t* base_b;
  auto offset = [&](auto T, uint32_t i, uint32_t r0, uint32_t rows, uint64_t ld) __attribute__((always_inline)) {
    if constexpr (decltype(T)::value) {
      const uint32_t r = 8 * i + 2 * wave + (lane >> 5), f = (r & 3) + 4 * ((r >> 3) & 1);
      const uint32_t c = min((r0 >> 3) + ((lane & 31) ^ (2 * f)), (rows - 1) >> 3);
      return (uint32_t)(r * ld * 2) + (c << 4);
    } else {
      const uint32_t r = 32 * i + 8 * wave + (lane >> 3);
      return (uint32_t)((min(r0 + r, rows - 1) - r0) * ld * 2) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
  };
  auto source = [&](auto T, const uint8_t* base, uint64_t ld, uint32_t step) __attribute__((always_inline)) {
    return uniform_ptr(base + (decltype(T)::value ? (uint64_t)step * KB * ld * 2 : (uint64_t)step * KB * 2));
  };
  // B's part of a step: the feed-forward block's has two sources, gate's and up's
  // weights, for alternate 16 rows of a tile (each wave's DMAs read one of them)
  // or for the two halves of k
  auto offset_b = [&](uint32_t i) __attribute__((always_inline)) {
    if constexpr (has_pair(EPI)) {
      const uint32_t r = 32 * i + 8 * wave + (lane >> 3), row = 16 * i + 8 * (wave & 1) + (lane >> 3);
      return (uint32_t)((min(n0 / 2 + row, p.n / 2 - 1) - n0 / 2) * p.ldb * 2) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    } else {
      return offset(std::bool_constant<BT>{}, i, n0, p.n, p.ldb);
    }
  };
  auto source_b = [&](uint32_t step) __attribute__((always_inline)) {
    if constexpr (BT && (EPI == kEpiStore || EPI == kEpiSum)) {
      if (step >= p.b_steps) return source(std::true_type{}, reinterpret_cast<const uint8_t*>(p.b2), p.ldb, step - p.b_steps);
    }
    return source(std::bool_constant<BT>{}, base_b, p.ldb, step);
  };
  constexpr std::bool_constant<AT> at{};
  constexpr std::bool_constant<BT> bt{};
  // a step may have fewer than 64 k rows of an operand, the last one
  constexpr bool kShort = BT && (EPI == kEpiAdd || (AT && EPI == kEpiStore));
  const uint32_t k_whole = AT && EPI == kEpiStore ? min(p.a_valid, p.k_valid) : p.k_valid;
  // DMA i of a step (A's first) into buffer s; CUT: such a step.  The rows that are
  // not there are read as zeros: the other operand's are, but a repeated row that
  // holds an infinity would make NaN of them.
  auto issue = [&](const uint8_t* sa, const uint8_t* sb, uint32_t s, uint32_t i, auto CUT,
                   uint32_t step) __attribute__((always_inline)) {
    constexpr bool kCut = decltype(CUT)::value;
    const uint32_t lds = lds0 + s * S::kStage + wave * 1024;
    auto source_of = [&](const uint8_t* base, uint32_t off, uint32_t i, uint32_t valid) __attribute__((always_inline)) {
      const uint32_t row = step * KB + 8 * i + 2 * wave + (lane >> 5);
      return row < valid ? base + off : reinterpret_cast<const uint8_t*>(&kNoRow);
    };
    if (i < (uint32_t)LA) {
      if constexpr (kCut && AT) dma16v(source_of(sa, off_a[i], i, p.a_valid), lds + i * 4096);
      else dma16(sa, off_a[i], lds + i * 4096);
    } else {
      i -= LA;
      // (few rows: the weights past the caches.  Of one row tile they are read
      // once: dx of 33 rows over 151936 x 1024 92 -> 72 us, the loss of 128 rows
      // 84 -> 79.  With two or three row tiles it still gains: the loss of 300
      // rows 150 -> 135 there, 435 -> 392 over 129280 x 4096, of 200 rows over
      // 32768 x 1024 26 -> 25; the other way dx of 128 rows there, 60 -> 67)
      if constexpr (kCut) dma16v(source_of(sb, off_b[i], i, p.k_valid), lds + S::kA + i * 4096);
      else if constexpr (ROWS <= 128) dma16nt(sb, off_b[i], lds + S::kA + i * 4096);
      else dma16(sb, off_b[i], lds + S::kA + i * 4096);
    }
  };
  // kEpiTeacherStats: of row tid of the tile the first and the end of its listed
  // columns (low and high half), and the first two of them
  uint32_t range = 0, key0 = 0, key1 = 0;
  // tile t and its first steps sent for; its rows' targets, log-sum-exps and
  // mantissas into half `which` of the panel (kNoTarget for every row whose g is 0)
  auto start = [&](uint32_t which) __attribute__((always_inline)) {
    split = t % p.splits;
    const uint32_t u = t / p.splits, strip = u / (8 * p.n_tiles), in_strip = u % (8 * p.n_tiles);
    const uint32_t high = min(8u, p.m_tiles - strip * 8);
    m0 = (strip * 8 + in_strip % high) * ROWS;
    n0 = in_strip / high * TB;
    s0 = min(split * per_split, all_steps);
    steps = min(s0 + per_split, all_steps) - s0;
    base_a = reinterpret_cast<const uint8_t*>(AT ? p.a : p.a + m0 * p.lda);
    if constexpr (has_pair(EPI)) base_b = reinterpret_cast<const uint8_t*>((wave & 2 ? p.b2 : p.b) + n0 / 2 * p.ldb);
    else base_b = reinterpret_cast<const uint8_t*>(BT ? p.b : p.b + n0 * p.ldb);
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)LA; ++i) off_a[i] = offset(at, i, m0, p.m, p.lda);
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)LB; ++i) off_b[i] = offset_b(i);
#pragma unroll
    for (uint32_t q = 0; q < (uint32_t)ST; ++q) {
      if (q >= steps) break;
      const uint8_t* sa = source(at, base_a, p.lda, s0 + q);
      const uint8_t* sb = source_b(s0 + q);
      auto all = [&](auto CUT) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t i = 0; i < (uint32_t)NL; ++i) issue(sa, sb, q, i, CUT, s0 + q);
      };
      if (kShort && (s0 + q + 1) * KB > k_whole) all(std::bool_constant<kShort>{});
      else all(std::false_type{});
    }
    if constexpr (EPI == kEpiStats || has_grad(EPI)) {
      if (tid < ROWS) {
        const uint32_t row = m0 + tid;
        uint32_t* const meta = reinterpret_cast<uint32_t*>(smem + S::kMeta + which * ROWS * 12);
        const uint32_t y = row < p.m ? p.target[row] : kNoTarget;
        meta[tid] = y < p.vocab ? y : kNoTarget;
        if constexpr (has_grad(EPI)) {
          meta[ROWS + tid] = __float_as_uint(row < p.m ? p.lse[row] : 0.0f);
          meta[2 * ROWS + tid] = __float_as_uint(row < p.m ? p.mantissa[row] : 1.0f);
        }
      }
    }
    if constexpr (EPI == kEpiTeacherStats) {
      range = 0;
      if (p.before && tid < ROWS && m0 + tid < p.m) {
        const uint16_t* const b = p.before + (uint64_t)(m0 + tid) * (p.n_tiles + 1) + n0 / TB;
        range = b[0] | (uint32_t)b[1] << 16;
      }
    }
  };

  // ---- fragments: 16 rows of the wave's, half q of the step
  auto frag = [&](auto T, uint32_t stage, uint32_t first, uint32_t q) __attribute__((always_inline)) -> v4i {
    const uint8_t* const from = smem + stage;
    if constexpr (decltype(T)::value) {
      const uint32_t r = 32 * q + 8 * lg + (lr >> 2), f = (lr >> 2) + 4 * (lg & 1);
      const uint8_t* const x = from + r * 512 + ((2 * first + 8 * (lr & 3)) ^ (32 * f));
      return join(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)x),
                  __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(x + 4 * 512)));
    } else {
      return *reinterpret_cast<const v4i*>(from + (first + lr) * 128 + (((4 * q + lg) ^ ((lr >> 1) & 7)) << 4));
    }
  };
  v4f acc[MB][NB];
  v4i fa[2][MB], fb[2][NB];
  // the fragments of a half, three or four beside each group of NB MFMAs: B's
  // first, which the next half's first group needs, and all of them a group or
  // two early (kLate: of the next step where two are resident, beside the last half
  // of the groups)
  constexpr uint32_t kLate = (MB + NB) / (MB / 2);
  constexpr uint32_t kReads = (MB + NB + MB - 2) / (MB - 1);
  auto read_one = [&](uint32_t s, uint32_t q, int to, uint32_t i) __attribute__((always_inline)) {
    if (i < (uint32_t)NB) fb[to][i] = frag(bt, s * S::kStage + S::kA, wn * NB * 16 + 16 * i, q);
    else if (i < (uint32_t)(NB + MB)) fa[to][i - NB] = frag(at, s * S::kStage, wm * MB * 16 + 16 * (i - NB), q);
  };
  // NB MFMAs, with beside(j) issued while MFMA j runs
  auto multiply = [&](int from, uint32_t i, auto&& beside) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, fb[from][j]),
                                                          __builtin_bit_cast(v8bf, fa[from][i]), acc[i][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
      beside((uint32_t)j);
      __builtin_amdgcn_sched_barrier(0);
    }
    pin(acc[i]);
  };
  uint32_t s;  // the buffer of the step being multiplied
  // kNext: the next step exists, with kLeft further steps in flight behind it;
  // kMore: step j + ST exists and is sent for (CUT: it is cut short)
  auto body = [&](uint32_t j, auto NEXT, auto LEFT, auto MORE, auto CUT) __attribute__((always_inline)) {
    constexpr bool kNext = decltype(NEXT)::value, kMore = decltype(MORE)::value;
    const uint32_t ns = s + 1 == ST ? 0 : s + 1;
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)MB; ++i) {
      multiply(0, i, [&](uint32_t j) __attribute__((always_inline)) {
        if (j < kReads) read_one(s, 1, 1, kReads * i + j);
      });
    }
    // this step read by this wave (and three resident: the next one arrived for it;
    // the first ST had before the tile was begun); then by all
    __builtin_amdgcn_s_waitcnt(kLdsRead);
    if (ST != 2 && j + 1 >= (uint32_t)ST) __builtin_amdgcn_s_waitcnt(vmcnt_at_most(decltype(LEFT)::value * NL));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint32_t step = s0 + j + ST;
    const uint8_t* sa = nullptr;
    const uint8_t* sb = nullptr;
    if constexpr (kMore) {
      sa = source(at, base_a, p.lda, step);
      sb = source_b(step);
    }
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)MB; ++i) {
      if constexpr (kNext && ST == 2) {
        if (i == MB / 2) {
          // the next step arrived for this wave (half of the one after it is sent
          // for), then for all
          if (j + 1 >= (uint32_t)ST) __builtin_amdgcn_s_waitcnt(vmcnt_at_most(kMore ? NL / 2 : 0));
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
        }
      }
      multiply(1, i, [&](uint32_t j) __attribute__((always_inline)) {
        if constexpr (kNext) {
          if constexpr (ST == 2) {
            if (i >= MB / 2 && j < kLate) read_one(ns, 0, 0, kLate * (i - MB / 2) + j);
          } else {
            if (j < kReads) read_one(ns, 0, 0, kReads * i + j);
          }
        }
        if constexpr (kMore) {
          // (DMAs behind the reads, MFMAs between them)
          const uint32_t first = i * NL / MB, count = (i + 1) * NL / MB - first;
#pragma unroll
          for (uint32_t e = 0; e < count; ++e)
            if (j == min(kReads + 2 * e, (uint32_t)NB - 1))
              issue(sa, sb, s, first + e, CUT, step);
        }
      });
    }
    s = ns;
  };
  constexpr std::true_type yes;
  constexpr std::false_type no;
  constexpr std::integral_constant<int, 0> none;
  constexpr std::integral_constant<int, ST - 2> full;

  // (on their way beside the K loop)
  auto fetch_keys = [&]() __attribute__((always_inline)) {
    if (EPI == kEpiTeacherStats && p.before) {
      const uint32_t from = range & 0xffffu, count = (range >> 16) - from;
      const uint32_t* const list = p.sorted + (uint64_t)(m0 + tid) * p.top_k + from;
      key0 = count > 0 ? list[0] : 0u;
      key1 = count > 1 ? list[1] : 0u;
    }
  };
  if (t >= end) return;
  uint32_t which = 0;
  start(which);
  fetch_keys();
  // a tile's first steps have arrived before it is begun; for the tiles after
  // the first that is waited for ahead of the results' stores, which so drain
  // while the next tile is multiplied (behind them, by the stores' count, took as
  // long); of kEpiStats and kEpiTeacherStats after the exponentials (the divergence of
  // 33 rows over 151936 x 1024 69.3 -> 68.0 us)
  auto arrived = []() __attribute__((always_inline)) { __builtin_amdgcn_s_waitcnt(vmcnt_at_most(0)); };
  arrived();
  while (true) {
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < MB; ++i) pin(acc[i]);
    __builtin_amdgcn_s_waitcnt(kLdsRead);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (steps) {
      s = 0;
#pragma unroll
      for (uint32_t i = 0; i < (uint32_t)(MB + NB); ++i) read_one(0, 0, 0, i);
      uint32_t j = 0;
#pragma unroll 1
      for (; j + ST + (kShort && (s0 + steps) * KB > k_whole ? 1 : 0) < steps; ++j) body(j, yes, full, yes, no);
      if constexpr (kShort)
        if (j + ST < steps) body(j++, yes, full, yes, yes);
      if constexpr (ST == 3)
        if (j + 2 < steps) body(j++, yes, std::integral_constant<int, 1>{}, no, no);
      if (j + 1 < steps) body(j++, yes, none, no, no);
      body(j, no, none, no, no);
    }
    const uint32_t cm = m0, cn = n0, csplit = split, listed = range;
    const uint32_t* const meta = reinterpret_cast<const uint32_t*>(smem + S::kMeta + which * ROWS * 12);
    const bool more = t + stride < end;
    which ^= 1;
    if (more) {
      // (every wave is past the barrier after its last read of a buffer)
      t += stride;
      start(which);
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) pin(acc[i]);

    // ---- results: acc[i][j][e] is row 16 i + lr, column 16 j + 4 lg + e of
    // the wave's part
    if constexpr (!has_grad(EPI) && !has_stats(EPI)) arrived();
    const uint32_t lrow = wm * MB * 16, wrow = cm + lrow, wcol = cn + wn * NB * 16;
    const float exponent = EPI == kEpiTeacherStats || has_teacher_grad(EPI) ? p.exponent : kLog2e;
    if constexpr (has_stats(EPI)) {
      // [column part][row]: maximum and sum
      float2* const parts = reinterpret_cast<float2*>(smem + kParts);
      static_assert(S::WN * ROWS * 8 <= 4 * S::kOutRows * S::kOutRow, "parts");
      const bool whole = cn + TB <= p.n;
      uint32_t* const lists = reinterpret_cast<uint32_t*>(smem + S::kMeta);  // [range, first, second][ROWS]
      if (EPI == kEpiTeacherStats && p.before) {
        if (tid < ROWS) {
          lists[tid] = listed;
          lists[ROWS + tid] = key0;
          lists[2 * ROWS + tid] = key1;
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        v4f (&l)[NB] = acc[i];
        if (EPI == kEpiTeacherStats && p.before) {
          // the row's listed columns: 16 or 8 rows x half of the wave's columns at a
          // time through its LDS, where the four lanes of a row take theirs in turn
          const uint32_t at_row = lrow + 16 * i + lr, mine = lists[at_row], from = mine & 0xffffu, count = (mine >> 16) - from;
          if (__builtin_amdgcn_ballot_w64(count != 0)) {
            const uint64_t list = (uint64_t)(cm + at_row) * p.top_k;
            uint8_t* const st = smem + S::kOut + wave * S::kOutRows * S::kOutRow;
#pragma unroll
            for (uint32_t r0 = 0; r0 < 16; r0 += S::kOutRows) {
              uint8_t* const row = st + (lr - r0) * S::kOutRow;
              const bool staged = lr - r0 < S::kOutRows;
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                if (staged) {
#pragma unroll
                  for (int j = 0; j < NB / 2; ++j) *reinterpret_cast<v4f*>(row + j * 64 + lg * 16) = l[half * NB / 2 + j];
                }
                wave_lds_order();
                for (uint32_t h = lg; staged && h < count; h += 4) {
                  const uint32_t k = h < 2 ? lists[(h + 1) * ROWS + at_row] : p.sorted[list + from + h];
                  const uint32_t place = (k >> 8) - (wcol + half * 8 * NB);
                  if (place < 8u * NB) p.logits[list + (k & 0xffu)] = *reinterpret_cast<const float*>(row + place * 4);
                }
                wave_lds_order();
              }
            }
          }
        }
        if (!whole) {
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (wcol + 16 * j + 4 * lg + e >= p.n) l[j][e] = -INFINITY;
        }
        if constexpr (EPI == kEpiStats) {
          const uint32_t target = meta[lrow + 16 * i + lr], place = target - wcol;
          if (place < 16u * NB && ((place >> 2) & 3) == lg && target < p.n) {
            float v = 0.0f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) v = (uint32_t)j == place >> 4 && (uint32_t)e == (place & 3) ? l[j][e] : v;
            p.target_logit[wrow + 16 * i + lr] = v;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j)
          top = fmaxf(top, fmaxf(fmaxf(l[j][0], l[j][1]), fmaxf(l[j][2], l[j][3])));
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float from = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          float part = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) part += __builtin_amdgcn_exp2f((l[j][e] - from) * exponent);
          sum += part;
        }
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lg == 0) parts[wn * ROWS + lrow + 16 * i + lr] = float2{top, sum};
      }
      __syncthreads();
      if (tid < ROWS && cm + tid < p.m) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < S::WN; ++w) top = fmaxf(top, parts[w * ROWS + tid].x);
#pragma unroll
        for (int w = 0; w < S::WN; ++w) {
          const float2 x = parts[w * ROWS + tid];
          sum += x.x == -INFINITY ? x.y : x.y * __builtin_amdgcn_exp2f((x.x - top) * exponent);
        }
        p.stats[(uint64_t)(cm + tid) * p.n_tiles + cn / TB] = float2{top, sum};
      }
    } else if constexpr (EPI == kEpiAdd || EPI == kEpiSum || EPI == kEpiGluSum) {
      float* const out = static_cast<float*>(p.out) + csplit * p.split_stride + wcol + 4 * lg;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const uint32_t row = wrow + 16 * i + lr;
        v4f* const o = reinterpret_cast<v4f*>(out + (uint64_t)min(row, p.m - 1) * p.ldo);
        v4f before[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          before[j] = v4f{0.f, 0.f, 0.f, 0.f};
          if (EPI == kEpiAdd && !p.first && wcol + 16 * j + 4 * lg < p.n) before[j] = o[4 * j];
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
          if (row < p.m && wcol + 16 * j + 4 * lg < p.n) o[4 * j] = before[j] + acc[i][j];
        // (16 rows at a time: registers for no more)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
    } else if constexpr (EPI == kEpiStore || EPI == kEpiGlu || EPI == kEpiGluGrad) {
      // 16 rows of BLOCKS 16-column blocks in bf16 through the wave's own LDS,
      // so that a store instruction writes whole lines
      uint8_t* const st = smem + S::kOut + wave * S::kOutRows * S::kOutRow;
      auto put = [&](auto BLOCKS, auto&& value, auto&& row_at, uint32_t row0, uint32_t col0, uint32_t rows,
                     uint32_t cols) __attribute__((always_inline)) {
        constexpr uint32_t kBlocks = decltype(BLOCKS)::value, kLanes = 2 * kBlocks;
        constexpr uint32_t kRowsAt = 64 / kLanes < S::kOutRows ? 64 / kLanes : S::kOutRows;
#pragma unroll
        for (uint32_t r0 = 0; r0 < 16; r0 += S::kOutRows) {
          if (lr - r0 < S::kOutRows) {
#pragma unroll
            for (uint32_t j = 0; j < kBlocks; ++j) {
              const v4f v = value(j);
              *reinterpret_cast<uint2*>(st + (lr - r0) * S::kOutRow + j * 32 + lg * 8) =
                  uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
            }
          }
          wave_lds_order();
#pragma unroll
          for (uint32_t h = 0; h < S::kOutRows / kRowsAt; ++h) {
            const uint32_t q = kRowsAt * h + lane / kLanes, r = row0 + r0 + q, c = col0 + 8 * (lane % kLanes);
            if (lane / kLanes >= kRowsAt) continue;
            const v4i o = *reinterpret_cast<const v4i*>(st + q * S::kOutRow + lane % kLanes * 16);
            if (r < rows && c < cols) *reinterpret_cast<v4i*>(row_at(r) + c) = o;
          }
          wave_lds_order();
        }
      };
      if constexpr (EPI == kEpiStore) {
        uint16_t* const out = static_cast<uint16_t*>(p.out);
        auto row_at = [&](uint32_t r) {
          return r < p.out_rows ? out + (uint64_t)r * p.ldo : p.out2 + (uint64_t)(r - p.out_rows) * p.ldo;
        };
#pragma unroll
        for (int i = 0; i < MB; ++i)
          put(std::integral_constant<int, NB>{}, [&](uint32_t j) { return acc[i][j]; }, row_at, wrow + 16 * i, wcol, p.m,
              p.n);
      } else if constexpr (EPI == kEpiGlu) {
        constexpr std::integral_constant<int, NB / 2> half;
        const uint32_t gcol = wcol / 2, cols = p.n / 2;
        auto plane = [&](uint16_t* base) { return [&, base](uint32_t r) { return base + (uint64_t)r * p.ldo; }; };
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if (p.gate) {
            put(half, [&](uint32_t j) { return acc[i][2 * j]; }, plane(p.gate), wrow + 16 * i, gcol, p.m, cols);
            put(half, [&](uint32_t j) { return acc[i][2 * j + 1]; }, plane(p.up), wrow + 16 * i, gcol, p.m, cols);
          }
          put(half, [&](uint32_t j) {
            v4f h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = activated(acc[i][2 * j][e], acc[i][2 * j + 1][e], p.limit);
            return h;
          }, plane(static_cast<uint16_t*>(p.out)), wrow + 16 * i, gcol, p.m, cols);
        }
      } else {
        // (the rows up to a multiple of 64 are written as zeros: the weights'
        // gradients read them)
        const uint32_t rows = (p.m + 63) / 64 * 64;
        constexpr std::integral_constant<int, NB> all;
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const uint32_t row = wrow + 16 * i + lr;
          const uint64_t at_row = (uint64_t)min(row, p.m - 1) * p.n;
          uint2 gate[NB], up[NB];
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            const uint64_t from = at_row + min(wcol + 16 * j + 4 * lg, p.n - 4);
            gate[j] = *reinterpret_cast<const uint2*>(p.gate + from);
            up[j] = *reinterpret_cast<const uint2*>(p.up + from);
          }
          v4f du[NB], h[NB];
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            const v4f g = bf16x4_to_f32(gate[j]), u = bf16x4_to_f32(up[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              GluGrad d = glu_grad(acc[i][j][e], g[e], u[e], p.limit);
              if (row >= p.m) d = GluGrad{0.0f, 0.0f, 0.0f};
              acc[i][j][e] = d.dgate;
              du[j][e] = d.dup;
              h[j][e] = d.h;
            }
          }
          uint16_t* const out = static_cast<uint16_t*>(p.out);
          put(all, [&](uint32_t j) { return acc[i][j]; }, [&](uint32_t r) { return out + (uint64_t)r * p.ldo; },
              wrow + 16 * i, wcol, rows, p.n);
          put(all, [&](uint32_t j) { return du[j]; }, [&](uint32_t r) { return out + (uint64_t)r * p.ldo + p.n; },
              wrow + 16 * i, wcol, rows, p.n);
          put(all, [&](uint32_t j) { return h[j]; }, [&](uint32_t r) { return p.h + (uint64_t)r * p.ldh; }, wrow + 16 * i,
              wcol, rows, p.n);
        }
      }
    } else {
      // bf16 through the wave's own LDS, 16 or 8 rows at a time, so that a store
      // instruction writes whole lines
      constexpr uint32_t kLanes = 2 * NB, kRowsAt = 64 / kLanes;  // lanes per row, rows per instruction
      uint8_t* const st = smem + S::kOut + wave * S::kOutRows * S::kOutRow;
      const bool whole = cn + TB <= p.n;
      const float scale = EPI == kEpiBf16 ? *p.scale : 1.0f;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        if constexpr (has_grad(EPI)) {
          const uint32_t at_row = lrow + 16 * i + lr, target = meta[at_row], place = target - p.v0 - wcol;
          const float shift = -__uint_as_float(meta[ROWS + at_row]) * kLog2e;
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], exponent, shift));
          if constexpr (EPI == kEpiTeacherGradLow) {
            // none exceeds their sum (but for the rounding of a large log-sum-exp)
            const float most = p.most[min(cm + at_row, p.m - 1)];
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][e] = at_most(acc[i][j][e], most);
          }
          if (EPI == kEpiGrad && __builtin_amdgcn_ballot_w64(place < 16u * NB)) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (place == 16u * j + 4 * lg + e) acc[i][j][e] -= 1.0f;
          }
          const float m = __uint_as_float(meta[2 * ROWS + at_row]);
          if (__builtin_amdgcn_ballot_w64(m != 1.0f)) {
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = v4f{acc[i][j][0] * m, acc[i][j][1] * m, acc[i][j][2] * m, acc[i][j][3] * m};
          }
          if (__builtin_amdgcn_ballot_w64(target == kNoTarget)) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
              if (target == kNoTarget) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
          }
          if (!whole) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (wcol + 16 * j + 4 * lg + e >= p.n) acc[i][j][e] = 0.0f;
          }
          if (i == 0) arrived();
        }
#pragma unroll
        for (uint32_t r0 = 0; r0 < 16; r0 += S::kOutRows) {
          if (lr - r0 < S::kOutRows) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
              v4f v = acc[i][j];
              if constexpr (EPI == kEpiBf16) v = v4f{v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale};
              *reinterpret_cast<uint2*>(st + (lr - r0) * S::kOutRow + j * 32 + lg * 8) =
                  uint2{f32x2_to_bf16x2(v[0], v[1]), f32x2_to_bf16x2(v[2], v[3])};
            }
          }
          wave_lds_order();
#pragma unroll
          for (uint32_t h = 0; h < S::kOutRows / kRowsAt; ++h) {
            const uint32_t q = kRowsAt * h + lane / kLanes, r = wrow + 16 * i + r0 + q, c = wcol + 8 * (lane % kLanes);
            const v4i o = *reinterpret_cast<const v4i*>(st + q * S::kOutRow + lane % kLanes * 16);
            // the rows of g up to a multiple of 64 and its columns up to the
            // tile's end are written as zeros: the products with g read them
            const bool in = has_grad(EPI) ? r < (p.m + 63) / 64 * 64 : r < p.m && c < p.n;
            if (!in) continue;
            v4i* const to = reinterpret_cast<v4i*>(static_cast<uint16_t*>(p.out) + (uint64_t)r * p.ldo + c);
            // (the weights' gradient is not read here again: past the caches,
            // 33 rows 614 -> 574 us over 129280 x 4096)
            if constexpr (EPI == kEpiBf16) __builtin_nontemporal_store(o, to);
            else *to = o;
          }
          wave_lds_order();
        }
      }
    }
    if (!more) return;
    // (hardly any stores to wait for too)
    if constexpr (has_stats(EPI)) arrived();
    fetch_keys();
  }
}

template <int ROWS, bool AT, bool BT, int EPI>
void launch_rows(BigArgs p, hipStream_t s) {
  p.m_tiles = (p.m + ROWS - 1) / ROWS;
  p.n_tiles = (p.n + TB - 1) / TB;
  if (p.splits == 0) p.splits = 1;
  const uint32_t grid = std::min((p.m_tiles * p.n_tiles * p.splits + 7) / 8 * 8, kCus);
  hipLaunchKernelGGL((loss_big_kernel<ROWS, AT, BT, EPI>), dim3(grid), dim3(256), 0, s, p);
}
inline float rows_cost(const BigArgs& p, uint32_t m, uint32_t rows) {
  return DmaRowsUs(m, p.n, p.k, std::max(p.splits, 1u), rows);
}
inline uint32_t tile_rows(const BigArgs& p, uint32_t m) {
  const float c256 = rows_cost(p, m, 256), c128 = rows_cost(p, m, 128), c64 = rows_cost(p, m, 64);
  return c64 < c128 && c64 < c256 ? 64 : c128 < c256 ? 128 : 256;
}
template <bool AT, bool BT, int EPI>
void launch_any(const BigArgs& p, hipStream_t s) {
  const uint32_t rows = tile_rows(p, p.m);
  if (rows == 64) launch_rows<64, AT, BT, EPI>(p, s);
  else if (rows == 128) launch_rows<128, AT, BT, EPI>(p, s);
  else launch_rows<256, AT, BT, EPI>(p, s);
}
// (the gradient of the weights has the vocabulary for rows: always many)
template <bool AT, bool BT, int EPI>
void launch_big(BigArgs p, hipStream_t s) {
  if constexpr (AT) {
    launch_rows<256, AT, BT, EPI>(p, s);
  } else {
    // the rows behind the last whole 256 in a launch of their own where that is
    // cheaper, although B is read once more (at 5 TB/s) and the launch costs 3
    // us: 800 rows over 151936 x 1024 309 -> 283 us; 257 rows would go 154 -> 171
    const uint32_t whole = p.m / 256 * 256, rest = p.m - whole;
    const float again = std::max(rows_cost(p, rest, tile_rows(p, rest)), (float)p.n * (float)p.k * (2.0f / 5.0e6f)) + 3.0f;
    if (whole && rest && rows_cost(p, whole, 256) + again < rows_cost(p, p.m, tile_rows(p, p.m))) {
      BigArgs q = p;
      q.m = whole;
      launch_rows<256, AT, BT, EPI>(q, s);
      p.m = rest;
      p.a += whole * p.lda;
      if constexpr (has_stats(EPI)) {
        p.stats += (uint64_t)whole * ((p.n + TB - 1) / TB);
        if constexpr (EPI == kEpiStats) {
          p.target_logit += whole;
        } else {
          p.sorted += (uint64_t)whole * p.top_k;
          if (p.before) p.before += (uint64_t)whole * ((p.n + TB - 1) / TB + 1);
          p.logits += (uint64_t)whole * p.top_k;
        }
      } else {
        p.out = static_cast<uint8_t*>(p.out) + whole * p.ldo * (EPI == kEpiAdd ? 4 : 2);
      }
      if constexpr (EPI == kEpiStats || has_grad(EPI)) p.target += whole;
      if constexpr (has_grad(EPI)) {
        p.lse += whole;
        p.mantissa += whole;
      }
      if constexpr (EPI == kEpiTeacherGradLow) p.most += whole;
    }
    launch_any<AT, BT, EPI>(p, s);
  }
}

}  // namespace
}  // namespace pih_amd
