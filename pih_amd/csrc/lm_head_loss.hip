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
// Measured: 4096 rows, 129280 x 4096 3.12-3.28 ms (1.32-1.39 PFLOP/s; a library
// product of that shape alone 3.25 ms) and 9.7-10.1 ms for the gradients, bound
// by the matrix pipe, 68 % busy, and the power it takes (1.9 GHz); 33 rows, 151936
// x 1024 64.5 us, of which the weights' 311 MB take 61 at 5.1 TB/s; the gradients
// of 1021 rows there 0.99 ms (0.96 PFLOP/s: of a 256 x 256 tile's 32 us 9 are the
// exponentials and the stores).  dx alone, for a frozen head: 33 rows 148 us over
// 151936 x 1024 and 373 over 129280 x 4096 (the weights twice from HBM), 4096 rows
// 6.6 ms over 129280 x 4096 (1.32 PFLOP/s).
//
// Rows without a target take no part in the gradients: their g is 0, and the
// x of dw's product is a copy with those rows as zeros, so that nothing an
// unused row holds (infinities, NaN) reaches dw.
#include <algorithm>
#include <type_traits>

#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kNoTarget = 0xffffffffu;
constexpr uint32_t kErrTarget = 1u, kErrLoss = 4u;
constexpr uint32_t TS = 64, KS = 64, kPitch = KS + 8;

typedef uint16_t Tile16[TS][kPitch];

enum : int { kEpiStats = 0, kEpiGrad = 1, kEpiBf16 = 2, kEpiAdd = 3 };

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
      // (rows and columns past the last up to the tile's end are read as zeros
      // by the products with g)
      float g = 0.0f;
      if (row < p.m && col < p.n) {
        const uint32_t target = p.target[row], at = p.v0 + col;
        if (target < p.vocab) g = p.mantissa[row] * (expf(v - p.lse[row]) - (target == at ? 1.0f : 0.0f));
      }
      static_cast<uint16_t*>(p.out)[(uint64_t)row * p.ldo + col] = (uint16_t)f32_to_bf16_bits(g);
    }
  }
}

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
// sent for, into the buffer just freed.  A block per CU walks its tiles; the
// next tile's first steps are sent for before the results of this one are
// worked on.
constexpr uint32_t TB = 256, KB = 64;

struct BigArgs {
  const uint16_t* a;
  const uint16_t* b;
  uint32_t m, n, k;        // k a multiple of 64
  uint32_t k_valid;        // columns layout of B: k rows that exist (the others repeat the last)
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
  __shared__ __align__(16) uint8_t smem[S::kLds];
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
  constexpr std::bool_constant<AT> at{};
  constexpr std::bool_constant<BT> bt{};
  // DMA i of a step (A's first) into buffer s
  auto issue = [&](const uint8_t* sa, const uint8_t* sb, uint32_t s, uint32_t i, bool short_b,
                   uint32_t step) __attribute__((always_inline)) {
    const uint32_t lds = lds0 + s * S::kStage + wave * 1024;
    if (i < (uint32_t)LA) {
      dma16(sa, off_a[i], lds + i * 4096);
    } else {
      i -= LA;
      uint32_t ob = off_b[i];
      if constexpr (BT) {
        if (short_b) {
          // k rows past the last repeat it (their factors in A are 0)
          const uint32_t r = 8 * i + 2 * wave + (lane >> 5), last = p.k_valid - 1 - step * KB;
          if (r > last) ob -= (uint32_t)((r - last) * p.ldb * 2);
        }
      }
      // (few rows: the weights past the caches.  Of one row tile they are read
      // once: dx of 33 rows over 151936 x 1024 92 -> 72 us, the loss of 128 rows
      // 84 -> 79.  With two or three row tiles it still gains: the loss of 300
      // rows 150 -> 135 there, 435 -> 392 over 129280 x 4096, of 200 rows over
      // 32768 x 1024 26 -> 25; the other way dx of 128 rows there, 60 -> 67)
      if constexpr (ROWS <= 128) dma16nt(sb, ob, lds + S::kA + i * 4096);
      else dma16(sb, ob, lds + S::kA + i * 4096);
    }
  };
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
    base_b = reinterpret_cast<const uint8_t*>(BT ? p.b : p.b + n0 * p.ldb);
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)LA; ++i) off_a[i] = offset(at, i, m0, p.m, p.lda);
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)LB; ++i) off_b[i] = offset(bt, i, n0, p.n, p.ldb);
#pragma unroll
    for (uint32_t q = 0; q < (uint32_t)ST; ++q) {
      if (q >= steps) break;
      const uint8_t* sa = source(at, base_a, p.lda, s0 + q);
      const uint8_t* sb = source(bt, base_b, p.ldb, s0 + q);
      const bool short_b = BT && (s0 + q + 1) * KB > p.k_valid;
#pragma unroll
      for (uint32_t i = 0; i < (uint32_t)NL; ++i) issue(sa, sb, q, i, short_b, s0 + q);
    }
    if constexpr (EPI == kEpiStats || EPI == kEpiGrad) {
      if (tid < ROWS) {
        const uint32_t row = m0 + tid;
        uint32_t* const meta = reinterpret_cast<uint32_t*>(smem + S::kMeta + which * ROWS * 12);
        const uint32_t y = row < p.m ? p.target[row] : kNoTarget;
        meta[tid] = y < p.vocab ? y : kNoTarget;
        if constexpr (EPI == kEpiGrad) {
          meta[ROWS + tid] = __float_as_uint(row < p.m ? p.lse[row] : 0.0f);
          meta[2 * ROWS + tid] = __float_as_uint(row < p.m ? p.mantissa[row] : 1.0f);
        }
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
  // two early
  constexpr uint32_t kReads = (MB + NB + MB - 2) / (MB - 1);
  auto read_one = [&](uint32_t s, uint32_t q, int to, uint32_t i) __attribute__((always_inline)) {
    if (i < (uint32_t)NB) fb[to][i] = frag(bt, s * S::kStage + S::kA, wn * NB * 16 + 16 * i, q);
    else if (i < (uint32_t)(NB + MB)) fa[to][i - NB] = frag(at, s * S::kStage, wm * MB * 16 + 16 * (i - NB), q);
  };
  auto read_group = [&](uint32_t s, uint32_t q, int to, uint32_t i) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t e = kReads * i; e < kReads * i + kReads; ++e) read_one(s, q, to, e);
  };
  auto multiply = [&](int from, uint32_t i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
      acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, fb[from][j]),
                                                          __builtin_bit_cast(v8bf, fa[from][i]), acc[i][j], 0, 0, 0);
    pin(acc[i]);
  };
  uint32_t s;  // the buffer of the step being multiplied
  // kNext: the next step exists, with kLeft further steps in flight behind it;
  // kMore: step j + ST exists and is sent for (kLast: it is the last one,
  // whose k rows may be short)
  auto body = [&](uint32_t j, auto NEXT, auto LEFT, auto MORE, auto LAST) __attribute__((always_inline)) {
    constexpr bool kNext = decltype(NEXT)::value, kMore = decltype(MORE)::value, kLast = decltype(LAST)::value;
    const uint32_t ns = s + 1 == ST ? 0 : s + 1;
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)MB; ++i) {
      // (the first MFMAs wait for every LDS read before them)
      if (i == 0) {
        multiply(0, i);
        __builtin_amdgcn_sched_barrier(0);
      }
      read_group(s, 1, 1, i);
      if (i) multiply(0, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    // this step read by this wave, the next one arrived for it (the first ST
    // had before the tile was begun); then by all
    __builtin_amdgcn_s_waitcnt(kLdsRead);
    if (j + 1 >= (uint32_t)ST) __builtin_amdgcn_s_waitcnt(vmcnt_at_most(decltype(LEFT)::value * NL));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const uint32_t step = s0 + j + ST;
    const uint8_t* sa = nullptr;
    const uint8_t* sb = nullptr;
    if constexpr (kMore) {
      sa = source(at, base_a, p.lda, step);
      sb = source(bt, base_b, p.ldb, step);
    }
#pragma unroll
    for (uint32_t i = 0; i < (uint32_t)MB; ++i) {
      if constexpr (kNext) read_group(ns, 0, 0, i);
      if constexpr (kMore) {
#pragma unroll
        for (uint32_t e = i * NL / MB; e < (i + 1) * NL / MB; ++e)
          issue(sa, sb, s, e, kLast && (step + 1) * KB > p.k_valid, step);
      }
      multiply(1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    s = ns;
  };
  constexpr std::true_type yes;
  constexpr std::false_type no;
  constexpr std::integral_constant<int, 0> none;
  constexpr std::integral_constant<int, ST - 2> full;

  if (t >= end) return;
  uint32_t which = 0;
  start(which);
  // a tile's first steps have arrived before it is begun; for the tiles after
  // the first that is waited for ahead of the results' stores, which so drain
  // while the next tile is multiplied
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
      for (; j + ST + (BT ? 1 : 0) < steps; ++j) body(j, yes, full, yes, no);
      if constexpr (BT)
        if (j + ST < steps) body(j++, yes, full, yes, yes);
      if constexpr (ST == 3)
        if (j + 2 < steps) body(j++, yes, std::integral_constant<int, 1>{}, no, no);
      if (j + 1 < steps) body(j++, yes, none, no, no);
      body(j, no, none, no, no);
    }
    const uint32_t cm = m0, cn = n0, csplit = split;
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
    if constexpr (EPI != kEpiGrad) arrived();
    const uint32_t lrow = wm * MB * 16, wrow = cm + lrow, wcol = cn + wn * NB * 16;
    constexpr float kLog2e = 1.44269504088896340736f;
    if constexpr (EPI == kEpiStats) {
      // [column part][row]: maximum and sum
      float2* const parts = reinterpret_cast<float2*>(smem + S::kOut);
      static_assert(S::WN * ROWS * 8 <= 4 * S::kOutRows * S::kOutRow, "parts");
      const bool whole = cn + TB <= p.n;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const uint32_t target = meta[lrow + 16 * i + lr];
        if (!whole) {
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (wcol + 16 * j + 4 * lg + e >= p.n) acc[i][j][e] = -INFINITY;
        }
        const uint32_t place = target - wcol;
        if (place < 16u * NB && ((place >> 2) & 3) == lg && target < p.n) {
          float v = 0.0f;
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) v = (uint32_t)j == place >> 4 && (uint32_t)e == (place & 3) ? acc[i][j][e] : v;
          p.target_logit[wrow + 16 * i + lr] = v;
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j)
          top = fmaxf(top, fmaxf(fmaxf(acc[i][j][0], acc[i][j][1]), fmaxf(acc[i][j][2], acc[i][j][3])));
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float from = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          float part = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) part += __builtin_amdgcn_exp2f((acc[i][j][e] - from) * kLog2e);
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
          sum += x.x == -INFINITY ? x.y : x.y * __builtin_amdgcn_exp2f((x.x - top) * kLog2e);
        }
        p.stats[(uint64_t)(cm + tid) * p.n_tiles + cn / TB] = float2{top, sum};
      }
    } else if constexpr (EPI == kEpiAdd) {
      float* const out = static_cast<float*>(p.out) + csplit * p.split_stride + wcol + 4 * lg;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const uint32_t row = wrow + 16 * i + lr;
        v4f* const o = reinterpret_cast<v4f*>(out + (uint64_t)min(row, p.m - 1) * p.ldo);
        v4f before[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          before[j] = v4f{0.f, 0.f, 0.f, 0.f};
          if (!p.first && wcol + 16 * j + 4 * lg < p.n) before[j] = o[4 * j];
        }
#pragma unroll
        for (int j = 0; j < NB; ++j)
          if (row < p.m && wcol + 16 * j + 4 * lg < p.n) o[4 * j] = before[j] + acc[i][j];
        // (16 rows at a time: registers for no more)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
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
        if constexpr (EPI == kEpiGrad) {
          const uint32_t at_row = lrow + 16 * i + lr, target = meta[at_row], place = target - p.v0 - wcol;
          const float shift = -__uint_as_float(meta[ROWS + at_row]) * kLog2e;
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[i][j][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, shift));
          if (__builtin_amdgcn_ballot_w64(place < 16u * NB)) {
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
            const bool in = EPI == kEpiGrad ? r < (p.m + 63) / 64 * 64 : r < p.m && c < p.n;
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
// Time (us) of m rows in tiles of `rows`: the rounds of tiles on the CUs, each a
// step's time and a tile's own beginning and end
//   256 rows 1.45 and 9,  128 rows 0.95 and 7,  64 rows 0.70 and 6.
inline float rows_cost(const BigArgs& p, uint32_t m, uint32_t rows) {
  const uint32_t splits = std::max(p.splits, 1u), steps = (p.k / KB + splits - 1) / splits;
  const uint64_t tiles = (uint64_t)((m + rows - 1) / rows) * ((p.n + TB - 1) / TB) * splits;
  const float tile = rows == 256 ? 9.0f + 1.45f * steps : rows == 128 ? 7.0f + 0.95f * steps : 6.0f + 0.70f * steps;
  return (float)((tiles + kCus - 1) / kCus) * tile;
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
      if constexpr (EPI == kEpiStats) {
        p.stats += (uint64_t)whole * ((p.n + TB - 1) / TB);
        p.target_logit += whole;
      } else {
        p.out = static_cast<uint8_t*>(p.out) + whole * p.ldo * (EPI == kEpiAdd ? 4 : 2);
      }
      if constexpr (EPI != kEpiAdd) p.target += whole;
      if constexpr (EPI == kEpiGrad) {
        p.lse += whole;
        p.mantissa += whole;
      }
    }
    launch_any<AT, BT, EPI>(p, s);
  }
}

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
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  uint16_t* const grad = reinterpret_cast<uint16_t*>(ws + plan.g);
  uint16_t* const live = reinterpret_cast<uint16_t*>(ws + plan.live);
  float* const sums = reinterpret_cast<float*>(ws + plan.sums);
  const uint32_t row_up = (a.rows + 63) / 64 * 64;
  float* const factor = reinterpret_cast<float*>(ws + plan.factor);
  float* const mantissa = reinterpret_cast<float*>(ws + plan.mantissa);
  hipLaunchKernelGGL(loss_factor_kernel, dim3(1), dim3(1024), 0, a.stream, a.loss_grad, a.target, factor, a.rows,
                     a.vocab);
  hipLaunchKernelGGL(loss_live_rows_kernel, dim3(row_up), dim3(256), 0, a.stream, a.x, a.target, a.loss_grad, factor,
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
      launch_big<false, false, kEpiGrad>(b, a.stream);
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
      launch_gemm<kEpiGrad>(g, a.stream);
    }
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
    b.splits = plan.splits;
    b.split_stride = (uint64_t)a.rows * a.hidden;
    b.first = v0 == 0;
    launch_big<false, true, kEpiAdd>(b, a.stream);
  }
  const uint64_t count = (uint64_t)a.rows * a.hidden;
  hipLaunchKernelGGL(loss_round_kernel, dim3((uint32_t)std::min<uint64_t>((count + 1023) / 1024, 1u << 20)), dim3(256), 0,
                     a.stream, sums,
                     a.target, a.loss_grad, mantissa, a.dx, a.hidden, a.vocab, count, plan.splits);
  return AfterLaunch("lm_head_loss_backward_launch_failed");
}

}  // namespace pih_amd
