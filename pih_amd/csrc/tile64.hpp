// A plain 64 x 64 product tile of bf16 operands in either layout and of any
// size, for shapes that the tiles fed by DMA do not take.
#pragma once

#include "device_common.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kT64 = 64, kT64Pitch = 64 + 8;
typedef uint16_t Plane64[kT64][kT64Pitch];

// 64 rows of an operand over 64 of k into LDS as [row][k], zeros outside.
// KROW: [k][row] in memory, else [row][k]; rows of memory ld elements apart,
// their length a multiple of 8.
template <bool KROW>
__device__ __forceinline__ void stage64(Plane64& s, const uint16_t* p, uint64_t ld, uint32_t r0, uint32_t rows,
                                        uint32_t k0, uint32_t k) {
  for (uint32_t i = threadIdx.x; i < kT64 * kT64 / 8; i += 256) {
    const uint32_t a = i / 8, c = i % 8 * 8;
    v4i v{0, 0, 0, 0};
    if constexpr (KROW) {
      if (k0 + a < k && r0 + c < rows) v = *reinterpret_cast<const v4i*>(p + (uint64_t)(k0 + a) * ld + r0 + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[c + e][a] = (uint16_t)((uint32_t)v[e / 2] >> (16 * (e & 1)));
    } else {
      if (r0 + a < rows && k0 + c < k) v = *reinterpret_cast<const v4i*>(p + (uint64_t)(r0 + a) * ld + k0 + c);
      *reinterpret_cast<v4i*>(&s[a][c]) = v;
    }
  }
}

struct Operand64 {
  const uint16_t* p;
  uint64_t ld;
  uint32_t rows;
};

// acc += A . B^T over k, for the block's tile at (m0, n0): four waves of 32 x
// 32.  The MFMA's first operand is B, so that a lane's four results
// acc[i][j][0..3] are columns 16 j + 4 lg + (0..3) of row 16 i + lr of the
// wave's quarter, lr = lane % 16, lg = lane / 16.
template <bool AK, bool BK>
__device__ __forceinline__ void multiply64(Plane64& sa, Plane64& sb, v4f (&acc)[2][2], Operand64 a, Operand64 b,
                                           uint32_t m0, uint32_t n0, uint32_t k) {
  const uint32_t lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  const uint32_t wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  for (uint32_t k0 = 0; k0 < k; k0 += kT64) {
    stage64<AK>(sa, a.p, a.ld, m0, a.rows, k0, k);
    stage64<BK>(sb, b.p, b.ld, n0, b.rows, k0, k);
    __syncthreads();
#pragma unroll
    for (uint32_t q = 0; q < kT64; q += 32) {
      v4i fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *reinterpret_cast<const v4i*>(&sa[wm + 16 * i + lr][q + 8 * lg]);
        fb[i] = *reinterpret_cast<const v4i*>(&sb[wn + 16 * i + lr][q + 8 * lg]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, fb[j]),
                                                              __builtin_bit_cast(v8bf, fa[i]), acc[i][j], 0, 0, 0);
    }
    __syncthreads();
  }
}

// f(row, column, i, j) for each of a lane's results acc[i][j], four columns from `column` on
template <typename F>
__device__ __forceinline__ void each64(uint32_t m0, uint32_t n0, F&& f) {
  const uint32_t lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  const uint32_t wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) f(m0 + wm + 16 * i + lr, n0 + wn + 16 * j + 4 * lg, i, j);
}

}  // namespace
}  // namespace pih_amd
