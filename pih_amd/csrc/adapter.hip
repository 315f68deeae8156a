// Low-rank adapters of many requests on top of a shared projection, for
// gfx950: out = base + s_a (x A_a^T) B_a^T for the rows of every segment (a
// request's rows, with an adapter a), and the gradients
//   dx = base + dh A_a,  da = dh^T x,  db = dy^T h
//   with  h = s_a x A_a^T,  dh = s_a dy B_a   (rank <= 128 columns).
//
// Two launches forward.  The first ("down") multiplies a 16-row tile of a
// segment with A and leaves fp32 sums [split][row][rank]: K is split over
// the blocks until they fill the card, since a decode batch has few rows.
// The second ("up") adds the splits, scales, and multiplies with B on top of
// base.  Tiles never cross a segment, so a tile has one adapter and no row
// permutation is needed; a tile finds its segment by a wave scan over the
// offsets.  The product between the two stays fp32 up to the second MFMA,
// which takes it as two bf16 values hi + lo (2^-16 of the value at most is
// lost): twice the MFMAs of a product that is bound by bytes, and the output
// is off by its own rounding only.
//
// The backward runs both downs (x A^T and dy B) in one launch, then sums the
// splits once, into [row][rank] for the up product with A and into bf16 hi
// and lo with the rows innermost for the gradients of A and B, whose
// contraction runs over the rows.
//
// MFMA operands: the weights (or the rows' side for da) come first, so that a
// lane's four results are consecutive in memory.
#include <algorithm>

#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kMaxRank = 128;
constexpr uint32_t kMaxColumns = 1u << 20;
constexpr uint32_t TR = 16;  // rows of a tile
constexpr uint32_t kErrAdapter = 1u, kErrOffsets = 2u;
constexpr uint32_t kNoAdapter = 0xffffffffu;

struct Segments {
  const uint32_t* offsets;
  const uint32_t* adapter;
  const float* scale;
  uint32_t segments, rows, adapters;
};

struct Tile {
  uint32_t row0, rows, adapter;
  float scale;
};

// Tile `index` of the segments' 16-row tiles, in order; false past the last.
// A segment whose offsets descend or pass the rows counts as empty.
__device__ __forceinline__ bool find_tile(const Segments& p, uint32_t index, Tile& t, uint32_t* err) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t s0 = 0; s0 < p.segments; s0 += 64) {
    const uint32_t s = s0 + lane;
    uint32_t lo = 0, hi = 0;
    if (s < p.segments) {
      lo = p.offsets[s];
      hi = p.offsets[s + 1];
      if (hi < lo || hi > p.rows) {
        if (index == 0 && threadIdx.x < 64) atomicOr(err, kErrOffsets);
        hi = lo = 0;
      }
    }
    const uint32_t n = (hi - lo + TR - 1) / TR;
    uint32_t upto = n;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
      const uint32_t v = __shfl_up(upto, d, 64);
      if (lane >= d) upto += v;
    }
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if (index - before < all) {
      const uint64_t past = __builtin_amdgcn_ballot_w64(upto > index - before);
      const uint32_t l = (uint32_t)__builtin_ctzll(past);
      const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)(upto - n), l);
      const uint32_t slo = (uint32_t)__builtin_amdgcn_readlane((int)lo, l);
      const uint32_t shi = (uint32_t)__builtin_amdgcn_readlane((int)hi, l);
      t.row0 = slo + (index - before - first) * TR;
      t.rows = min(TR, shi - t.row0);
      t.adapter = p.adapter[s0 + l];
      t.scale = 1.0f;
      if (t.adapter < p.adapters) {
        if (p.scale) t.scale = p.scale[t.adapter];
      } else if (t.adapter != kNoAdapter) {
        if (threadIdx.x == 0) atomicOr(err, kErrAdapter);
      }
      return true;
    }
    before += all;
  }
  return false;
}

__device__ __forceinline__ v4i load16(const uint16_t* p) { return *reinterpret_cast<const v4i*>(p); }
__device__ __forceinline__ v4f mfma(v4i a, v4i b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// eight values `stride` elements apart, those from `count` on as 0
__device__ __forceinline__ v4i load_column(const uint16_t* p, uint64_t stride, uint32_t count) {
  v4i v{0, 0, 0, 0};
#pragma unroll
  for (uint32_t i = 0; i < 8; ++i) {
    const uint32_t e = i < count ? p[i * stride] : 0u;
    v[i / 2] |= (int)(e << (16 * (i & 1)));
  }
  return v;
}
// fp32 values as bf16 hi + lo, eight of them
__device__ __forceinline__ void split8(const float* v, v4i& hi, v4i& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t h = f32x2_to_bf16x2(v[2 * i], v[2 * i + 1]);
    const float l0 = v[2 * i] - bf16_bits_to_f32(h & 0xffffu), l1 = v[2 * i + 1] - bf16_bits_to_f32(h >> 16);
    hi[i] = (int)h;
    lo[i] = (int)f32x2_to_bf16x2(l0, l1);
  }
}

// ------------------------------------------------------------------ down
struct DownSide {
  const uint16_t* src;  // [rows][cols]
  const uint16_t* w;    // [adapters][rank][cols], or [adapters][cols][rank] (kColumns)
  float* out;           // [splits][rows][rank]
  uint32_t stride, cols, per_split, splits;
};
struct DownParams {
  Segments seg;
  DownSide side[2];
  uint32_t* err;
  uint32_t rank;
};

// One tile of rows times the rank columns of its adapter over a range of
// cols.  The four waves take 128-column pieces in turn.
template <int NJ, bool kColumns>
__device__ void down_tile(const DownParams& p, const DownSide& d, const Tile& t, uint32_t split) {
  __shared__ float sums[4][TR][NJ * 16 + 4];
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const uint32_t c0 = split * d.per_split, c1 = min(c0 + d.per_split, d.cols);
  v4f acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint16_t* const src = d.src + (uint64_t)(t.row0 + min(lr, t.rows - 1)) * d.stride;
  const uint16_t* const w = d.w + (uint64_t)t.adapter * p.rank * d.cols;
  for (uint32_t c = c0 + 128 * wave; c < c1; c += 512) {
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q) {
      const uint32_t at = c + 32 * q + 8 * lg;
      v4i x{0, 0, 0, 0};
      if (at < c1) x = load16(src + at);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint32_t row = min(16 * j + lr, p.rank - 1);
        v4i a{0, 0, 0, 0};
        if (at < c1) {
          if constexpr (kColumns) a = load_column(w + (uint64_t)at * p.rank + row, p.rank, 8);
          else a = load16(w + (uint64_t)row * d.cols + at);
        }
        acc[j] = mfma(a, x, acc[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][lr][16 * j + 4 * lg + i] = acc[j][i];
  __syncthreads();
  float* const out = d.out + ((uint64_t)split * p.seg.rows + t.row0) * p.rank;
  for (uint32_t i = tid; i < t.rows * p.rank; i += 256) {
    const uint32_t r = i / p.rank, j = i % p.rank;
    out[i] = (sums[0][r][j] + sums[1][r][j]) + (sums[2][r][j] + sums[3][r][j]);
  }
}

template <int NJ, bool kBackward>
__global__ __launch_bounds__(256) void adapter_down_kernel(DownParams p) {
  Tile t;
  const DownSide& d = p.side[blockIdx.z];
  if (blockIdx.y >= d.splits || !find_tile(p.seg, blockIdx.x, t, p.err) || t.adapter >= p.seg.adapters) return;
  if constexpr (kBackward) {
    if (blockIdx.z) {
      down_tile<NJ, true>(p, d, t, blockIdx.y);
      return;
    }
  }
  down_tile<NJ, false>(p, d, t, blockIdx.y);
}

// -------------------------------------------------------------------- up
struct UpParams {
  Segments seg;
  const float* h;       // [splits][rows][rank]
  const uint16_t* w;    // [adapters][cols][rank], or [adapters][rank][cols] (kColumns)
  const uint16_t* base;
  uint16_t* out;
  uint32_t* err;
  uint32_t splits, rank, cols, base_stride, out_stride, groups;  // groups of 64 columns per wave
  uint32_t scaled;      // h holds the scale
};

// out rows of a tile: 64 columns at a time per wave.  Row rho of MFMA u holds
// column 16 (rho >> 2) + 4 u + (rho & 3), so that a lane's results over the
// four are 16 consecutive columns.
template <int KJ, bool kColumns>
__global__ __launch_bounds__(256) void adapter_up_kernel(UpParams p) {
  __shared__ float hs[TR][KJ * 32 + 4];
  Tile t;
  if (!find_tile(p.seg, blockIdx.x, t, p.err)) return;
  if (t.adapter >= p.seg.adapters && t.adapter != kNoAdapter) return;
  const bool live = t.adapter != kNoAdapter;
  if (!live && p.base == p.out) return;
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4, wave = tid >> 6;
  if (live) {
    const float s = p.scaled ? 1.0f : t.scale;
    for (uint32_t i = tid; i < TR * KJ * 32; i += 256) {
      const uint32_t r = i / (KJ * 32), j = i % (KJ * 32);
      float v = 0.0f;
      if (r < t.rows && j < p.rank)
        for (uint32_t q = 0; q < p.splits; ++q) v += p.h[((uint64_t)q * p.seg.rows + t.row0 + r) * p.rank + j];
      hs[r][j] = v * s;
    }
  }
  __syncthreads();
  v4i hi[KJ], lo[KJ];
#pragma unroll
  for (int q = 0; q < KJ; ++q)
    if (live) split8(&hs[lr][32 * q + 8 * lg], hi[q], lo[q]);
  const uint16_t* const w = p.w + (uint64_t)(live ? t.adapter : 0) * p.rank * p.cols;
  const uint32_t g0 = (blockIdx.y * 4 + wave) * p.groups;
  for (uint32_t g = g0; g < g0 + p.groups; ++g) {
    const uint32_t c0 = g * 64;
    if (c0 >= p.cols) return;
    const uint32_t row = t.row0 + lr;
    const bool in = lr < t.rows;
    v4i b[2];
#pragma unroll
    for (uint32_t v = 0; v < 2; ++v) {
      b[v] = v4i{0, 0, 0, 0};
      const uint32_t c = c0 + 16 * lg + 8 * v;
      if (p.base && in && c < p.cols) b[v] = load16(p.base + (uint64_t)row * p.base_stride + c);
    }
    v4f acc[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) acc[u] = v4f{0.f, 0.f, 0.f, 0.f};
    if (live) {
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t c = min(c0 + 16 * (lr >> 2) + 4 * u + (lr & 3), p.cols - 1);
#pragma unroll
        for (int q = 0; q < KJ; ++q) {
          const uint32_t j = 32 * q + 8 * lg;
          v4i x{0, 0, 0, 0};
          if (j < p.rank) {
            if constexpr (kColumns) x = load_column(w + (uint64_t)j * p.cols + c, p.cols, 8);
            else x = load16(w + (uint64_t)c * p.rank + j);
          }
          acc[u] = mfma(x, lo[q], acc[u]);
          acc[u] = mfma(x, hi[q], acc[u]);
        }
      }
    }
#pragma unroll
    for (uint32_t v = 0; v < 2; ++v) {
      const uint32_t c = c0 + 16 * lg + 8 * v;
      v4i o;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t bits = (uint32_t)b[v][i];
        const float y0 = acc[2 * v + i / 2][2 * (i & 1)], y1 = acc[2 * v + i / 2][2 * (i & 1) + 1];
        o[i] = (int)f32x2_to_bf16x2(bf16_bits_to_f32(bits & 0xffffu) + y0, bf16_bits_to_f32(bits >> 16) + y1);
      }
      // (without an adapter base goes through bit for bit, a -0 too)
      if (in && c < p.cols) *reinterpret_cast<v4i*>(p.out + (uint64_t)row * p.out_stride + c) = live ? o : b[v];
    }
  }
}

// ---------------------------------------------------- splits of a backward
struct FinishParams {
  Segments seg;
  const float* part[2];   // [splits][rows][rank]: x A^T, dy B
  float* dh;              // [rows][rank], scaled
  uint16_t* hi[2];        // [rank][row_pitch], scaled, bf16 hi ...
  uint16_t* lo[2];        // ... and lo
  uint32_t* err;
  uint32_t splits[2];
  uint32_t rank, row_pitch;
};
__global__ __launch_bounds__(256) void adapter_finish_kernel(FinishParams p) {
  Tile t;
  if (!find_tile(p.seg, blockIdx.x, t, p.err) || t.adapter >= p.seg.adapters) return;
  const uint32_t side = blockIdx.y;
  for (uint32_t i = threadIdx.x; i < TR * p.rank; i += 256) {
    const uint32_t r = i & (TR - 1), j = i / TR;
    if (r >= t.rows) continue;
    const uint64_t row = t.row0 + r;
    float v = 0.0f;
    for (uint32_t q = 0; q < p.splits[side]; ++q) v += p.part[side][((uint64_t)q * p.seg.rows + row) * p.rank + j];
    v *= t.scale;
    if (side) p.dh[row * p.rank + j] = v;
    const uint32_t h = f32_to_bf16_bits(v);
    p.hi[side][(uint64_t)j * p.row_pitch + row] = (uint16_t)h;
    p.lo[side][(uint64_t)j * p.row_pitch + row] = (uint16_t)f32_to_bf16_bits(v - bf16_bits_to_f32(h));
  }
}

// ------------------------------------------------- gradients of A and of B
struct GradSide {
  const uint16_t* src;   // [rows][cols]: x for A, dy for B
  const uint16_t* hi;    // [rank][row_pitch]
  const uint16_t* lo;
  float* out;            // [adapters][rank][cols], or (B) [adapters][cols][rank]
  float* part;           // [splits] of those when the rows are split
  uint32_t stride, cols;
};
struct GradParams {
  Segments seg;
  GradSide side[2];
  uint32_t rank, row_pitch, splits;
};

// 64 columns (16 a wave) of one adapter's gradient over its rows, in blocks
// of 32 rows at multiples of 32; with several splits, every splits-th block.
template <int NJ, bool kB>
__device__ void grad_tile(const GradParams& p, const GradSide& d, uint32_t adapter) {
  const uint32_t lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4, wave = threadIdx.x >> 6;
  const uint32_t c0 = blockIdx.x * 64 + wave * 16;
  if (c0 >= d.cols) return;
  v4f acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint32_t c = min(c0 + lr, d.cols - 1);
  uint32_t turn = 0;
  for (uint32_t s = 0; s < p.seg.segments; ++s) {
    if (p.seg.adapter[s] != adapter) continue;
    const uint32_t lo_row = p.seg.offsets[s], hi_row = p.seg.offsets[s + 1];
    if (hi_row < lo_row || hi_row > p.seg.rows) continue;
    for (uint32_t r0 = lo_row & ~31u; r0 < hi_row; r0 += 32) {
      const bool mine = turn == blockIdx.y;
      turn = turn + 1 == p.splits ? 0 : turn + 1;
      if (!mine) continue;
      const uint32_t r = r0 + 8 * lg;
      v4i src{0, 0, 0, 0};
      int mask[4];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const bool in = r + i >= lo_row && r + i < hi_row;
        const uint32_t e = in ? d.src[(uint64_t)(r + i) * d.stride + c] : 0u;
        src[i / 2] |= (int)(e << (16 * (i & 1)));
        if (i & 1) mask[i / 2] |= in ? (int)0xffff0000 : 0;
        else mask[i / 2] = in ? 0xffff : 0;
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint64_t at = (uint64_t)min(16 * j + lr, p.rank - 1) * p.row_pitch + r;
        v4i h = load16(d.hi + at), l = load16(d.lo + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          h[i] &= mask[i];
          l[i] &= mask[i];
        }
        if constexpr (kB) {
          acc[j] = mfma(l, src, acc[j]);
          acc[j] = mfma(h, src, acc[j]);
        } else {
          acc[j] = mfma(src, l, acc[j]);
          acc[j] = mfma(src, h, acc[j]);
        }
      }
    }
  }
  float* const out = p.splits > 1 ? d.part + (uint64_t)blockIdx.y * p.seg.adapters * p.rank * d.cols : d.out;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    if constexpr (kB) {
      // lane: column c0 + lr, ranks 16 j + 4 lg ..
      const uint32_t rk = 16 * j + 4 * lg;
      if (c0 + lr < d.cols && rk < p.rank)
        *reinterpret_cast<v4f*>(out + ((uint64_t)adapter * d.cols + c0 + lr) * p.rank + rk) = acc[j];
    } else {
      const uint32_t rk = 16 * j + lr, cc = c0 + 4 * lg;
      if (rk < p.rank && cc < d.cols)
        *reinterpret_cast<v4f*>(out + ((uint64_t)adapter * p.rank + rk) * d.cols + cc) = acc[j];
    }
  }
}

template <int NJ>
__global__ __launch_bounds__(256) void adapter_grad_kernel(GradParams p) {
  const uint32_t adapter = blockIdx.z >> 1;
  if (blockIdx.z & 1) grad_tile<NJ, true>(p, p.side[1], adapter);
  else grad_tile<NJ, false>(p, p.side[0], adapter);
}

// the splits of the gradients, in order
__global__ __launch_bounds__(256) void adapter_grad_reduce_kernel(const float* part, float* out, uint64_t count,
                                                                  uint32_t splits) {
  const uint64_t i = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  v4f v = *reinterpret_cast<const v4f*>(part + i);
  for (uint32_t s = 1; s < splits; ++s) v += *reinterpret_cast<const v4f*>(part + s * count + i);
  *reinterpret_cast<v4f*>(out + i) = v;
}

// ------------------------------------------------------------------ host
bool shape_ok(const AdapterArgs& a) {
  return a.rows && a.segments && a.adapters && a.rank && a.rank <= kMaxRank && a.rank % 8 == 0 && a.n && a.k &&
         a.n % 8 == 0 && a.k % 8 == 0 && a.rows <= 0x7fffffffu && a.segments <= 0x7fffffffu &&
         a.adapters <= 0x7fffu && a.n <= kMaxColumns && a.k <= kMaxColumns;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// tiles of the segments at most: every segment ends in at most one short one
uint32_t tile_bound(const AdapterArgs& a) {
  const uint64_t t = ((uint64_t)a.rows + (uint64_t)std::min(a.segments, a.rows) * (TR - 1)) / TR;
  return (uint32_t)std::min<uint64_t>(t, a.rows);
}
// K splits of the down product: up to two rounds of blocks, 256 columns each
// at least; `tiles` 16-row tiles
uint32_t down_splits(uint32_t tiles, uint32_t cols) {
  return std::max<uint32_t>(1, std::min<uint32_t>((cols + 255) / 256, 512 / std::max(tiles, 1u)));
}
uint32_t per_split(uint32_t cols, uint32_t splits) { return ((cols + splits - 1) / splits + 127) / 128 * 128; }

template <typename F>
void with_pow2(uint32_t n, F&& f) {
  if (n <= 1) f(std::integral_constant<int, 1>{});
  else if (n <= 2) f(std::integral_constant<int, 2>{});
  else if (n <= 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

template <bool kColumns>
void launch_up(UpParams p, uint32_t tiles, hipStream_t s) {
  // a wave takes several 64-column groups once the blocks fill the card
  const uint32_t all = (p.cols + 63) / 64;
  p.groups = std::max<uint32_t>(1, std::min<uint32_t>(8, (uint64_t)tiles * all / 4 / 1024));
  const dim3 grid(tiles, (all + 4 * p.groups - 1) / (4 * p.groups));
  with_pow2((p.rank + 31) / 32, [&](auto kj) {
    constexpr int KJ = decltype(kj)::value;
    if constexpr (KJ <= 4) hipLaunchKernelGGL((adapter_up_kernel<KJ, kColumns>), grid, dim3(256), 0, s, p);
  });
}

Segments segments_of(const AdapterArgs& a) {
  return Segments{a.offsets, a.adapter, a.scale, a.segments, a.rows, a.adapters};
}

struct BackwardPlan {
  uint32_t tiles, splits[2], row_pitch, grad_splits;
  uint64_t part[2], dh, hi[2], lo[2], grads[2], bytes;
};
BackwardPlan backward_plan(const AdapterArgs& a) {
  BackwardPlan p{};
  p.tiles = tile_bound(a);
  p.splits[0] = down_splits(p.tiles, a.k);
  p.splits[1] = down_splits(p.tiles, a.n);
  p.row_pitch = (a.rows + 31) / 32 * 32;
  // row splits of the gradients: two rounds of blocks, 256 rows each at least
  const uint64_t blocks = (uint64_t)a.adapters * ((a.n + 63) / 64 + (a.k + 63) / 64);
  p.grad_splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((a.rows + 255) / 256, 1024 / blocks));
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int s = 0; s < 2; ++s) p.part[s] = take((uint64_t)p.splits[s] * a.rows * a.rank * 4);
  p.dh = take((uint64_t)a.rows * a.rank * 4);
  for (int s = 0; s < 2; ++s) {
    p.hi[s] = take((uint64_t)a.rank * p.row_pitch * 2);
    p.lo[s] = take((uint64_t)a.rank * p.row_pitch * 2);
  }
  if (p.grad_splits > 1)
    for (int s = 0; s < 2; ++s) p.grads[s] = take((uint64_t)p.grad_splits * a.adapters * a.rank * (s ? a.n : a.k) * 4);
  p.bytes = at;
  return p;
}

}  // namespace

uint64_t AdapterGemmWorkspaceBytes(uint32_t rows, uint32_t rank, uint32_t k) {
  if (!rows || !rank || rank > kMaxRank || !k) return 0;
  // as many splits as segments can lead to: at least rows / 16 tiles
  return (uint64_t)down_splits((rows + TR - 1) / TR, k) * rows * rank * 4;
}

uint64_t AdapterBackwardWorkspaceBytes(const AdapterArgs& a) { return shape_ok(a) ? backward_plan(a).bytes : 0; }

St LaunchAdapterGemm(const AdapterArgs& a) {
  if (!a.x || !a.a || !a.b || !a.offsets || !a.adapter || !a.out || !a.workspace || !a.error_flag || !a.stream)
    return Invalid("adapter_gemm_null_argument");
  if (!shape_ok(a)) return Invalid("adapter_gemm_shape_invalid");
  if (a.x_stride < a.k || a.out_stride < a.n || (a.base && a.base_stride < a.n) || a.x_stride % 8 ||
      a.out_stride % 8 || (a.base && a.base_stride % 8) || (a.base == a.out && a.base_stride != a.out_stride))
    return Invalid("adapter_gemm_stride_invalid");
  if (!aligned16(a.x) || !aligned16(a.a) || !aligned16(a.b) || !aligned16(a.base) || !aligned16(a.out) ||
      !aligned4(a.scale) || !aligned4(a.offsets) || !aligned4(a.adapter) || !aligned4(a.error_flag))
    return Invalid("adapter_gemm_alignment_invalid");
  const uint32_t tiles = tile_bound(a), splits = down_splits(tiles, a.k);
  if (a.workspace_bytes < AdapterGemmWorkspaceBytes(a.rows, a.rank, a.k) || !aligned16(a.workspace))
    return Invalid("adapter_gemm_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  DownParams d{};
  d.seg = segments_of(a);
  d.side[0] = DownSide{a.x, a.a, static_cast<float*>(a.workspace), a.x_stride, a.k, per_split(a.k, splits), splits};
  d.err = a.error_flag;
  d.rank = a.rank;
  with_pow2((a.rank + 15) / 16, [&](auto nj) {
    hipLaunchKernelGGL((adapter_down_kernel<decltype(nj)::value, false>), dim3(tiles, splits), dim3(256), 0, a.stream,
                       d);
  });
  UpParams u{};
  u.seg = d.seg;
  u.h = d.side[0].out;
  u.w = a.b;
  u.base = a.base;
  u.out = a.out;
  u.err = a.error_flag;
  u.splits = splits;
  u.rank = a.rank;
  u.cols = a.n;
  u.base_stride = a.base_stride;
  u.out_stride = a.out_stride;
  launch_up<false>(u, tiles, a.stream);
  return AfterLaunch("adapter_gemm_launch_failed");
}

St LaunchAdapterBackward(const AdapterArgs& a) {
  if (!a.dy || !a.x || !a.a || !a.b || !a.offsets || !a.adapter || !a.out || !a.da || !a.db || !a.workspace ||
      !a.error_flag || !a.stream)
    return Invalid("adapter_backward_null_argument");
  if (!shape_ok(a)) return Invalid("adapter_backward_shape_invalid");
  if (a.dy_stride < a.n || a.x_stride < a.k || a.out_stride < a.k || (a.base && a.base_stride < a.k) ||
      a.dy_stride % 8 || a.x_stride % 8 || a.out_stride % 8 || (a.base && a.base_stride % 8) ||
      (a.base == a.out && a.base_stride != a.out_stride))
    return Invalid("adapter_backward_stride_invalid");
  if (!aligned16(a.dy) || !aligned16(a.x) || !aligned16(a.a) || !aligned16(a.b) || !aligned16(a.base) ||
      !aligned16(a.out) || !aligned16(a.da) || !aligned16(a.db) || !aligned4(a.scale) || !aligned4(a.offsets) ||
      !aligned4(a.adapter) || !aligned4(a.error_flag))
    return Invalid("adapter_backward_alignment_invalid");
  const BackwardPlan plan = backward_plan(a);
  if (a.workspace_bytes < plan.bytes || !aligned16(a.workspace)) return Invalid("adapter_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  auto f32 = [&](uint64_t at) { return reinterpret_cast<float*>(ws + at); };
  auto u16 = [&](uint64_t at) { return reinterpret_cast<uint16_t*>(ws + at); };
  DownParams d{};
  d.seg = segments_of(a);
  d.side[0] = DownSide{a.x,   a.a, f32(plan.part[0]), a.x_stride, a.k, per_split(a.k, plan.splits[0]), plan.splits[0]};
  d.side[1] = DownSide{a.dy,  a.b, f32(plan.part[1]), a.dy_stride, a.n, per_split(a.n, plan.splits[1]), plan.splits[1]};
  d.err = a.error_flag;
  d.rank = a.rank;
  with_pow2((a.rank + 15) / 16, [&](auto nj) {
    hipLaunchKernelGGL((adapter_down_kernel<decltype(nj)::value, true>),
                       dim3(plan.tiles, std::max(plan.splits[0], plan.splits[1]), 2), dim3(256), 0, a.stream, d);
  });
  FinishParams f{};
  f.seg = d.seg;
  f.dh = f32(plan.dh);
  for (int s = 0; s < 2; ++s) {
    f.part[s] = d.side[s].out;
    f.splits[s] = plan.splits[s];
    f.hi[s] = u16(plan.hi[s]);
    f.lo[s] = u16(plan.lo[s]);
  }
  f.err = a.error_flag;
  f.rank = a.rank;
  f.row_pitch = plan.row_pitch;
  hipLaunchKernelGGL(adapter_finish_kernel, dim3(plan.tiles, 2), dim3(256), 0, a.stream, f);
  UpParams u{};
  u.seg = d.seg;
  u.h = f.dh;
  u.w = a.a;
  u.base = a.base;
  u.out = a.out;
  u.err = a.error_flag;
  u.splits = 1;
  u.rank = a.rank;
  u.cols = a.k;
  u.base_stride = a.base_stride;
  u.out_stride = a.out_stride;
  u.scaled = 1;
  launch_up<true>(u, plan.tiles, a.stream);
  GradParams g{};
  g.seg = d.seg;
  g.rank = a.rank;
  g.row_pitch = plan.row_pitch;
  g.splits = plan.grad_splits;
  // da = dh^T x, db = dy^T h
  g.side[0] = GradSide{a.x, f.hi[1], f.lo[1], a.da, f32(plan.grads[0]), a.x_stride, a.k};
  g.side[1] = GradSide{a.dy, f.hi[0], f.lo[0], a.db, f32(plan.grads[1]), a.dy_stride, a.n};
  with_pow2((a.rank + 15) / 16, [&](auto nj) {
    hipLaunchKernelGGL((adapter_grad_kernel<decltype(nj)::value>),
                       dim3((std::max(a.n, a.k) + 63) / 64, plan.grad_splits, 2 * a.adapters), dim3(256), 0, a.stream,
                       g);
  });
  if (plan.grad_splits > 1)
    for (int s = 0; s < 2; ++s) {
      const uint64_t count = (uint64_t)a.adapters * a.rank * (s ? a.n : a.k);
      hipLaunchKernelGGL(adapter_grad_reduce_kernel, dim3((uint32_t)((count / 4 + 255) / 256)), dim3(256), 0, a.stream,
                         g.side[s].part, s ? a.db : a.da, count, plan.grad_splits);
    }
  return AfterLaunch("adapter_backward_launch_failed");
}

}  // namespace pih_amd
