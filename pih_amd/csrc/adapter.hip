// Low-rank adapters of many requests on top of a shared projection, for
// gfx950: out = base + s_a (x A_a^T) B_a^T for the rows of every segment (a
// request's rows, with an adapter a), and the gradients
//   dx = base + dh A_a,  da = dh^T x,  db = dy^T h
//   with  h = s_a x A_a^T,  dh = s_a dy B_a   (rank <= 128 columns).
//
// Two launches forward.  The first ("down") multiplies a tile of a segment's
// rows with A and leaves fp32 sums [split][row][rank]: K is split over the
// blocks until they fill the card, since a decode batch has few rows.  The
// second ("up") adds the splits, scales, and multiplies with B on top of base.
// The product between the two stays fp32 up to the second MFMA, which takes it
// as two bf16 values hi + lo (2^-16 of the value at most is lost): twice the
// MFMAs of a product that is bound by bytes, and the output is off by its own
// rounding only.  (One launch, every block with the whole product with A for
// itself: 57 requests 17.9 us of GPU time against 13.1, since a CU then takes in
// all of A.)
//
// A tile has one adapter: rows of one segment, found by a wave scan over the
// offsets, 16 or (segments of 64 rows) 64 in the product with A, 16, 32 or 64 in
// the product with B; or, where segments are a row or two, 16 rows of an adapter
// from all segments, so that the adapter is read once for them.
//
// Both products move bytes: rows of 64 columns and fewer are taken through LDS,
// so that every load and store of a wave has whole 128-byte lines (half lines
// ran at 3.3 TB/s where whole ones reach 4.9).  Measured, us of GPU time:
//   1 row, rank 16, 4096 x 4096                4.4 + 4.4   (latency)
//   57 one-row requests, 16 adapters, rank 32, 12288 x 4096   6.0 + 6.8
//   4099 rows, rank 64, 4096 x 12288           26 (4.1 TB/s) + 25 (2.7 TB/s)
//   8000 rows, rank 32, 12288 outputs          up 81 (4.9 TB/s)
//   backward, 8192 rows, rank 16, 4096 x 4096  36 (3.7 TB/s) + 5 + 30 (4.5) + 27 (4.9) + 5
//
// The backward runs both downs (x A^T and dy B) in one launch, then sums the
// splits once, into [row][rank] for the up product with A and into three bf16
// parts (all 24 bits: these gradients are fp32) for the gradients of A and B,
// whose contraction runs over the rows.
//
// MFMA operands: the weights (or the rows' side for da) come first, so that a
// lane's four results are consecutive in memory.
#include <algorithm>
#include <type_traits>

#include "device_common.hpp"
#include "kernels.hpp"

namespace pih_amd {
namespace {

constexpr uint32_t kMaxRank = 128;
constexpr uint32_t kMaxColumns = 1u << 20;
constexpr uint32_t kMaxRows = 1u << 26;      // a grid has fewer than 2^32 threads
constexpr uint32_t kMaxSegments = 1u << 16;  // every block reads the offsets
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

// Offsets that descend or pass the rows, of the segments from `from` on.
__device__ __forceinline__ void report_offsets(const Segments& p, uint32_t from, uint32_t* err) {
  for (uint32_t s = from + threadIdx.x; s < p.segments; s += blockDim.x)
    if (p.offsets[s + 1] < p.offsets[s] || p.offsets[s + 1] > p.rows) atomicOr(err, kErrOffsets);
}

// Tile `index` of the segments' tiles of `height` rows, in order; false past
// the last.  A segment whose offsets descend or pass the rows counts as empty.
// The first tile's block reports such segments among the 64 that its search
// ends in and before, with all_offsets (one launch
// of a call) also those behind.
__device__ __forceinline__ bool find_tile(const Segments& p, uint32_t height, uint32_t index, Tile& t, uint32_t* err,
                                          bool all_offsets = false) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t before = 0;
  for (uint32_t s0 = 0; s0 < p.segments; s0 += 64) {
    const uint32_t s = s0 + lane;
    uint32_t lo = 0, hi = 0, adapter = kNoAdapter;
    if (s < p.segments) {
      lo = p.offsets[s];
      hi = p.offsets[s + 1];
      adapter = p.adapter[s];
      if (hi < lo || hi > p.rows) {
        if (index == 0 && threadIdx.x < 64) atomicOr(err, kErrOffsets);
        hi = lo = 0;
      }
    }
    const uint32_t n = (hi - lo + height - 1) / height;
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
      t.row0 = slo + (index - before - first) * height;
      t.rows = min(height, shi - t.row0);
      t.adapter = (uint32_t)__builtin_amdgcn_readlane((int)adapter, l);
      t.scale = 1.0f;
      if (t.adapter < p.adapters) {
        if (p.scale) t.scale = p.scale[t.adapter];
      } else if (t.adapter != kNoAdapter) {
        if (threadIdx.x == 0) atomicOr(err, kErrAdapter);
      }
      if (all_offsets && index == 0) report_offsets(p, s0 + 64, err);
      return true;
    }
    before += all;
  }
  return false;
}

// Tiles of 16 rows with one adapter picked from all segments: where segments
// are a token or two, as in a decode batch, a tile per segment would read the
// adapter again for every one of them.  Tiles go by adapter (without one last),
// a tile's rows in the order of the segments.  Every block finds its tile by
// itself: rows per adapter counted in LDS, the adapters' tiles and then the
// adapter's rows by block scans (~2 us).
constexpr uint32_t kGroupAdapters = 1023, kGroupSegments = 2048;
struct GroupShared {
  uint32_t count[kGroupAdapters + 1];
  uint32_t wave[4];
  uint32_t adapter, tile;
  uint32_t rows[16];
};
// inclusive scan of a block's values, and their sum
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t& total, uint32_t* wave_sums) {
  const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
#pragma unroll
  for (uint32_t d = 1; d < 64; d <<= 1) {
    const uint32_t u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  if (lane == 63) wave_sums[wave] = v;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (uint32_t w = 0; w < 4; ++w) {
    if (w < wave) before += wave_sums[w];
    total += wave_sums[w];
  }
  __syncthreads();
  return v + before;
}
// Segment s: first row, rows (0 past the last and where the offsets are bad)
// and its place in count[] (`adapters` without one, kNoAdapter a bad id).
struct Segment {
  uint32_t first, rows, place;
};
__device__ __forceinline__ Segment segment_at(const Segments& p, uint32_t s, bool report, uint32_t* err) {
  Segment v{0, 0, kNoAdapter};
  if (s >= p.segments) return v;
  const uint32_t lo = p.offsets[s], hi = p.offsets[s + 1], a = p.adapter[s];
  if (hi < lo || hi > p.rows) {
    if (report) atomicOr(err, kErrOffsets);
    return v;
  }
  v = Segment{lo, hi - lo, a < p.adapters ? a : a == kNoAdapter ? p.adapters : kNoAdapter};
  if (report && v.place == kNoAdapter && v.rows) atomicOr(err, kErrAdapter);
  return v;
}
__device__ __forceinline__ bool group_tile(const Segments& p, uint32_t index, Tile& t, GroupShared& g, uint32_t* err) {
  const uint32_t tid = threadIdx.x, places = p.adapters + 1;
  for (uint32_t i = tid; i < places; i += 256) g.count[i] = 0;
  __syncthreads();
  for (uint32_t s = tid; s < p.segments; s += 256) {
    const Segment v = segment_at(p, s, index == 0, err);
    if (v.rows && v.place != kNoAdapter) atomicAdd(&g.count[v.place], v.rows);
  }
  __syncthreads();
  uint32_t before = 0;
  bool found = false;
  for (uint32_t b = 0; b < places && !found; b += 256) {
    const uint32_t n = b + tid < places ? (g.count[b + tid] + 15) / 16 : 0;
    uint32_t total;
    const uint32_t upto = block_scan(n, total, g.wave);
    const uint32_t at = index - before;
    if (at < total && at < upto && at >= upto - n) {
      g.adapter = b + tid;
      g.tile = at - (upto - n);
    }
    found = at < total;
    before += total;
  }
  if (!found) return false;
  __syncthreads();
  const uint32_t place = g.adapter, p0 = 16 * g.tile, rows = min(16u, g.count[place] - p0);
  before = 0;
  for (uint32_t s0 = 0; s0 < p.segments && before < p0 + rows; s0 += 256) {
    const Segment v = segment_at(p, s0 + tid, false, err);
    const uint32_t n = v.place == place ? v.rows : 0;
    uint32_t total;
    const uint32_t first = before + block_scan(n, total, g.wave) - n;
    for (uint32_t q = max(first, p0); q < min(first + n, p0 + rows); ++q) g.rows[q - p0] = v.first + (q - first);
    before += total;
  }
  __syncthreads();
  t = Tile{0, rows, place < p.adapters ? place : kNoAdapter, 1.0f};
  if (place < p.adapters && p.scale) t.scale = p.scale[place];
  return true;
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* lds_v4s;

__device__ __forceinline__ v4i load16(const uint16_t* p) { return *reinterpret_cast<const v4i*>(p); }
// (read once)
__device__ __forceinline__ v4i load16_once(const uint16_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p));
}
__device__ __forceinline__ v4f mfma(v4i a, v4i b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
// An operand whose contraction runs over LDS rows: lane l of 16 points at 4
// values of row l / 4 and receives value l % 4 of piece l / 4 of the four rows
// (ds_read_b64_tr_b16); x: the lane's place in rows 0-3 of its eight.
__device__ __forceinline__ v4i transposed(const uint8_t* x, uint32_t pitch) {
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)x);
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(x + 4 * pitch));
  const uint2 u = __builtin_bit_cast(uint2, a), v = __builtin_bit_cast(uint2, b);
  return v4i{(int)u.x, (int)u.y, (int)v.x, (int)v.y};
}
// A part of a value in bf16 that leaves the rest to the next: at most the
// largest bf16, so that an infinity stays in the rest (infinite parts would
// leave inf - inf), as does what a value past that number has above it.
__device__ __forceinline__ float part_of(float v) { return __builtin_amdgcn_fmed3f(v, -0x1.fep127f, 0x1.fep127f); }
// fp32 values as bf16 hi + lo, eight of them
__device__ __forceinline__ void split8(const float* v, v4i& hi, v4i& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t h = f32x2_to_bf16x2(part_of(v[2 * i]), part_of(v[2 * i + 1]));
    const float l0 = v[2 * i] - bf16_bits_to_f32(h & 0xffffu), l1 = v[2 * i + 1] - bf16_bits_to_f32(h >> 16);
    hi[i] = (int)h;
    lo[i] = (int)f32x2_to_bf16x2(l0, l1);
  }
}

// eight bf16 and as many fp32 sums, rounded once
__device__ __forceinline__ v4i added(v4i base, const float* sums) {
  const v4f y[2] = {*reinterpret_cast<const v4f*>(sums), *reinterpret_cast<const v4f*>(sums + 4)};
  v4i o;
#pragma unroll
  for (uint32_t i = 0; i < 4; ++i) {
    const uint32_t bits = (uint32_t)base[i];
    o[i] = (int)f32x2_to_bf16x2(bf16_bits_to_f32(bits & 0xffffu) + y[i / 2][2 * (i & 1)],
                                bf16_bits_to_f32(bits >> 16) + y[i / 2][2 * (i & 1) + 1]);
  }
  return o;
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

// a wave's LDS: 16 rows of 64 columns, and (kColumns) 32 rows of the weights
constexpr uint32_t kTurnPitch = 128 + 16, kTurn = 16 * kTurnPitch;
template <int NJ, bool kColumns>
constexpr uint32_t kDownWave = kTurn + (kColumns ? 32 * (NJ * 32 + 16) : 0);
// a block's: that, or the sums of its waves
template <int NJ, bool kColumns>
constexpr uint32_t kDownLds = std::max(4 * kDownWave<NJ, kColumns>, 4u * 16 * (NJ * 16 + 4) * 4);

// One tile of 16 RB rows times the rank columns of its adapter over a range
// of cols; the four waves take 128-column pieces in turn.  kColumns: 32 rows
// of the weights (one contiguous piece of memory) go through the wave's LDS
// and are read transposed.
template <int NJ, int RB, bool kColumns, typename F>
__device__ __forceinline__ void down_tile(const DownParams& p, const DownSide& d, const Tile& t, F&& row_of,
                                          uint32_t split, uint8_t* lds) {
  constexpr uint32_t kSumRow = NJ * 16 + 4;
  float* const sums = reinterpret_cast<float*>(lds);  // [4][16][kSumRow]
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t c0 = split * d.per_split, c1 = min(c0 + d.per_split, d.cols), rank = p.rank;
  v4f acc[RB][NJ];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[r][j] = v4f{0.f, 0.f, 0.f, 0.f};
  // 64 columns of 16 rows at a time: rows 8 h + (lane >> 3), 8 columns a lane,
  // so that a load has whole lines; turned in the wave's LDS to a row per lane
  const uint16_t* src[RB][2];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
      src[r][h] = d.src + (uint64_t)row_of(min(16 * r + 8 * h + (lane >> 3), t.rows - 1)) * d.stride;
  uint8_t* const turn = lds + wave * kDownWave<NJ, kColumns>;
  auto turned = [&](const v4i (&v)[2], v4i (&to)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h)
      *reinterpret_cast<v4i*>(turn + (8 * h + (lane >> 3)) * kTurnPitch + (lane & 7) * 16) = v[h];
    wave_lds_order();
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) to[q] = *reinterpret_cast<const v4i*>(turn + lr * kTurnPitch + 64 * q + 16 * lg);
    wave_lds_order();
  };
  const uint16_t* const w = d.w + (uint64_t)t.adapter * rank * d.cols;
  if constexpr (!kColumns) {
    // 128 columns together while registers hold them, else 64
    constexpr uint32_t U = NJ + RB <= 6 ? 2 : 1;
    const uint16_t* const wl = w + (uint64_t)(lane >> 3) * d.cols;
    for (uint32_t c = c0 + 128 * wave; c < c1; c += 512) {
#pragma unroll
      for (uint32_t u0 = 0; u0 < 2; u0 += U) {
        v4i x[U][RB][2], a[U][NJ][2];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint32_t at = c + 64 * (u0 + u) + 8 * (lane & 7);
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < RB; ++r) {
              x[u][r][h] = v4i{0, 0, 0, 0};
              if (at < c1) x[u][r][h] = load16(src[r][h] + at);
            }
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              // (rows past the rank repeat its last eight)
              a[u][j][h] = v4i{0, 0, 0, 0};
              if (at < c1) a[u][j][h] = load16(wl + (uint64_t)min(16u * j + 8 * h, rank - 8) * d.cols + at);
            }
          }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          if (c + 64 * (u0 + u) >= c1) break;
          v4i at[NJ][2];
#pragma unroll
          for (int j = 0; j < NJ; ++j) turned(a[u][j], at[j]);
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            v4i xt[2];
            turned(x[u][r], xt);
#pragma unroll
            for (uint32_t q = 0; q < 2; ++q)
#pragma unroll
              for (int j = 0; j < NJ; ++j) acc[r][j] = mfma(at[j][q], xt[q], acc[r][j]);
          }
        }
      }
    }
    __syncthreads();
  } else {
    // LDS rows of 2 rank + 16 bytes; 16-byte piece i of a lane is number
    // 64 i + lane of the 4 rank pieces of 32 rows
    const uint32_t pitch = 2 * rank + 16, per_row = rank / 8, pieces = 32 * per_row;
    uint8_t* const st = turn + kTurn;
    uint32_t put[NJ];
#pragma unroll
    for (int i = 0; i < NJ; ++i) {
      const uint32_t e = min(64 * i + lane, pieces - 1);
      put[i] = e / per_row * pitch + e % per_row * 16;
    }
    // (as many columns' loads together as registers hold, as above)
    constexpr int U = NJ + RB <= 6 ? 2 : 1;
    for (uint32_t c = c0 + 128 * wave; c < c1; c += 512) {
#pragma unroll
      for (uint32_t u0 = 0; u0 < 2; u0 += U) {
        v4i x[U][RB][2], m[U][2][NJ];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint32_t cu = c + 64 * (u0 + u), at = cu + 8 * (lane & 7);
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < RB; ++r) {
              x[u][r][h] = v4i{0, 0, 0, 0};
              if (at < c1) x[u][r][h] = load16(src[r][h] + at);
            }
            const uint32_t cq = cu + 32 * h, valid = cq < c1 ? min(32u, c1 - cq) * per_row : 0;
#pragma unroll
            for (int i = 0; i < NJ; ++i) {
              m[u][h][i] = v4i{0, 0, 0, 0};
              if (64u * i + lane < valid) m[u][h][i] = load16(w + (uint64_t)cq * rank + 8 * (64 * i + lane));
            }
          }
        }
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          if (c + 64 * (u0 + u) >= c1) break;
          v4i xt[RB][2];
#pragma unroll
          for (int r = 0; r < RB; ++r) turned(x[u][r], xt[r]);
#pragma unroll
          for (uint32_t q = 0; q < 2; ++q) {
#pragma unroll
            for (int i = 0; i < NJ; ++i)
              if (64u * i + lane < pieces) *reinterpret_cast<v4i*>(st + put[i]) = m[u][q][i];
            wave_lds_order();
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              const v4i a = transposed(st + (8 * lg + (lr >> 2)) * pitch + 32 * j + 8 * (lr & 3), pitch);
#pragma unroll
              for (int r = 0; r < RB; ++r) acc[r][j] = mfma(a, xt[r][q], acc[r][j]);
            }
            wave_lds_order();
          }
        }
      }
    }
    __syncthreads();
  }
  float* const out = d.out + (uint64_t)split * p.seg.rows * rank;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (16u * r >= t.rows) break;
#pragma unroll
    for (int j = 0; j < NJ; ++j) *reinterpret_cast<v4f*>(sums + (wave * 16 + lr) * kSumRow + 16 * j + 4 * lg) = acc[r][j];
    __syncthreads();
    for (uint32_t i = tid; i < min(16u, t.rows - 16 * r) * (rank / 4); i += 256) {
      const uint32_t row = i / (rank / 4), j = i % (rank / 4) * 4;
      const float* const from = sums + row * kSumRow + j;
      auto part = [&](uint32_t v) { return *reinterpret_cast<const v4f*>(from + v * 16 * kSumRow); };
      *reinterpret_cast<v4f*>(out + (uint64_t)row_of(16 * r + row) * rank + j) = (part(0) + part(1)) + (part(2) + part(3));
    }
    __syncthreads();
  }
}

// blocks of the down kernel that a CU holds, by its registers (nj: 16-column
// pieces of the rank)
constexpr int down_occupancy(int nj, int rb) {
  if (rb == 1) return nj <= 2 ? 6 : nj <= 4 ? 4 : 3;
  return nj == 1 ? 4 : nj == 2 ? 3 : nj <= 4 ? 2 : 1;
}

template <int NJ, int RB, bool kBackward>
__global__ __launch_bounds__(256, down_occupancy(NJ, RB)) void adapter_down_kernel(DownParams p) {
  __shared__ __align__(16) uint8_t lds[kDownLds<NJ, kBackward>];
  Tile t;
  const DownSide& d = p.side[blockIdx.z];
  // (a backward's finish reports all offsets: here it cost the loads' order
  // below, 34 -> 43 us for 4000 rows of rank 64 over 12288 + 4096 columns)
  if (blockIdx.y >= d.splits || !find_tile(p.seg, 16 * RB, blockIdx.x, t, p.err, !kBackward && blockIdx.y == 0) ||
      t.adapter >= p.seg.adapters)
    return;
  auto row_of = [&](uint32_t r) { return t.row0 + r; };
  if constexpr (kBackward) {
    if (blockIdx.z) {
      down_tile<NJ, RB, true>(p, d, t, row_of, blockIdx.y, lds);
      return;
    }
  }
  down_tile<NJ, RB, false>(p, d, t, row_of, blockIdx.y, lds);
}
// the same on tiles of rows from several segments
template <int NJ>
__global__ __launch_bounds__(256, down_occupancy(NJ, 1)) void adapter_down_group_kernel(DownParams p) {
  __shared__ __align__(16) uint8_t lds[kDownLds<NJ, false>];
  __shared__ GroupShared group;
  Tile t;
  if (!group_tile(p.seg, blockIdx.x, t, group, p.err) || t.adapter >= p.seg.adapters) return;
  down_tile<NJ, 1, false>(p, p.side[0], t, [&](uint32_t r) { return group.rows[r]; }, blockIdx.y, lds);
}

// -------------------------------------------------------------------- up
struct UpParams {
  Segments seg;
  const float* h;       // [splits][rows][rank]
  const uint16_t* w;    // [adapters][cols][rank], or [adapters][rank][cols] (kColumns)
  const uint16_t* base;
  uint16_t* out;
  uint32_t* err;
  uint32_t splits, rank, cols, base_stride, out_stride, groups;  // groups per wave
  uint32_t scaled;      // h holds the scale
};

// blocks of the up kernels that a CU holds, by registers and LDS (kj: 32-column
// pieces of the rank)
constexpr int up_occupancy(int kj, int rb) { return kj == 1 ? (rb == 1 ? 4 : 3) : kj == 2 ? 3 : 2; }
constexpr int tall_occupancy(int kj) { return kj == 4 ? 2 : 4; }

// out rows of a tile of 16 RB: 64 columns ("a group") at a time per wave, the
// next group's loads under way.  Row rho of MFMA u holds column
// 32 (u >> 1) + 8 (rho >> 2) + 4 (u & 1) + (rho & 3): a lane's results of two
// MFMAs are 8 consecutive columns.  kColumns: the weights' rows of the 64
// columns go through the wave's LDS and are read transposed.
template <int KJ, int RB, bool kColumns, bool kGroup>
__global__ __launch_bounds__(256, up_occupancy(KJ, RB)) void adapter_up_kernel(UpParams p) {
  static_assert(!kGroup || RB == 1, "a group's tile has 16 rows");
  constexpr uint32_t kRow = KJ * 32 + 4, kPitch = 128 + 16, kSumRow = 64 + 4;
  __shared__ __align__(16) float hs[16 * RB * kRow];
  __shared__ __align__(16) float sums[4 * 16 * kSumRow];
  __shared__ __align__(16) uint8_t staged[kColumns ? 4 * 32 * kPitch : 16];
  __shared__ std::conditional_t<kGroup, GroupShared, char> group;
  Tile t;
  if constexpr (kGroup) {
    if (!group_tile(p.seg, blockIdx.x, t, group, p.err)) return;
  } else {
    if (!find_tile(p.seg, 16 * RB, blockIdx.x, t, p.err)) return;
  }
  auto row_of = [&](uint32_t r) -> uint32_t {
    if constexpr (kGroup) return group.rows[r];
    else return t.row0 + r;
  };
  if (t.adapter >= p.seg.adapters && t.adapter != kNoAdapter) return;
  const bool live = t.adapter != kNoAdapter;
  if (!live && p.base == p.out) return;
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), rank = p.rank;
  const uint16_t* const w = p.w + (uint64_t)(live ? t.adapter : 0) * rank * p.cols;
  uint8_t* const st = staged + (kColumns ? wave * 32 * kPitch : 0);
  float* const mine = sums + wave * 16 * kSumRow;
  // base and out: rows 8 h + (lane >> 3) of 16, 8 columns a lane
  uint64_t base_row[RB][2], out_row[RB][2];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t row = row_of(min(16 * r + 8 * h + (lane >> 3), t.rows - 1));
      base_row[r][h] = (uint64_t)row * p.base_stride;
      out_row[r][h] = (uint64_t)row * p.out_stride;
    }

  struct Group {
    v4i x[KJ][4], b[RB][2];
  };
  auto load = [&](uint32_t g, Group& v) __attribute__((always_inline)) {
    const uint32_t c0 = g * 64;
#pragma unroll
    for (int q = 0; q < KJ; ++q)
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        v.x[q][u] = v4i{0, 0, 0, 0};
        if constexpr (kColumns) {
          // weight rows 32 q + 8 u + (lane >> 3), 8 columns a lane
          const uint32_t j = 32 * q + 8 * u + (lane >> 3), c = c0 + 8 * (lane & 7);
          if (j < rank && c < p.cols) v.x[q][u] = load16(w + (uint64_t)j * p.cols + c);
        } else {
          const uint32_t j = 32 * q + 8 * lg, c = c0 + 32 * (u >> 1) + 8 * (lr >> 2) + 4 * (u & 1) + (lr & 3);
          if (j < rank && c < p.cols) v.x[q][u] = load16(w + (uint64_t)c * rank + j);
        }
      }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        v.b[r][h] = v4i{0, 0, 0, 0};
        const uint32_t c = c0 + 8 * (lane & 7);
        if (p.base && c < p.cols) v.b[r][h] = load16_once(p.base + base_row[r][h] + c);
      }
  };
  v4i hi[RB][KJ], lo[RB][KJ];
  auto finish = [&](uint32_t g, Group& v) __attribute__((always_inline)) {
    const uint32_t c0 = g * 64;
    v4f acc[RB][4];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) acc[r][u] = v4f{0.f, 0.f, 0.f, 0.f};
    if (live) {
#pragma unroll
      for (int q = 0; q < KJ; ++q) {
        if constexpr (kColumns) {
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u)
            *reinterpret_cast<v4i*>(st + (8 * u + (lane >> 3)) * kPitch + 16 * (lane & 7)) = v.x[q][u];
          wave_lds_order();
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
          v4i x = v.x[q][u];
          if constexpr (kColumns)
            x = transposed(st + (8 * lg + (lr >> 2)) * kPitch + 2 * (32 * (u >> 1) + 8 * (lr & 3) + 4 * (u & 1)), kPitch);
#pragma unroll
          for (int r = 0; r < RB; ++r) {
            acc[r][u] = mfma(x, lo[r][q], acc[r][u]);
            acc[r][u] = mfma(x, hi[r][q], acc[r][u]);
          }
        }
        if constexpr (kColumns) wave_lds_order();
      }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      // through the wave's LDS, so that a load or store has whole lines
      if (live) {
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
          *reinterpret_cast<v4f*>(mine + lr * kSumRow + 32 * (u >> 1) + 8 * lg + 4 * (u & 1)) = acc[r][u];
        wave_lds_order();
      }
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t row = 8 * h + (lane >> 3), c = 8 * (lane & 7);
        v4i o = v.b[r][h];  // (without an adapter base goes through bit for bit, a -0 too)
        if (live) o = added(o, mine + row * kSumRow + c);
        if (16 * r + row < t.rows && c0 + c < p.cols) *reinterpret_cast<v4i*>(p.out + out_row[r][h] + c0 + c) = o;
      }
      if (live) wave_lds_order();
    }
  };

  // the wave's groups: wave, wave + 4, .. of the block's
  const uint32_t all = (p.cols + 63) / 64, end = min((blockIdx.y + 1) * 4 * p.groups, all);
  uint32_t g = blockIdx.y * 4 * p.groups + wave;
  Group even, odd;
  load(g, even);
  if (live) {
    const float s = p.scaled ? 1.0f : t.scale;
    for (uint32_t i = tid; i < 16 * RB * KJ * 8; i += 256) {
      const uint32_t r = i / (KJ * 8), j = i % (KJ * 8) * 4;
      v4f v{0.f, 0.f, 0.f, 0.f};
      if (r < t.rows && j < rank) {
        const float* from = p.h + (uint64_t)row_of(r) * rank + j;
        const uint64_t step = (uint64_t)p.seg.rows * rank;
#pragma unroll 8
        for (uint32_t q = 0; q < p.splits; ++q) v += *reinterpret_cast<const v4f*>(from + q * step);
      }
      *reinterpret_cast<v4f*>(hs + r * kRow + j) = v4f{v[0] * s, v[1] * s, v[2] * s, v[3] * s};
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int q = 0; q < KJ; ++q)
      if (live) split8(hs + (16 * r + lr) * kRow + 32 * q + 8 * lg, hi[r][q], lo[r][q]);
  while (g < end) {
    if (g + 4 < end) load(g + 4, odd);
    finish(g, even);
    if (g + 4 >= end) break;
    if (g + 8 < end) load(g + 8, even);
    finish(g + 4, odd);
    g += 8;
  }
}

// The same for tiles of 64 rows, 16 a wave, whose weights the waves share: the
// block's 64 columns of them lie in LDS (the next ones' loads under way), so
// that they are read once per 64 rows.
template <int KJ, bool kColumns>
__global__ __launch_bounds__(256, tall_occupancy(KJ)) void adapter_up_tall_kernel(UpParams p) {
  constexpr uint32_t kSumRow = 64 + 4, kPitch = kColumns ? 128 + 16 : KJ * 64 + 16, kStage = (kColumns ? KJ * 32 : 64) * kPitch;
  __shared__ __align__(16) uint8_t staged[2 * kStage];
  __shared__ __align__(16) float sums[4 * 16 * kSumRow];
  Tile t;
  if (!find_tile(p.seg, 64, blockIdx.x, t, p.err)) return;
  if (t.adapter >= p.seg.adapters && t.adapter != kNoAdapter) return;
  const bool live = t.adapter != kNoAdapter;
  if (!live && p.base == p.out) return;
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), rank = p.rank;
  const uint16_t* const w = p.w + (uint64_t)(live ? t.adapter : 0) * rank * p.cols;
  float* const mine = sums + wave * 16 * kSumRow;
  const bool some = 16 * wave < t.rows;  // rows for this wave
  // base and out: rows 8 h + (lane >> 3) of 16, 8 columns a lane
  uint64_t base_row[2], out_row[2];
#pragma unroll
  for (uint32_t h = 0; h < 2; ++h) {
    const uint64_t row = t.row0 + min(16 * wave + 8 * h + (lane >> 3), t.rows - 1);
    base_row[h] = row * p.base_stride;
    out_row[h] = row * p.out_stride;
  }
  // 16-byte piece 256 i + tid of the 64 columns' weights: kColumns 8 of every
  // rank row, else rank / 8 of every column, contiguous
  const uint32_t per_row = kColumns ? 8 : rank / 8;
  uint32_t put[KJ];
#pragma unroll
  for (int i = 0; i < KJ; ++i) {
    const uint32_t e = 256 * i + tid;
    put[i] = e / per_row * kPitch + e % per_row * 16;
  }
  struct Group {
    v4i x[KJ], b[2];
  };
  auto load = [&](uint32_t g, Group& v) __attribute__((always_inline)) {
    const uint32_t c0 = g * 64, valid = min(64u, p.cols - c0);
    if (live) {
#pragma unroll
      for (int i = 0; i < KJ; ++i) {
        const uint32_t e = 256 * i + tid;
        v.x[i] = v4i{0, 0, 0, 0};
        if constexpr (kColumns) {
          if (e < 8 * rank && 8 * (e & 7) < valid) v.x[i] = load16(w + (uint64_t)(e >> 3) * p.cols + c0 + 8 * (e & 7));
        } else {
          if (e < valid * per_row) v.x[i] = load16(w + (uint64_t)c0 * rank + 8 * e);
        }
      }
    }
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      v.b[h] = v4i{0, 0, 0, 0};
      if (p.base && some && 8 * (lane & 7) < valid) v.b[h] = load16_once(p.base + base_row[h] + c0 + 8 * (lane & 7));
    }
  };
  auto stage = [&](uint32_t to, const Group& v) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < KJ; ++i)
      if (256u * i + tid < (kColumns ? 8 * rank : 64 * per_row))
        *reinterpret_cast<v4i*>(staged + to * kStage + put[i]) = v.x[i];
  };
  const uint32_t all = (p.cols + 63) / 64, end = min((blockIdx.y + 1) * p.groups, all);
  uint32_t g = blockIdx.y * p.groups;
  Group now, next;
  load(g, now);
  v4i hi[KJ], lo[KJ];
  if (live) {
    // (ranks past the last: zeros on both sides)
    if (rank < KJ * 32u)
      for (uint32_t i = tid; i < 2 * kStage / 16; i += 256) *reinterpret_cast<v4i*>(staged + 16 * i) = v4i{0, 0, 0, 0};
    const float s = p.scaled ? 1.0f : t.scale;
    const uint64_t step = (uint64_t)p.seg.rows * rank;
    const float* const from = p.h + (t.row0 + min(16 * wave + lr, t.rows - 1)) * (uint64_t)rank + 8 * lg;
#pragma unroll
    for (int q = 0; q < KJ; ++q) {
      v4f v0{0.f, 0.f, 0.f, 0.f}, v1 = v0;
      if (32 * q + 8 * lg < rank) {
#pragma unroll 4
        for (uint32_t i = 0; i < p.splits; ++i) {
          v0 += *reinterpret_cast<const v4f*>(from + i * step + 32 * q);
          v1 += *reinterpret_cast<const v4f*>(from + i * step + 32 * q + 4);
        }
      }
      const float f[8] = {v0[0] * s, v0[1] * s, v0[2] * s, v0[3] * s, v1[0] * s, v1[1] * s, v1[2] * s, v1[3] * s};
      split8(f, hi[q], lo[q]);
    }
    __syncthreads();
    stage(0, now);
  }
  __syncthreads();
  for (uint32_t at = 0; g < end; ++g, at ^= 1) {
    if (g + 1 < end) load(g + 1, next);
    if (some) {
      const uint32_t c0 = g * 64;
      if (live) {
        v4f acc[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) acc[u] = v4f{0.f, 0.f, 0.f, 0.f};
        const uint8_t* const st = staged + at * kStage;
#pragma unroll
        for (int q = 0; q < KJ; ++q)
#pragma unroll
          for (uint32_t u = 0; u < 4; ++u) {
            v4i x;
            if constexpr (kColumns)
              x = transposed(st + (32 * q + 8 * lg + (lr >> 2)) * kPitch + 2 * (32 * (u >> 1) + 8 * (lr & 3) + 4 * (u & 1)), kPitch);
            else
              x = *reinterpret_cast<const v4i*>(st + (32 * (u >> 1) + 8 * (lr >> 2) + 4 * (u & 1) + (lr & 3)) * kPitch + 64 * q + 16 * lg);
            acc[u] = mfma(x, lo[q], acc[u]);
            acc[u] = mfma(x, hi[q], acc[u]);
          }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
          *reinterpret_cast<v4f*>(mine + lr * kSumRow + 32 * (u >> 1) + 8 * lg + 4 * (u & 1)) = acc[u];
        wave_lds_order();
      }
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        const uint32_t row = 8 * h + (lane >> 3), c = 8 * (lane & 7);
        v4i o = now.b[h];  // (without an adapter base goes through bit for bit, a -0 too)
        if (live) o = added(o, mine + row * kSumRow + c);
        if (16 * wave + row < t.rows && c0 + c < p.cols) *reinterpret_cast<v4i*>(p.out + out_row[h] + c0 + c) = o;
      }
      if (live) wave_lds_order();
    }
    if (live && g + 1 < end) stage(at ^ 1, next);
    now = next;
    block_lds_barrier();
  }
}

// ---------------------------------------------------- splits of a backward
// h and dh from the splits: dh in fp32 for dx, and both as three bf16 that add
// up to the value, in the order of the gradients' MFMA operands, so that a wave
// loads 1 KB in one piece: [32 rows][part][16 ranks][lane (rank lr, rows 8 lg
// ..)][8 rows].
constexpr uint32_t kFinishRows = 16;
struct FinishParams {
  Segments seg;
  const float* part[2];   // [splits][rows][rank]: x A^T, dy B
  float* dh;              // [rows][rank], scaled
  uint16_t* parts[2];
  uint32_t* err;
  uint32_t splits[2];
  uint32_t rank;
};
__global__ __launch_bounds__(256) void adapter_finish_kernel(FinishParams p) {
  __shared__ float sums[kFinishRows][kMaxRank + 1];
  Tile t;
  if (!find_tile(p.seg, kFinishRows, blockIdx.x, t, p.err, blockIdx.y == 0) || t.adapter >= p.seg.adapters) return;
  const uint32_t side = blockIdx.y, pieces = p.rank / 4;
  for (uint32_t i = threadIdx.x; i < t.rows * pieces; i += 256) {
    const uint32_t r = i / pieces, j = i % pieces * 4;
    const uint64_t at = (uint64_t)(t.row0 + r) * p.rank + j, step = (uint64_t)p.seg.rows * p.rank;
    v4f v{0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (uint32_t q = 0; q < p.splits[side]; ++q) v += *reinterpret_cast<const v4f*>(p.part[side] + q * step + at);
    v = v4f{v[0] * t.scale, v[1] * t.scale, v[2] * t.scale, v[3] * t.scale};
    if (side) *reinterpret_cast<v4f*>(p.dh + at) = v;
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[r][j + e] = v[e];
  }
  __syncthreads();
  const uint32_t blocks = (p.rank + 15) / 16;
  for (uint32_t i = threadIdx.x; i < kFinishRows * p.rank; i += 256) {
    const uint32_t r = i & (kFinishRows - 1), j = i / kFinishRows;
    if (r >= t.rows) continue;
    const uint32_t row = t.row0 + r;
    float v = sums[r][j];
    uint16_t* const part = p.parts[side] + ((uint64_t)(row / 32) * 3 * blocks + j / 16) * 512 +
                           (row / 8 % 4 * 16 + j % 16) * 8 + row % 8;
#pragma unroll
    for (uint32_t q = 0; q < 3; ++q) {
      const uint32_t h = f32_to_bf16_bits(q < 2 ? part_of(v) : v);
      part[q * blocks * 512] = (uint16_t)h;
      v -= bf16_bits_to_f32(h);
    }
  }
}

// ------------------------------------------------- gradients of A and of B
struct GradSide {
  const uint16_t* src;   // [rows][cols]: x for A, dy for B
  const uint16_t* parts; // as above
  float* out;            // [adapters][rank][cols], or (B) [adapters][cols][rank]
  float* part;           // [splits] of those when the rows are split
  uint32_t stride, cols;
};
struct GradParams {
  Segments seg;
  GradSide side[2];
  uint32_t rank, splits;
};

// the block's sums, [64 columns][rank], to the gradient or the split's part
template <int NJ, bool kB>
__device__ __forceinline__ void write_grads(const GradParams& p, const GradSide& d, uint32_t adapter, uint32_t c0,
                                            const float* sums) {
  constexpr uint32_t kSumRow = NJ * 16 + 4;
  const uint32_t tid = threadIdx.x;
  float* const out = p.splits > 1 ? d.part + (uint64_t)blockIdx.y * p.seg.adapters * p.rank * d.cols : d.out;
  const uint32_t cols = min(64u, d.cols - c0);
  if constexpr (kB) {
    // one contiguous piece: columns c0 .., rank values each
    float* const o = out + ((uint64_t)adapter * d.cols + c0) * p.rank;
    for (uint32_t i = tid; i < cols * (p.rank / 4); i += 256) {
      const uint32_t col = i / (p.rank / 4), j = i % (p.rank / 4) * 4;
      *reinterpret_cast<v4f*>(o + 4 * (uint64_t)i) = *reinterpret_cast<const v4f*>(sums + col * kSumRow + j);
    }
  } else {
    for (uint32_t i = tid; i < p.rank * 16; i += 256) {
      const uint32_t j = i / 16, col = i % 16 * 4;
      if (col >= cols) continue;
      const float* const from = sums + col * kSumRow + j;
      *reinterpret_cast<v4f*>(out + ((uint64_t)adapter * p.rank + j) * d.cols + c0 + col) =
          v4f{from[0], from[kSumRow], from[2 * kSumRow], from[3 * kSumRow]};
    }
  }
}

// 64 columns of one adapter's gradient over its rows, in blocks of 32 rows at
// multiples of 32; with several splits, every splits-th group of four blocks.
// The four waves take the blocks of a group and add up in LDS, in order.  The
// rows' 64 columns go through the wave's LDS and are read transposed.
template <int NJ, bool kB>
__device__ __forceinline__ void grad_tile(const GradParams& p, const GradSide& d, uint32_t adapter, uint8_t* lds) {
  constexpr uint32_t kPitch = 128 + 16, kSumRow = NJ * 16 + 4;
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t c0 = blockIdx.x * 64;
  if (c0 >= d.cols) return;
  uint8_t* const st = lds + wave * 32 * kPitch;
  v4f acc[4][NJ];
#pragma unroll
  for (int u = 0; u < 4; ++u)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[u][j] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint32_t c = c0 + 8 * (lane & 7);
  uint32_t turn = 0;  // of the block, modulo 4 splits
  const uint32_t mine = 4 * blockIdx.y + wave;
  for (uint32_t s = 0; s < p.seg.segments; ++s) {
    if (p.seg.adapter[s] != adapter) continue;
    const uint32_t lo_row = p.seg.offsets[s], hi_row = p.seg.offsets[s + 1];
    if (hi_row <= lo_row || hi_row > p.seg.rows) continue;
    const uint32_t first = lo_row / 32, blocks = (hi_row + 31) / 32 - first, all = 4 * p.splits;
    for (uint32_t i = (mine + all - turn) % all; i < blocks; i += all) {
      const uint32_t r0 = (first + i) * 32, r = r0 + 8 * lg;
      v4i m[4];
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q) {
        const uint32_t row = r0 + 8 * q + (lane >> 3);
        m[q] = v4i{0, 0, 0, 0};
        if (row >= lo_row && row < hi_row && c < d.cols) m[q] = load16(d.src + (uint64_t)row * d.stride + c);
      }
      v4i h[3][NJ], mask;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        mask[q] = (r + 2 * q >= lo_row && r + 2 * q < hi_row ? 0xffff : 0) |
                  (r + 2 * q + 1 >= lo_row && r + 2 * q + 1 < hi_row ? (int)0xffff0000 : 0);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        // (a rank of less than 16 j + 16: what its places hold goes to results
        // that are not written)
        const uint32_t blocks = (p.rank + 15) / 16;
        const uint16_t* const from =
            d.parts + ((uint64_t)(first + i) * 3 * blocks + min((uint32_t)j, blocks - 1)) * 512 + 8 * lane;
#pragma unroll
        for (uint32_t q = 0; q < 3; ++q) h[q][j] = load16(from + q * blocks * 512) & mask;
      }
#pragma unroll
      for (uint32_t q = 0; q < 4; ++q)
        *reinterpret_cast<v4i*>(st + (8 * q + (lane >> 3)) * kPitch + 16 * (lane & 7)) = m[q];
      wave_lds_order();
#pragma unroll
      for (uint32_t u = 0; u < 4; ++u) {
        const v4i x = transposed(st + (8 * lg + (lr >> 2)) * kPitch + 2 * (16 * u + 4 * (lr & 3)), kPitch);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
          for (int q = 2; q >= 0; --q) acc[u][j] = kB ? mfma(h[q][j], x, acc[u][j]) : mfma(x, h[q][j], acc[u][j]);
        }
      }
      wave_lds_order();
    }
    turn = (turn + blocks) % all;
  }
  // [64 columns][rank], the waves in order
  float* const sums = reinterpret_cast<float*>(lds);
  for (uint32_t v = 0; v < 4; ++v) {
    __syncthreads();
    if (wave != v) continue;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (kB) {  // lane: column 16 u + lr, ranks 16 j + 4 lg ..
          v4f* const o = reinterpret_cast<v4f*>(sums + (16 * u + lr) * kSumRow + 16 * j + 4 * lg);
          *o = v ? *o + acc[u][j] : acc[u][j];
        } else {  // lane: rank 16 j + lr, columns 16 u + 4 lg ..
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float* const o = sums + (16 * u + 4 * lg + e) * kSumRow + 16 * j + lr;
            *o = v ? *o + acc[u][j][e] : acc[u][j][e];
          }
        }
      }
  }
  __syncthreads();
  write_grads<NJ, kB>(p, d, adapter, c0, sums);
}

// The same for ranks above 64 and 128 columns: the waves take NJ / 4 of the
// 16-rank pieces each and all the rows, whose columns they share in LDS, two
// pieces' loads under way: nothing is added up between them, and the parts of h,
// six times the rows' bytes, are read once for 128 columns.  Rank 128, 300 rows,
// 12288 + 4096 columns 44 -> 16 us, 4099 rows 92 -> 74; at rank 64 the waves' own
// rows are faster (4099 rows: 51 us against 68).
template <int NJ, bool kB>
__device__ __forceinline__ void grad_ranks_tile(const GradParams& p, const GradSide& d, uint32_t adapter, uint8_t* lds) {
  constexpr uint32_t kPitch = 256 + 16, kStage = 32 * kPitch, kSumRow = NJ * 16 + 4, JW = NJ / 4;
  const uint32_t tid = threadIdx.x, lane = tid & 63, lr = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t c0 = blockIdx.x * 128, c = c0 + 8 * (tid & 7), blocks16 = (p.rank + 15) / 16;
  if (c0 >= d.cols) return;
  // the block's 32-row pieces: every splits-th of the adapter's
  uint32_t s = 0, lo = 0, hi = 0, first = 0, blocks = 0, at = blockIdx.y;
  auto find = [&]() -> bool {
    while (at >= blocks) {
      at -= blocks;
      blocks = 0;
      for (; s < p.seg.segments; ++s) {
        if (p.seg.adapter[s] != adapter) continue;
        lo = p.seg.offsets[s], hi = p.seg.offsets[s + 1];
        if (hi > lo && hi <= p.seg.rows) break;
      }
      if (s >= p.seg.segments) return false;
      ++s;
      first = lo / 32;
      blocks = (hi + 31) / 32 - first;
    }
    return true;
  };
  struct Rows {
    v4i x[2], h[JW][3];
  };
  auto load = [&](Rows& v) __attribute__((always_inline)) {
    const uint32_t r0 = (first + at) * 32, row = r0 + (tid >> 3), r = r0 + 8 * lg;
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) {
      v.x[q] = v4i{0, 0, 0, 0};
      if (row >= lo && row < hi && c + 64 * q < d.cols) v.x[q] = load16(d.src + (uint64_t)row * d.stride + c + 64 * q);
    }
    v4i mask;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      mask[q] = (r + 2 * q >= lo && r + 2 * q < hi ? 0xffff : 0) |
                (r + 2 * q + 1 >= lo && r + 2 * q + 1 < hi ? (int)0xffff0000 : 0);
#pragma unroll
    for (uint32_t j = 0; j < JW; ++j) {
      const uint16_t* const from =
          d.parts + ((uint64_t)(first + at) * 3 * blocks16 + min(JW * wave + j, blocks16 - 1)) * 512 + 8 * lane;
#pragma unroll
      for (uint32_t q = 0; q < 3; ++q) v.h[j][q] = load16(from + q * blocks16 * 512) & mask;
    }
  };
  v4f acc[8][JW];
#pragma unroll
  for (int u = 0; u < 8; ++u)
#pragma unroll
    for (uint32_t j = 0; j < JW; ++j) acc[u][j] = v4f{0.f, 0.f, 0.f, 0.f};
  // two pieces' loads under way
  Rows now, next, after;
  bool more = find(), later = false;
  if (more) {
    load(now);
    at += p.splits;
    later = find();
    if (later) load(next);
  }
  for (uint32_t b = 0; more; b ^= 1) {
    more = later;
    if (later) {
      at += p.splits;
      later = find();
      if (later) load(after);
    }
    uint8_t* const st = lds + b * kStage;
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q)
      *reinterpret_cast<v4i*>(st + (tid >> 3) * kPitch + 16 * (tid & 7) + 128 * q) = now.x[q];
    block_lds_barrier();
#pragma unroll
    for (uint32_t u = 0; u < 8; ++u) {
      const v4i x = transposed(st + (8 * lg + (lr >> 2)) * kPitch + 2 * (16 * u + 4 * (lr & 3)), kPitch);
#pragma unroll
      for (uint32_t j = 0; j < JW; ++j)
#pragma unroll
        for (int q = 2; q >= 0; --q) acc[u][j] = kB ? mfma(now.h[j][q], x, acc[u][j]) : mfma(x, now.h[j][q], acc[u][j]);
    }
    now = next;
    next = after;
  }
  float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
  for (uint32_t half = 0; half < 2; ++half) {
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
      for (uint32_t j = 0; j < JW; ++j) {
        const uint32_t rank16 = 16 * (JW * wave + j);
        const v4f v = acc[4 * half + u][j];
        if constexpr (kB) {  // lane: column 16 u + lr, ranks 4 lg ..
          *reinterpret_cast<v4f*>(sums + (16 * u + lr) * kSumRow + rank16 + 4 * lg) = v;
        } else {  // lane: rank lr, columns 16 u + 4 lg ..
#pragma unroll
          for (int e = 0; e < 4; ++e) sums[(16 * u + 4 * lg + e) * kSumRow + rank16 + lr] = v[e];
        }
      }
    __syncthreads();
    if (c0 + 64 * half < d.cols) write_grads<NJ, kB>(p, d, adapter, c0 + 64 * half, sums);
  }
}

template <int NJ>
__global__ __launch_bounds__(256) void adapter_grad_kernel(GradParams p) {
  constexpr uint32_t kStaged = NJ == 8 ? 2 * 32 * 272 : 4 * 32 * 144, kSums = 64 * (NJ * 16 + 4) * 4;
  __shared__ __align__(16) uint8_t lds[kSums > kStaged ? kSums : kStaged];
  const uint32_t adapter = blockIdx.z >> 1;
  if constexpr (NJ == 8) {
    if (blockIdx.z & 1) grad_ranks_tile<NJ, true>(p, p.side[1], adapter, lds);
    else grad_ranks_tile<NJ, false>(p, p.side[0], adapter, lds);
  } else {
    if (blockIdx.z & 1) grad_tile<NJ, true>(p, p.side[1], adapter, lds);
    else grad_tile<NJ, false>(p, p.side[0], adapter, lds);
  }
}

// the splits of the gradients, in order: of A, then (blocks from `first_b`
// on) of B
__global__ __launch_bounds__(256) void adapter_grad_reduce_kernel(GradParams p, uint32_t first_b) {
  const uint32_t side = blockIdx.x >= first_b;
  const uint64_t count = (uint64_t)p.seg.adapters * p.rank * p.side[side].cols;
  const uint64_t i = ((uint64_t)(blockIdx.x - side * first_b) * 256 + threadIdx.x) * 4;
  if (i >= count) return;
  const float* const part = p.side[side].part + i;
  v4f v = *reinterpret_cast<const v4f*>(part);
#pragma unroll 4
  for (uint32_t s = 1; s < p.splits; ++s) v += *reinterpret_cast<const v4f*>(part + s * count);
  *reinterpret_cast<v4f*>(p.side[side].out + i) = v;
}

// ------------------------------------------------------------------ host
bool shape_ok(const AdapterArgs& a) {
  return a.rows && a.segments && a.adapters && a.rank && a.rank <= kMaxRank && a.rank % 8 == 0 && a.n && a.k &&
         a.n % 8 == 0 && a.k % 8 == 0 && a.rows <= kMaxRows && a.segments <= kMaxSegments &&
         a.adapters <= 0x7fffu && a.n <= kMaxColumns && a.k <= kMaxColumns;
}
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// row blocks of 16 in a tile: four where segments have 64 rows on average
uint32_t tile_blocks(const AdapterArgs& a) { return a.rows / 64 >= a.segments ? 4 : 1; }
// tiles of the segments at most: every segment ends in at most one short one
uint32_t tile_bound(const AdapterArgs& a, uint32_t height) {
  const uint64_t t = ((uint64_t)a.rows + (uint64_t)std::min(a.segments, a.rows) * (height - 1)) / height;
  return (uint32_t)std::min<uint64_t>(t, a.rows);
}
// Columns of a K split of the down product, of one side or both: of one to
// three rounds of the blocks that the card holds at once the cheapest by the
// rounds' columns and 512 more for a round's beginning and end (a short second
// round costs as much as a full one); 512 at least, since every block of the up
// product adds the splits (64 one-row requests of rank 128 over 12288 columns 30
// us against 43 with 256 columns; 1024 wins with one adapter, 29 us, and loses
// with 16 at rank 64, 22.4 against 20.4).
constexpr uint32_t kRounds = 3, kSplitColumns = 512;
uint32_t held_blocks(uint32_t rank, uint32_t blocks) { return kCus * down_occupancy((rank + 15) / 16, blocks); }
uint32_t split_columns(uint32_t tiles, uint32_t cols, uint32_t other, uint32_t rank, uint32_t blocks) {
  const uint32_t held = held_blocks(rank, blocks), most = std::max(cols, other);
  auto parts = [&](uint32_t at) { return (uint64_t)tiles * ((cols + at - 1) / at + (other + at - 1) / at); };
  uint32_t best = (most + 127) / 128;  // in 128 columns, as the waves take them
  uint64_t cost = (parts(128 * best) + held - 1) / held * (128 * best + 512);
  for (uint32_t r = 1; r <= kRounds; ++r) {
    // the shortest split whose blocks fit r rounds
    uint32_t low = kSplitColumns / 128, high = (most + 127) / 128;
    if (low >= high || parts(128 * high) > (uint64_t)r * held) continue;
    while (low < high) {
      const uint32_t mid = (low + high) / 2;
      if (parts(128 * mid) <= (uint64_t)r * held) high = mid;
      else low = mid + 1;
    }
    const uint64_t c = (uint64_t)r * (128 * high + 512);
    if (c < cost) {
      cost = c;
      best = high;
    }
  }
  return 128 * best;
}
uint32_t splits_of(uint32_t cols, uint32_t at) { return (cols + at - 1) / at; }

template <typename F>
void with_pow2(uint32_t n, F&& f) {
  if (n <= 1) f(std::integral_constant<int, 1>{});
  else if (n <= 2) f(std::integral_constant<int, 2>{});
  else if (n <= 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

// Whether tiles take the rows of one adapter from all segments: where segments
// have a row or two and an adapter two segments or more, as many as a block's
// scans hold.  256 one-row requests of 16 adapters of rank 128 over 12288
// columns: 42 us against 130 with a tile per segment, 1024 of them 75 against
// 496.  With an adapter of its own per request the scans are lost (256 requests
// of rank 16 51 us against 41), and below 32 segments the tiles are few either
// way (one request 19 us with both).
bool grouped(const AdapterArgs& a) {
  return a.segments >= 32 && a.segments <= kGroupSegments && a.rows / 2 <= a.segments &&
         a.adapters <= std::min(a.segments / 2, kGroupAdapters);
}
// tiles of the groups at most: every adapter, and none, ends in a short one
uint32_t group_bound(const AdapterArgs& a) {
  return std::min<uint32_t>(a.rows, a.rows / 16 + std::min(a.adapters + 1, a.segments));
}

template <bool kColumns>
void launch_up(UpParams p, const AdapterArgs& a, bool group) {
  const bool tall = tile_blocks(a) == 4;
  if (tall && p.rank > 32) {
    // two blocks a CU, each with as many groups as there are splits of h, which
    // every block adds up, while that leaves a block for every other CU (4099 x
    // 4096 outputs of rank 64: 25 us; one block a CU 32, four 29; tiles of 32 rows
    // that read the weights themselves 31.  4099 x 12288 of rank 128: 60 us, 213
    // with 16-row tiles.  1000 x 1024 of rank 128: 13 us; 20 with fewer blocks, 19
    // with one for every CU)
    with_pow2((p.rank + 31) / 32, [&](auto kj) {
      constexpr int KJ = decltype(kj)::value;
      if constexpr (KJ == 2 || KJ == 4) {
        const uint32_t tiles = tile_bound(a, 64), all = (p.cols + 63) / 64, columns = std::max(1u, 2 * kCus / tiles);
        p.groups = std::max((all + columns - 1) / columns, std::min(p.splits, std::max(1u, 2 * all * tiles / kCus)));
        hipLaunchKernelGGL((adapter_up_tall_kernel<KJ, kColumns>), dim3(tiles, (all + p.groups - 1) / p.groups),
                           dim3(256), 0, a.stream, p);
      }
    });
    return;
  }
  // column blocks for as many blocks as the card holds at once (tiles of few
  // rows: every further round repeats the search and the sum of h; 57 one-row
  // requests 10.2 us against 12.7 with three rounds) or, with long segments,
  // for three rounds of that, whose last costs little (8192 rows 117 us a
  // backward call against 126 with one)
  const uint32_t blocks = tall ? 2 : 1;
  const uint32_t tiles = group ? group_bound(a) : tile_bound(a, 16 * blocks), all = (p.cols + 63) / 64;
  with_pow2((p.rank + 31) / 32, [&](auto kj) {
    constexpr int KJ = decltype(kj)::value;
    if constexpr (KJ <= 4) {
      auto launch = [&](auto rb) {
        constexpr int RB = decltype(rb)::value;
        const uint32_t columns = std::max<uint32_t>(1, (RB == 1 ? 1 : 3) * kCus * up_occupancy(KJ, RB) / tiles);
        p.groups = std::max<uint32_t>(1, (all + 4 * columns - 1) / (4 * columns));
        const dim3 grid(tiles, (all + 4 * p.groups - 1) / (4 * p.groups));
        if constexpr (RB == 1 && !kColumns) {
          if (group) {
            hipLaunchKernelGGL((adapter_up_kernel<KJ, 1, false, true>), grid, dim3(256), 0, a.stream, p);
            return;
          }
        }
        hipLaunchKernelGGL((adapter_up_kernel<KJ, RB, kColumns, false>), grid, dim3(256), 0, a.stream, p);
      };
      if constexpr (KJ == 1) {
        if (blocks == 2) {
          launch(std::integral_constant<int, 2>{});
          return;
        }
      }
      launch(std::integral_constant<int, 1>{});
    }
  });
}

Segments segments_of(const AdapterArgs& a) {
  return Segments{a.offsets, a.adapter, a.scale, a.segments, a.rows, a.adapters};
}

template <bool kBackward>
void launch_down(const DownParams& d, uint32_t tiles, uint32_t blocks, uint32_t splits, hipStream_t s) {
  const dim3 grid(tiles, splits, kBackward ? 2 : 1);
  with_pow2((d.rank + 15) / 16, [&](auto nj) {
    constexpr int NJ = decltype(nj)::value;
    if (blocks == 4) hipLaunchKernelGGL((adapter_down_kernel<NJ, 4, kBackward>), grid, dim3(256), 0, s, d);
    else hipLaunchKernelGGL((adapter_down_kernel<NJ, 1, kBackward>), grid, dim3(256), 0, s, d);
  });
}

// columns of a block of the gradients
uint32_t grad_columns(const AdapterArgs& a) { return a.rank > 64 ? 128 : 64; }

struct BackwardPlan {
  uint32_t blocks, tiles, finish_tiles, per_split, splits[2], grad_splits;
  uint64_t part[2], dh, parts[2], grads[2], bytes;
};
BackwardPlan backward_plan(const AdapterArgs& a) {
  BackwardPlan p{};
  p.blocks = tile_blocks(a);
  p.tiles = tile_bound(a, 16 * p.blocks);
  p.finish_tiles = tile_bound(a, kFinishRows);
  p.per_split = split_columns(p.tiles, a.k, a.n, a.rank, p.blocks);
  p.splits[0] = splits_of(a.k, p.per_split);
  p.splits[1] = splits_of(a.n, p.per_split);
  // row splits of the gradients: two rounds of blocks (of 128 columns: one), 512
  // rows each at least
  const uint32_t width = grad_columns(a);
  const uint64_t blocks = (uint64_t)a.adapters * ((a.n + width - 1) / width + (a.k + width - 1) / width);
  p.grad_splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((a.rows + 511) / 512, (a.rank > 64 ? 512 : 1024) / blocks));
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int s = 0; s < 2; ++s) p.part[s] = take((uint64_t)p.splits[s] * a.rows * a.rank * 4);
  p.dh = take((uint64_t)a.rows * a.rank * 4);
  for (int s = 0; s < 2; ++s) p.parts[s] = take(3ull * ((a.rank + 15) / 16 * 16) * ((a.rows + 31ull) / 32 * 32) * 2);
  if (p.grad_splits > 1)
    for (int s = 0; s < 2; ++s) p.grads[s] = take((uint64_t)p.grad_splits * a.adapters * a.rank * (s ? a.n : a.k) * 4);
  p.bytes = at;
  return p;
}

}  // namespace

uint64_t AdapterGemmWorkspaceBytes(uint32_t rows, uint32_t rank, uint32_t k) {
  if (!rows || rows > kMaxRows || !rank || rank > kMaxRank || !k || k > kMaxColumns) return 0;
  // as many splits as any segments lead to: every block has a tile of 64 rows at
  // most, or of 16
  const uint64_t tall = (uint64_t)kRounds * held_blocks(rank, 4) / ((rows + 63) / 64);
  const uint64_t low = (uint64_t)kRounds * held_blocks(rank, 1) / ((rows + 15) / 16);
  const uint64_t splits = std::min<uint64_t>(splits_of(k, kSplitColumns), std::max<uint64_t>(1, std::max(tall, low)));
  return splits * rows * rank * 4;
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
  const bool group = grouped(a);
  const uint32_t blocks = tile_blocks(a), tiles = group ? group_bound(a) : tile_bound(a, 16 * blocks);
  const uint32_t per_split = split_columns(tiles, a.k, 0, a.rank, blocks), splits = splits_of(a.k, per_split);
  if (a.workspace_bytes < AdapterGemmWorkspaceBytes(a.rows, a.rank, a.k) || !aligned16(a.workspace))
    return Invalid("adapter_gemm_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  DownParams d{};
  d.seg = segments_of(a);
  d.side[0] = DownSide{a.x, a.a, static_cast<float*>(a.workspace), a.x_stride, a.k, per_split, splits};
  d.err = a.error_flag;
  d.rank = a.rank;
  if (group)
    with_pow2((a.rank + 15) / 16, [&](auto nj) {
      hipLaunchKernelGGL((adapter_down_group_kernel<decltype(nj)::value>), dim3(tiles, splits), dim3(256), 0, a.stream,
                         d);
    });
  else launch_down<false>(d, tiles, blocks, splits, a.stream);
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
  launch_up<false>(u, a, group);
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
  // (dx is written before the weights' gradients read x and dy)
  if (a.out == a.x || a.out == a.dy) return Invalid("adapter_backward_alias_invalid");
  const BackwardPlan plan = backward_plan(a);
  if (a.workspace_bytes < plan.bytes || !aligned16(a.workspace)) return Invalid("adapter_backward_workspace_invalid");
  St clean = RequireCleanLastError();
  if (!clean.ok()) return clean;
  uint8_t* const ws = static_cast<uint8_t*>(a.workspace);
  auto f32 = [&](uint64_t at) { return reinterpret_cast<float*>(ws + at); };
  auto u16 = [&](uint64_t at) { return reinterpret_cast<uint16_t*>(ws + at); };
  DownParams d{};
  d.seg = segments_of(a);
  d.side[0] = DownSide{a.x,   a.a, f32(plan.part[0]), a.x_stride, a.k, plan.per_split, plan.splits[0]};
  d.side[1] = DownSide{a.dy,  a.b, f32(plan.part[1]), a.dy_stride, a.n, plan.per_split, plan.splits[1]};
  d.err = a.error_flag;
  d.rank = a.rank;
  launch_down<true>(d, plan.tiles, plan.blocks, std::max(plan.splits[0], plan.splits[1]), a.stream);
  FinishParams f{};
  f.seg = d.seg;
  f.dh = f32(plan.dh);
  for (int s = 0; s < 2; ++s) {
    f.part[s] = d.side[s].out;
    f.splits[s] = plan.splits[s];
    f.parts[s] = u16(plan.parts[s]);
  }
  f.err = a.error_flag;
  f.rank = a.rank;
  hipLaunchKernelGGL(adapter_finish_kernel, dim3(plan.finish_tiles, 2), dim3(256), 0, a.stream, f);
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
  launch_up<true>(u, a, false);
  GradParams g{};
  g.seg = d.seg;
  g.rank = a.rank;
  g.splits = plan.grad_splits;
  // da = dh^T x, db = dy^T h
  g.side[0] = GradSide{a.x, f.parts[1], a.da, f32(plan.grads[0]), a.x_stride, a.k};
  g.side[1] = GradSide{a.dy, f.parts[0], a.db, f32(plan.grads[1]), a.dy_stride, a.n};
  with_pow2((a.rank + 15) / 16, [&](auto nj) {
    hipLaunchKernelGGL((adapter_grad_kernel<decltype(nj)::value>),
                       dim3((std::max(a.n, a.k) + grad_columns(a) - 1) / grad_columns(a), plan.grad_splits, 2 * a.adapters), dim3(256), 0, a.stream,
                       g);
  });
  if (plan.grad_splits > 1) {
    auto blocks = [&](uint32_t cols) { return (uint32_t)(((uint64_t)a.adapters * a.rank * cols / 4 + 255) / 256); };
    hipLaunchKernelGGL(adapter_grad_reduce_kernel, dim3(blocks(a.k) + blocks(a.n)), dim3(256), 0, a.stream, g,
                       blocks(a.k));
  }
  return AfterLaunch("adapter_backward_launch_failed");
}

}  // namespace pih_amd
