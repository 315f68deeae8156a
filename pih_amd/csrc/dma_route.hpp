// How the rows of a product on the DMA tiles (dma_tile.hpp) run: host arithmetic
// alone, no HIP, so that a CPU build can walk the rules over their ranges.
#pragma once

#include <math.h>

#include "dense_route.hpp"

namespace pih_amd {

constexpr uint32_t TB = 256, KB = 64;  // a tile's columns, a step of k

// Time (us) of m rows in tiles of `rows`: the rounds of tiles on the CUs, each a
// step's time and a tile's own beginning and end
//   256 rows 1.45 and 9,  128 rows 0.95 and 7,  64 rows 0.70 and 6.
inline float DmaRowsUs(uint32_t m, uint32_t n, uint32_t k, uint32_t splits, uint32_t rows) {
  const uint32_t steps = (k / KB + splits - 1) / splits;
  const uint64_t tiles = (uint64_t)((m + rows - 1) / rows) * ((n + TB - 1) / TB) * splits;
  const float tile = rows == 256 ? 9.0f + 1.45f * steps : rows == 128 ? 7.0f + 0.95f * steps : 6.0f + 0.70f * steps;
  return (float)((tiles + kCus - 1) / kCus) * tile;
}

// How the rows of a product [m][n] over k run: tiles of `rows` rows, k in
// `splits` parts.  Time (us): the rounds of tiles on the CUs, each its beginning
// and end and a step's time (DmaRowsUs), no less than B takes at
// the CUs' share of 5.1 TB/s, and for splits the sums written and read at 4 TB/s and a launch.
struct Tiling {
  uint32_t rows, splits;
  float us;
};
inline Tiling tiling_of(uint32_t m, uint32_t n, uint32_t k) {
  Tiling best{256, 1, INFINITY};
  for (uint32_t rows : {64u, 128u, 256u}) {
    if (m <= rows / 2 && rows > 64) break;  // (as many tiles as of half the rows, each slower)
    // (four steps a part, where there are parts)
    for (uint32_t splits = 1; splits <= 64 && (splits == 1 || k / KB / splits >= 4); ++splits) {
      // (no split is empty)
      const uint32_t steps = k / KB, part = (steps + splits - 1) / splits;
      if ((steps + part - 1) / part != splits) continue;
      const uint64_t tiles = (uint64_t)((m + rows - 1) / rows) * ((n + TB - 1) / TB) * splits;
      const float busy = (float)std::min<uint64_t>(tiles, kCus) / kCus;
      const float us = std::max(DmaRowsUs(m, n, k, splits, rows), (float)n * k * (2.0f / 5.1e6f) / busy) +
                       (splits > 1 ? 7.0f + (float)splits * m * n * (8.0f / 4.0e6f) : 0.0f);
      if (us < best.us) best = {rows, splits, us};
    }
  }
  return best;
}
// All rows alike, or the whole 256 without splits and the rest by itself, where B
// is read once more (at 5 TB/s) and the launch costs 3 us
struct Route {
  uint32_t whole;  // rows in tiles of 256, unsplit
  Tiling rest;     // of those behind
  uint64_t sums;   // fp32 elements
  float us;
};
inline Route route_of(uint32_t m, uint32_t n, uint32_t k) {
  const Tiling all = tiling_of(m, n, k);
  const uint32_t whole = m / 256 * 256, rest = m - whole;
  Route r{0, all, all.splits > 1 ? (uint64_t)all.splits * m * n : 0, all.us};
  if (whole && rest) {
    const Tiling last = tiling_of(rest, n, k);
    const float us = DmaRowsUs(whole, n, k, 1, 256) + last.us + 3.0f;
    if (us < all.us) r = {whole, last, last.splits > 1 ? (uint64_t)last.splits * rest * n : 0, us};
  }
  return r;
}

}  // namespace pih_amd
