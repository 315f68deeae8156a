// dma_route.hpp behind a C interface, for test_dma_route.py
#include "dma_route.hpp"

using namespace pih_amd;

extern "C" {
// {whole, rows, splits of the rest}, and the estimate
float route(uint32_t m, uint32_t n, uint32_t k, uint32_t* out) {
  const Route r = route_of(m, n, k);
  out[0] = r.whole;
  out[1] = r.rest.rows;
  out[2] = r.rest.splits;
  return r.us;
}
float rows_us(uint32_t m, uint32_t n, uint32_t k, uint32_t splits, uint32_t rows) { return DmaRowsUs(m, n, k, splits, rows); }
}
