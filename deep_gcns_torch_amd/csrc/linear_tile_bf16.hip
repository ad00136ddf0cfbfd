// Products of bf16 rows (linear_tile.h, linear_small.h).
#include "linear_small.h"

int dgcn::mat_tile_bf16(const MatParams& P, int ta, int tb, int tile, hipStream_t s) {
  return tile_layout<__bf16>(P, ta, tb, tile, s);
}

int dgcn::mat_small_bf16(const MatParams& P, hipStream_t s) { return small_launch<__bf16, __bf16>(P, s); }
