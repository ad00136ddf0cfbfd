// Products of fp32 rows (linear_tile.h, linear_small.h).
#include "linear_small.h"

int dgcn::mat_tile_f32(const MatParams& P, int ta, int tb, int tile, hipStream_t s) {
  return tile_layout<float>(P, ta, tb, tile, s);
}

int dgcn::mat_small_f32(const MatParams& P, hipStream_t s) { return small_launch<float, float>(P, s); }
