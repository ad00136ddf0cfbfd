// Products of fp16 rows (linear_tile.h, linear_small.h).
#include "linear_small.h"

int dgcn::mat_tile_f16(const MatParams& P, int ta, int tb, int tile, hipStream_t s) {
  return tile_layout<_Float16>(P, ta, tb, tile, s);
}

int dgcn::mat_small_f16(const MatParams& P, hipStream_t s) { return small_launch<_Float16, _Float16>(P, s); }
