// Tiled products of bf16 rows (linear_tile.h).
#include "linear_tile.h"

int dgcn::mat_tile_bf16(const MatParams& P, int ta, int tb, int tile, hipStream_t s) {
  return tile_layout<__bf16>(P, ta, tb, tile, s);
}
