// Products of e4m3 rows (linear_tile.h, linear_small.h).
#include "linear_small.h"

int dgcn::mat_tile_e4m3(const MatParams& P, int out_type, int tile, hipStream_t s) {
  switch (out_type) {
    case DGCN_T_F32: return tile_size<WideE4m3, float, 0, 0>(P, tile, s);
    case DGCN_T_BF16: return tile_size<uint8_t, __bf16, 0, 0>(P, tile, s);
    case DGCN_T_F16: return tile_size<uint8_t, _Float16, 0, 0>(P, tile, s);
    default: return DGCN_E_MODE;
  }
}

int dgcn::mat_small_e4m3(const MatParams& P, int out_type, hipStream_t s) {
  switch (out_type) {
    case DGCN_T_F32: return small_launch<WideE4m3, float>(P, s);
    case DGCN_T_BF16: return small_launch<WideE4m3, __bf16>(P, s);
    case DGCN_T_F16: return small_launch<WideE4m3, _Float16>(P, s);
    default: return DGCN_E_MODE;
  }
}
