// Results in f32: see gemm_q8_tile.hpp.
#include "gemm_q8_tile.hpp"

namespace axhip {
int launch_q8_tile_f32(const Q8Args &g, int tile, bool aligned, hipStream_t s) { return launch_q8_tile_as<AXHIP_DTYPE_F32>(g, tile, aligned, s); }
} // namespace axhip
