// Results in bf16: see gemm_q8_tile.hpp.
#include "gemm_q8_tile.hpp"

namespace axhip {
int launch_q8_tile_bf16(const Q8Args &g, int tile, bool aligned, hipStream_t s) { return launch_q8_tile_as<AXHIP_DTYPE_BF16>(g, tile, aligned, s); }
} // namespace axhip
