#include "sdpa_tile.hpp"
namespace axhip {
int launch_tile_bf16(const CacheArgs &a, int waves, hipStream_t s) { return launch_tile<true>(a, waves, s); }
} // namespace axhip
