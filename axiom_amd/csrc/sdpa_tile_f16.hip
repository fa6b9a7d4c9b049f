#include "sdpa_tile.hpp"
namespace axhip {
int launch_tile_f16(const CacheArgs &a, int waves, hipStream_t s) { return launch_tile<false>(a, waves, s); }
} // namespace axhip
