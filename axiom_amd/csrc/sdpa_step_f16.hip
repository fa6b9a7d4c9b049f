#include "sdpa_step.hpp"
namespace axhip {
int launch_step_f16(const CacheArgs &a, hipStream_t s) { return launch_step<false>(a, s); }
} // namespace axhip
