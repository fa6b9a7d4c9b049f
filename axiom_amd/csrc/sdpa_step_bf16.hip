#include "sdpa_step.hpp"
namespace axhip {
int launch_step_bf16(const CacheArgs &a, hipStream_t s) { return launch_step<true>(a, s); }
} // namespace axhip
