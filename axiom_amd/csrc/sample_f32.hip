// Logits in f32: see sample_kernel.hpp.
#include "sample_kernel.hpp"

namespace axhip {
int launch_sample_f32(const SampleArgs &a, int64_t rows, hipStream_t s) { return launch<AXHIP_DTYPE_F32>(a, rows, s); }
} // namespace axhip
