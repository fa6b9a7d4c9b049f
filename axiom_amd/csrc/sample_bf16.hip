// Logits in bf16: see sample_kernel.hpp.
#include "sample_kernel.hpp"

namespace axhip {
int launch_sample_bf16(const SampleArgs &a, int64_t rows, hipStream_t s) { return launch<AXHIP_DTYPE_BF16>(a, rows, s); }
} // namespace axhip
