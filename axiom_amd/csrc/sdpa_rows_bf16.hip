#include "sdpa_rows.hpp"
namespace axhip {
int launch_rows_own_bf16(const CacheArgs &a, hipStream_t s) { return launch_rows_own<AXHIP_DTYPE_BF16>(a, s); }
int launch_rows_whole_bf16(const CacheArgs &a, hipStream_t s) { return launch_rows_whole<AXHIP_DTYPE_BF16>(a, s); }
int launch_rows_packed_bf16(const CacheArgs &a, hipStream_t s) { return launch_rows_packed<AXHIP_DTYPE_BF16>(a, s); }
int launch_join_bf16(const CacheArgs &a, hipStream_t s) { return launch_join<AXHIP_DTYPE_BF16>(a, s); }
} // namespace axhip
