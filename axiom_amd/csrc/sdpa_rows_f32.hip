#include "sdpa_rows.hpp"
namespace axhip {
int launch_rows_own_f32(const CacheArgs &a, hipStream_t s) { return launch_rows_own<AXHIP_DTYPE_F32>(a, s); }
int launch_rows_whole_f32(const CacheArgs &a, hipStream_t s) { return launch_rows_whole<AXHIP_DTYPE_F32>(a, s); }
int launch_join_f32(const CacheArgs &a, hipStream_t s) { return launch_join<AXHIP_DTYPE_F32>(a, s); }
int launch_rows_packed_f32(const CacheArgs &a, bool apart, hipStream_t s) {
    if (!apart) return launch_rows_packed<AXHIP_DTYPE_F32>(a, s);
    return launch_rows_mode<AXHIP_DTYPE_F32, ROWS_APART>(a, (a.total_q * a.each / (ROWS * ROWS_WAVES) + a.entries) * a.kv_heads, s);
}
int launch_prefix_f32(const CacheArgs &a, hipStream_t s) {
    return launch_rows_mode<AXHIP_DTYPE_F32, ROWS_PREFIX>(a, (static_cast<int64_t>(a.entries) * a.new_tokens * a.each / ROWS + a.groups) * a.parts * a.kv_heads, s);
}
} // namespace axhip
