// A decoding step with prefixes, 16 bits: the tiles of the prefixes and the shares of the own keys in one launch, so that what is bound by the matrix pipe and by a chain of latencies
// runs beside what is bound by memory: 64 sequences of 300 keys behind 8192, 32 heads on 8 of 128 dims, 44.5 us with the join (two launches one behind the other: 58).
#pragma once

#include "sdpa_rows.hpp"
#include "sdpa_tile.hpp"

namespace axhip {

template <bool BF16, int D, int DE, bool PAD>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void sdpa_step_kernel(const CacheArgs a, int prefix_blocks) {
    if (static_cast<int>(blockIdx.x) < prefix_blocks) tile_body<BF16, D, DE, 4, TILE_PREFIX>(a, blockIdx.x);
    else rows_body<BF16 ? AXHIP_DTYPE_BF16 : AXHIP_DTYPE_F16, D, PAD, ROWS_OWN>(a, blockIdx.x - prefix_blocks);
}

template <bool BF16, int D, int DE, bool PAD> int launch_step_as(const CacheArgs &a, hipStream_t s) {
    constexpr int tile = 4 * TK * 2 * D, lds = tile > rows_lds_bytes<D>() ? tile : rows_lds_bytes<D>();
    if constexpr (lds > 65536) {
        static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(&sdpa_step_kernel<BF16, D, DE, PAD>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        AXHIP_CHECK_HIP(attr);
    }
    const int64_t prefix = (static_cast<int64_t>(a.entries) * a.new_tokens * a.each / 128 + a.groups) * a.parts * a.kv_heads, all = prefix + own_blocks(a); // at most
    AXHIP_REQUIRE(launch_fits(all, 256), AXHIP_ERR_UNSUPPORTED, "axhip_sdpa_paged: grid too large");
    hipLaunchKernelGGL((sdpa_step_kernel<BF16, D, DE, PAD>), dim3(static_cast<unsigned>(all)), dim3(256), lds, s, a, static_cast<int>(prefix));
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}
template <bool BF16> int launch_step(const CacheArgs &a, hipStream_t s) {
    if (a.D == 64) return launch_step_as<BF16, 64, 64, false>(a, s);
    if (a.D == 128) return launch_step_as<BF16, 128, 128, false>(a, s);
    if (a.D < 64) return launch_step_as<BF16, 64, 64, true>(a, s);
    if (a.D <= 96) return launch_step_as<BF16, 128, 96, true>(a, s);
    if (a.D < 128) return launch_step_as<BF16, 128, 128, true>(a, s);
    return launch_step_as<BF16, 256, 256, true>(a, s);
}

} // namespace axhip
