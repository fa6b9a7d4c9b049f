// Shared by gemm_q8.hip and the gemm_q8_*.hip translation units: products of int8 rows with scales.
#pragma once
#include "gemm_small.hpp"

namespace axhip {

// Kernel arguments.  Kept within 96 bytes, as those of the other products.
struct Q8Args {
    const int8_t *a, *b;
    void *c;
    const void *bias, *residual;
    const float *scale_a, *scale_b;
    int M, N, K, lda, ldb, ldc;
    int epilogue;
};
static_assert(sizeof(Q8Args) <= 96, "kernel arguments");

// The launchers.  The tiles are those of the 16-bit products (TileShape, SmallShape): a k of int8 is half as many bytes, so their k-tiles
// hold twice as many k.  `aligned`: every row of a and b starts on a 16-byte boundary and K is a multiple of 16.  All but the skinny kernel's
// grid are their own; K >= 16 for all.
// one more tile: 128 x 128 on four wavefronts, of which a CU holds two work-groups
constexpr int Q8_128x128_PAIR = TILE_SHAPES;

int launch_q8_big(const Q8Args &g, int dtype, hipStream_t s);  // 256 x 256: aligned, K a multiple of 128
int launch_q8_tile_f32(const Q8Args &g, int shape, bool aligned, hipStream_t s); // (not aligned: TILE_128x128)
int launch_q8_tile_f16(const Q8Args &g, int shape, bool aligned, hipStream_t s);
int launch_q8_tile_bf16(const Q8Args &g, int shape, bool aligned, hipStream_t s);
int launch_q8_small(const Q8Args &g, int dtype, int shape, int waves, hipStream_t s);
int launch_q8_skinny(const Q8Args &g, int dtype, int rows_per_wave, hipStream_t s); // M <= 8

} // namespace axhip
