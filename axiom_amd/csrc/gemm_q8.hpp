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

// Work-group tiles (M x N) of the middle-sized and large products.  Q8_128x128_PAIR: on four wavefronts, of which a CU holds two work-groups.
enum Q8Tile { Q8_256x256, Q8_256x128, Q8_192x128, Q8_128x128, Q8_128x128_PAIR, Q8_64x128, Q8_TILES };
struct Q8Geometry { int tm, tn; };
constexpr Q8Geometry Q8_GEOMETRY[Q8_TILES] = {{256, 256}, {256, 128}, {192, 128}, {128, 128}, {128, 128}, {64, 128}};

// The launchers, K >= 16.  `aligned`: every row of a and b starts on a 16-byte boundary and K is a multiple of 16 (if not: Q8_128x128, through registers).  The small products' tiles are
// those of the 16-bit ones (SmallShape).
int launch_q8_tile_f32(const Q8Args &g, int tile, bool aligned, hipStream_t s);
int launch_q8_tile_f16(const Q8Args &g, int tile, bool aligned, hipStream_t s);
int launch_q8_tile_bf16(const Q8Args &g, int tile, bool aligned, hipStream_t s);
int launch_q8_small(const Q8Args &g, int dtype, int shape, int waves, hipStream_t s);
int launch_q8_skinny(const Q8Args &g, int dtype, int rows_per_wave, hipStream_t s); // M 1 or 2; 1 or 2 rows of b to a wavefront

} // namespace axhip
