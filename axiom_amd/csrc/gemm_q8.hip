// Products of int8 rows with scales: axhip_gemm_q8.
#include "gemm_q8_device.hpp"

#include <algorithm>
#include <utility>

namespace axhip {
namespace {
thread_local const char *q8_last_kernel = "none";

struct GenericArgs {
    const int8_t *a, *b;
    void *c;
    const float *scale_a, *scale_b;
    const void *bias, *residual;
    int64_t M, N, K, lda, ldb, ldc;
    int dtype, epilogue;
};

// Any size and alignment: a work-group owns 16 x 16 of C, k goes through LDS.
__global__ __launch_bounds__(256) void gemm_q8_generic_kernel(const GenericArgs g, int64_t tiles_n) {
    __shared__ int8_t As[16][68], Bs[16][68];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t m0 = blockIdx.x / tiles_n * 16, n0 = blockIdx.x % tiles_n * 16;
    int acc = 0;
    for (int64_t k0 = 0; k0 < g.K; k0 += 64) {
        for (int i = tx; i < 64; i += 16) {
            As[ty][i] = m0 + ty < g.M && k0 + i < g.K ? g.a[(m0 + ty) * g.lda + k0 + i] : 0;
            Bs[ty][i] = n0 + ty < g.N && k0 + i < g.K ? g.b[(n0 + ty) * g.ldb + k0 + i] : 0;
        }
        __syncthreads();
        for (int k = 0; k < 64; ++k) acc += As[ty][k] * Bs[tx][k];
        __syncthreads();
    }
    const int64_t m = m0 + ty, n = n0 + tx;
    if (m < g.M && n < g.N) {
        float y[1] = {q8_scaled(acc, g.scale_a[m], g.scale_b[n], g.bias ? load_any(g.bias, g.dtype, n) : 0.0f)};
        if (g.residual) y[0] += load_any(g.residual, g.dtype, m * g.ldc + n);
        if (g.dtype == AXHIP_DTYPE_F32) q8_activation<AXHIP_DTYPE_F32>(g.epilogue, y);
        else if (g.dtype == AXHIP_DTYPE_F16) q8_activation<AXHIP_DTYPE_F16>(g.epilogue, y);
        else q8_activation<AXHIP_DTYPE_BF16>(g.epilogue, y);
        store_any(g.c, g.dtype, m * g.ldc + n, y[0]);
    }
}

// Within the 32-bit offsets the matrix-core kernels address with, and a whole chunk of k.
bool takes_q8_kernels(const AxhipGemmQ8Params &p) {
    constexpr int64_t LD = int64_t(1) << 22;
    return p.k >= 16 && p.lda < LD && p.ldb < LD && p.ldc < (int64_t(1) << 31);
}

// The candidates with the time each takes, in us: start + k (per_k + per_k_full u) r + per_round (r - 1), k in steps of 128, r being the rounds its work-groups
// take on the 256 CUs (whole rounds of the tile kernels, of which a CU holds one, or two of a pair; the small ones share a CU, and a part of a round costs
// about half of what is missing from a whole one) and u how full the first is.  Fitted to 460 products of m 9 .. 8192, n and k 64 .. 8192, results in bfloat16, every
// candidate timed (mean error 5 - 12 %); the one picked takes 1.022 of the fastest one's time on average, 1.26 at worst (303 x 883 x 6416, 14.0 us instead of 11.1).
// The same numbers serve fp32 results, residuals, activations and n beyond 8192, of which none were in the fit.
struct Q8Kernel {
    bool small;
    int tile, waves; // a Q8Tile, or a SmallShape and its wavefronts
    float start, per_k, per_k_full, per_round;
    bool ragged;
    const char *name;
};
constexpr Q8Kernel Q8_KERNELS[] = {
    {false, Q8_256x256, 8, 10.00f, 0.01722f, 0.00783f, 7.45f, false, "tile_256x256"},
    {false, Q8_256x128, 8, 7.85f, 0.00961f, 0.00463f, 6.97f, false, "tile_256x128"},
    {false, Q8_192x128, 8, 6.62f, 0.00736f, 0.00380f, 5.91f, false, "tile_192x128"},
    {false, Q8_128x128, 8, 5.49f, 0.00542f, 0.00339f, 4.63f, false, "tile_128x128"},
    {false, Q8_128x128_PAIR, 4, 5.23f, 0.00909f, 0.00089f, 2.35f, false, "tile_128x128_pair"},
    {false, Q8_64x128, 8, 5.43f, 0.00333f, 0.00156f, 4.48f, false, "tile_64x128"},
    {false, Q8_128x128, 8, 7.55f, 0.00981f, 0.00180f, 6.69f, true, "tile_128x128_ragged"}, // (through registers)
    {true, SMALL_64x64, 8, 4.75f, 0.00246f, 0.00260f, 3.91f, false, "small_64x64_8"},
    {true, SMALL_64x64, 4, 5.09f, 0.00338f, 0.00092f, 2.07f, false, "small_64x64_4"},
    {true, SMALL_32x64, 8, 3.55f, 0.00158f, 0.00160f, 2.49f, false, "small_32x64_8"},
    {true, SMALL_32x64, 4, 3.67f, 0.00207f, 0.00062f, 0.80f, false, "small_32x64_4"},
    {true, SMALL_32x32, 8, 3.28f, 0.00095f, 0.00075f, 0.71f, false, "small_32x32_8"},
    {true, SMALL_32x32, 4, 3.23f, 0.00129f, 0.00049f, 0.22f, false, "small_32x32_4"},
    {true, SMALL_32x16, 8, 3.29f, 0.00054f, 0.00065f, 0.26f, false, "small_32x16_8"},
    {true, SMALL_32x16, 4, 3.28f, 0.00075f, 0.00052f, 0.02f, false, "small_32x16_4"},
    {true, SMALL_16x16, 8, 3.36f, 0.00019f, 0.00053f, 0.08f, false, "small_16x16_8"},
    {true, SMALL_16x16, 4, 3.30f, 0.00040f, 0.00034f, 0.00f, false, "small_16x16_4"},
};
constexpr size_t Q8_CANDIDATES = sizeof(Q8_KERNELS) / sizeof(Q8_KERNELS[0]);
// Rows off the 16-byte grid, or k no whole chunks: what that costs the small kernels per k.
constexpr float Q8_MISALIGNED = 1.8f;

struct Q8Choice { const Q8Kernel *best; float cost; };
// One candidate.  (A parameter of the template, so that its tiles are constants here: divisions by what a table holds cost a small product's caller.)
template <size_t I> void consider(const AxhipGemmQ8Params &p, bool aligned, Q8Choice &c) {
    constexpr const Q8Kernel &h = Q8_KERNELS[I];
    if (!h.small && h.ragged == aligned) return;
    constexpr uint32_t tm = h.small ? SMALL_GEOMETRY[h.small ? h.tile : 0].tm : Q8_GEOMETRY[h.small ? 0 : h.tile].tm;
    constexpr uint32_t tn = h.small ? SMALL_GEOMETRY[h.small ? h.tile : 0].tn : Q8_GEOMETRY[h.small ? 0 : h.tile].tn;
    const uint32_t rows = (static_cast<uint32_t>(p.m) + tm - 1) / tm, cols = (static_cast<uint32_t>(p.n) + tn - 1) / tn;
    if (!launch_fits(static_cast<int64_t>(rows) * cols + 7, 64 * h.waves)) return;
    const float k = static_cast<float>((p.k + 127) / 128 * 64);
    const float full = static_cast<float>(rows) * static_cast<float>(cols) * (1.0f / 256.0f);
    auto whole = [](float x) { // (rounded up)
        const float down = x < 1e9f ? static_cast<float>(static_cast<int>(x)) : x;
        return down < x ? down + 1.0f : down;
    };
    float r = 1.0f;
    if (full > 1.0f) r = h.small ? 0.5f * (whole(full) + full) : !h.ragged && h.tile == Q8_128x128_PAIR ? whole(0.5f * full) + 0.5f * full : whole(full);
    const float cost = h.start + k * (h.per_k + h.per_k_full * std::min(full, 1.0f)) * (h.small && !aligned ? Q8_MISALIGNED : 1.0f) * r + h.per_round * (r - 1.0f);
    if (!c.best || cost < c.cost) c = {&h, cost};
}
template <size_t... I> const Q8Kernel *choose(const AxhipGemmQ8Params &p, bool aligned, std::index_sequence<I...>) {
    Q8Choice c{nullptr, 0.0f};
    (consider<I>(p, aligned, c), ...);
    return c.best;
}

int launch_chosen(const Q8Args &g, const AxhipGemmQ8Params &p, bool aligned, hipStream_t s) {
    // One or two rows of x: the weights are read once, along k (1 x 4096 x 4096 5.2 us, on the small kernels 5.4; 1 x 1280 x 5120 4.1 and 5.3; of three rows and more the small
    // ones take less).  Two rows of W to a wavefront where k is short (51865 x 1280 15.8 -> 11.9 us) or x has two and W is large (2 x 16384 x 16384 52.7 -> 48.2).
    const int rows_per_wave = p.k < 2048 || (p.m == 2 && p.n * p.k >= int64_t(1) << 26) ? 2 : 1;
    if (p.m <= 2 && launch_fits((p.n + 4 * rows_per_wave - 1) / (4 * rows_per_wave), 256)) { // (vocabularies of 2^26 and more go on)
        q8_last_kernel = "skinny";
        return launch_q8_skinny(g, p.dtype, rows_per_wave, s);
    }
    const Q8Kernel *k = choose(p, aligned, std::make_index_sequence<Q8_CANDIDATES>{});
    AXHIP_REQUIRE(k != nullptr, AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
    q8_last_kernel = k->name;
    if (k->small) return launch_q8_small(g, p.dtype, k->tile, k->waves, s);
    return p.dtype == AXHIP_DTYPE_F32 ? launch_q8_tile_f32(g, k->tile, aligned, s) : p.dtype == AXHIP_DTYPE_F16 ? launch_q8_tile_f16(g, k->tile, aligned, s) : launch_q8_tile_bf16(g, k->tile, aligned, s);
}
} // namespace
} // namespace axhip
using namespace axhip;

extern "C" int axhip_gemm_q8(const int8_t *a, const int8_t *b, void *c, const AxhipGemmQ8Params *params, void *stream) {
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: params is NULL");
    const AxhipGemmQ8Params &p = *params;
    AXHIP_REQUIRE(valid_dtype(p.dtype), AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: bad dtype %d", p.dtype);
    constexpr int64_t SIDE = int64_t(1) << 30;
    AXHIP_REQUIRE(p.m >= 0 && p.n >= 0 && p.k >= 0 && p.m < SIDE && p.n < SIDE, AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: bad extent");
    AXHIP_REQUIRE(p.k <= 131071, AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: sums of %lld products may not fit 32 bits (131071 do)", static_cast<long long>(p.k));
    AXHIP_REQUIRE(p.lda >= p.k && p.ldb >= p.k && p.ldc >= p.n, AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: bad leading dimension");
    AXHIP_REQUIRE(p.lda < (SIDE << 10) && p.ldb < (SIDE << 10) && p.ldc < (SIDE << 10), AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: leading dimension too large");
    AXHIP_REQUIRE(p.epilogue_op == 0 || p.epilogue_op == AXHIP_OP_RELU || p.epilogue_op == AXHIP_OP_GELU || p.epilogue_op == AXHIP_OP_SILU ||
                      p.epilogue_op == AXHIP_OP_SIGMOID || p.epilogue_op == AXHIP_OP_TANH,
                  AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: unsupported epilogue op %d", p.epilogue_op);
    q8_last_kernel = "empty";
    if (p.m == 0 || p.n == 0) return AXHIP_OK;
    AXHIP_REQUIRE(c && p.scale_a && p.scale_b && (p.k == 0 || (a && b)), AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: NULL matrix or scales");
    const uintptr_t unit = dtype_size(p.dtype) - 1;
    AXHIP_REQUIRE(((reinterpret_cast<uintptr_t>(c) | reinterpret_cast<uintptr_t>(p.bias) | reinterpret_cast<uintptr_t>(p.residual)) & unit) == 0 &&
                      ((reinterpret_cast<uintptr_t>(p.scale_a) | reinterpret_cast<uintptr_t>(p.scale_b)) & 3u) == 0,
                  AXHIP_ERR_INVALID_ARG, "axhip_gemm_q8: a buffer is not aligned to its elements");
    int rc = ensure_init();
    if (rc) return rc;
    hipStream_t s = resolve_stream(stream);
    if (takes_q8_kernels(p)) {
        const Q8Args g{a, b, c, p.bias, p.residual, p.scale_a, p.scale_b, static_cast<int>(p.m), static_cast<int>(p.n), static_cast<int>(p.k),
                       static_cast<int>(p.lda), static_cast<int>(p.ldb), static_cast<int>(p.ldc), p.epilogue_op};
        const bool aligned = ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) == 0 && (p.k | p.lda | p.ldb) % 16 == 0;
        rc = launch_chosen(g, p, aligned, s);
        if (rc) return rc;
    } else {
        const GenericArgs g{a, b, c, p.scale_a, p.scale_b, p.bias, p.residual, p.m, p.n, p.k, p.lda, p.ldb, p.ldc, p.dtype, p.epilogue_op};
        const int64_t tiles_n = (p.n + 15) / 16, tiles = (p.m + 15) / 16 * tiles_n;
        AXHIP_REQUIRE(launch_fits(tiles, 256), AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
        hipLaunchKernelGGL(gemm_q8_generic_kernel, dim3(static_cast<unsigned>(tiles)), dim3(256), 0, s, g, tiles_n);
        q8_last_kernel = "generic";
    }
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}

extern "C" const char *axhip_gemm_q8_last_kernel(void) { return q8_last_kernel; }
