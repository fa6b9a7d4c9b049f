// Products of int8 rows with scales: axhip_gemm_q8.
#include "gemm_q8.hpp"
#include "gemm_skinny.hpp"

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
        float y = static_cast<float>(acc) * (g.scale_a[m] * g.scale_b[n]);
        if (g.bias) y += load_any(g.bias, g.dtype, n);
        if (g.residual) y += load_any(g.residual, g.dtype, m * g.ldc + n);
        store_any(g.c, g.dtype, m * g.ldc + n, gemm_epilogue(g.epilogue, y));
    }
}

// Within the 32-bit offsets the matrix-core kernels address with, and a whole chunk of k.
bool takes_q8_kernels(const AxhipGemmQ8Params &p) {
    constexpr int64_t LD = int64_t(1) << 22;
    return p.k >= 16 && p.lda < LD && p.ldb < LD && p.ldc < (int64_t(1) << 31);
}

// The candidates with the time each takes, in us: start + k (per_k + per_k_full u) r + per_round (r - 1), r being the rounds its work-groups take on
// the 256 CUs and u how full the first is.
struct Q8Kernel {
    enum Kind { BIG256, TILE, PAIR, SMALL } kind;
    int shape, waves;
    float start, per_k, per_k_full, per_round;
    bool ragged;
    const char *name;
};
constexpr Q8Kernel Q8_KERNELS[] = {
    {Q8Kernel::BIG256, 0, 8, 7.0f, 0.0160f, 0.0057f, 4.0f, false, "big"},
    {Q8Kernel::TILE, TILE_256x128, 8, 6.5f, 0.0080f, 0.0034f, 6.4f, false, "tile_256x128"},
    {Q8Kernel::TILE, TILE_192x128, 8, 5.7f, 0.0063f, 0.0024f, 4.9f, false, "tile_192x128"},
    {Q8Kernel::TILE, TILE_128x128, 8, 4.9f, 0.0048f, 0.0014f, 4.1f, false, "tile_128x128"},
    {Q8Kernel::TILE, TILE_64x128, 8, 4.9f, 0.0032f, 0.0009f, 3.7f, false, "tile_64x128"},
    {Q8Kernel::TILE, TILE_128x128, 8, 6.5f, 0.0080f, 0.0f, 5.9f, true, "tile_128x128_ragged"},
    {Q8Kernel::PAIR, Q8_128x128_PAIR, 4, 4.9f, 0.0048f, 0.0014f, 4.1f, false, "tile_128x128_pair"},
    {Q8Kernel::SMALL, SMALL_64x64, 8, 4.35f, 0.00245f, 0.00148f, 3.6f, false, "small_64x64_8"},
    {Q8Kernel::SMALL, SMALL_64x64, 4, 4.15f, 0.00324f, 0.00047f, 1.65f, false, "small_64x64_4"},
    {Q8Kernel::SMALL, SMALL_32x64, 8, 3.50f, 0.00170f, 0.00085f, 2.3f, false, "small_32x64_8"},
    {Q8Kernel::SMALL, SMALL_32x64, 4, 3.30f, 0.00210f, 0.00030f, 0.6f, false, "small_32x64_4"},
    {Q8Kernel::SMALL, SMALL_32x32, 8, 3.07f, 0.00105f, 0.00045f, 0.76f, false, "small_32x32_8"},
    {Q8Kernel::SMALL, SMALL_32x32, 4, 2.95f, 0.00148f, 0.00005f, 0.26f, false, "small_32x32_4"},
    {Q8Kernel::SMALL, SMALL_32x16, 8, 2.92f, 0.00074f, 0.00032f, 0.33f, false, "small_32x16_8"},
    {Q8Kernel::SMALL, SMALL_32x16, 4, 2.91f, 0.00102f, 0.00004f, 0.10f, false, "small_32x16_4"},
    {Q8Kernel::SMALL, SMALL_16x16, 8, 2.95f, 0.00045f, 0.00024f, 0.19f, false, "small_16x16_8"},
    {Q8Kernel::SMALL, SMALL_16x16, 4, 2.94f, 0.00069f, 0.00004f, 0.02f, false, "small_16x16_4"},
};
constexpr size_t Q8_CANDIDATES = sizeof(Q8_KERNELS) / sizeof(Q8_KERNELS[0]);

struct Q8Choice { const Q8Kernel *best; float cost; };
// One candidate.  (A parameter of the template, so that its tiles are constants here: divisions by what a table holds cost a small product's caller.)
template <size_t I> void consider(const AxhipGemmQ8Params &p, bool aligned, Q8Choice &c) {
    constexpr const Q8Kernel &h = Q8_KERNELS[I];
    if (h.kind != Q8Kernel::SMALL && h.ragged == aligned) return;
    if (h.kind == Q8Kernel::BIG256 && (p.k % 128 != 0 || p.m < 256 || p.n < 256)) return;
    constexpr uint32_t tm = h.kind == Q8Kernel::BIG256 ? 256 : h.kind == Q8Kernel::PAIR ? 128 : h.kind == Q8Kernel::TILE ? TILE_GEOMETRY[h.kind == Q8Kernel::TILE ? h.shape : 0].tm : SMALL_GEOMETRY[h.kind == Q8Kernel::SMALL ? h.shape : 0].tm;
    constexpr uint32_t tn = h.kind == Q8Kernel::BIG256 ? 256 : h.kind == Q8Kernel::PAIR ? 128 : h.kind == Q8Kernel::TILE ? TILE_GEOMETRY[h.kind == Q8Kernel::TILE ? h.shape : 0].tn : SMALL_GEOMETRY[h.kind == Q8Kernel::SMALL ? h.shape : 0].tn;
    const uint32_t rows = (static_cast<uint32_t>(p.m) + tm - 1) / tm, cols = (static_cast<uint32_t>(p.n) + tn - 1) / tn;
    if (!launch_fits(static_cast<int64_t>(rows) * cols + 7, 64 * h.waves)) return;
    const float k = static_cast<float>((p.k + 127) / 128 * 64);
    const float full = static_cast<float>(rows) * static_cast<float>(cols) * (1.0f / 256.0f);
    float r = 1.0f;
    if (full > 1.0f) {
        float whole = full < 1e9f ? static_cast<float>(static_cast<int>(full)) : full;
        if (whole < full) whole += 1.0f;
        r = h.kind == Q8Kernel::SMALL ? 0.5f * (whole + full) : whole;
    }
    const float slower = aligned ? 1.0f : h.kind == Q8Kernel::SMALL ? 1.5f : 1.0f;
    const float cost = h.start + k * (h.per_k + h.per_k_full * std::min(full, 1.0f)) * slower * r + h.per_round * (r - 1.0f);
    if (!c.best || cost < c.cost) c = {&h, cost};
}
template <size_t... I> const Q8Kernel *choose(const AxhipGemmQ8Params &p, bool aligned, std::index_sequence<I...>) {
    Q8Choice c{nullptr, 0.0f};
    (consider<I>(p, aligned, c), ...);
    return c.best;
}

int launch_chosen(const Q8Args &g, const AxhipGemmQ8Params &p, bool aligned, hipStream_t s) {
    if (p.m <= 8) {
        q8_last_kernel = "skinny";
        return launch_q8_skinny(g, p.dtype, 1, s);
    }
    const Q8Kernel *k = choose(p, aligned, std::make_index_sequence<Q8_CANDIDATES>{});
    AXHIP_REQUIRE(k != nullptr, AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
    q8_last_kernel = k->name;
    if (k->kind == Q8Kernel::BIG256) return launch_q8_big(g, p.dtype, s);
    if (k->kind == Q8Kernel::SMALL) return launch_q8_small(g, p.dtype, k->shape, k->waves, s);
    return p.dtype == AXHIP_DTYPE_F32 ? launch_q8_tile_f32(g, k->shape, aligned, s) : p.dtype == AXHIP_DTYPE_F16 ? launch_q8_tile_f16(g, k->shape, aligned, s) : launch_q8_tile_bf16(g, k->shape, aligned, s);
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
