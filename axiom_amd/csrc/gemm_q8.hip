// Products of int8 rows with scales: axhip_gemm_q8.
#include "gemm_skinny.hpp"

namespace axhip {
namespace {
thread_local const char *q8_last_kernel = "none";

struct Q8Args {
    const int8_t *a, *b;
    void *c;
    const float *scale_a, *scale_b;
    const void *bias, *residual;
    int64_t M, N, K, lda, ldb, ldc;
    int dtype, epilogue;
};

// Any size and alignment: a work-group owns 16 x 16 of C, k goes through LDS.
__global__ __launch_bounds__(256) void gemm_q8_generic_kernel(const Q8Args g, int64_t tiles_n) {
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
    const Q8Args g{a, b, c, p.scale_a, p.scale_b, p.bias, p.residual, p.m, p.n, p.k, p.lda, p.ldb, p.ldc, p.dtype, p.epilogue_op};
    const int64_t tiles_n = (p.n + 15) / 16, tiles = (p.m + 15) / 16 * tiles_n;
    AXHIP_REQUIRE(launch_fits(tiles, 256), AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
    hipLaunchKernelGGL(gemm_q8_generic_kernel, dim3(static_cast<unsigned>(tiles)), dim3(256), 0, s, g, tiles_n);
    q8_last_kernel = "generic";
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}

extern "C" const char *axhip_gemm_q8_last_kernel(void) { return q8_last_kernel; }
