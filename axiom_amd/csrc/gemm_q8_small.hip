// Products of int8 rows with few rows or few output tiles: see the kernel's comment.
#include "gemm_q8_device.hpp"

namespace axhip {
namespace {

// The W wavefronts' sums meet in LDS; scales, bias, residual, activation, store.
template <int DT, int MI, int NJ, int W>
__device__ __forceinline__ void small_finish(const Q8Args &g, const int4_t (&acc)[MI][NJ], int m0, int n0, unsigned char *lds) {
    constexpr int F = MI * NJ;
    const int tid = threadIdx.x, wave = tid / WAVE, lane = tid % WAVE;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) *reinterpret_cast<int4_t *>(lds + ((wave * F + i * NJ + j) * 64 + lane) * 16) = acc[i][j];
    __syncthreads();
    for (int x = tid; x < F * 64; x += 64 * W) {
        const int f = x / 64, row = m0 + 16 * (f / NJ) + (x % 16), col = n0 + 16 * (f % NJ) + 4 * ((x % 64) / 16);
        int4_t v = *reinterpret_cast<const int4_t *>(lds + x * 16);
#pragma unroll
        for (int w = 1; w < W; ++w) v += *reinterpret_cast<const int4_t *>(lds + (w * F * 64 + x) * 16);
        const int last = min(4, g.N - col);
        if (row >= g.M || last <= 0) continue;
        float b[4], sb[4];
        int sum[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum[e] = v[e];
            sb[e] = e < last ? g.scale_b[col + e] : 0.0f;
            b[e] = g.bias && e < last ? Elem<DT>::load(g.bias, col + e) : 0.0f;
        }
        q8_finish<DT, 4>(g, sum, g.scale_a[row], sb, b, static_cast<int64_t>(row) * g.ldc + col, last);
    }
}

// C = A B^T, any alignment: work-group tile 16 MI x 16 NJ, W wavefronts that split k between them (wavefront w takes the pieces of 128 k
// w, w + W, ...) and meet in LDS once, at the end.  Such products are bound by latency: every wavefront has a stage of LDS of its own and waits for
// nobody until the sums are added, and the tile is as narrow as it takes to give every CU work.  A piece travels through registers, the next one's loads in flight while one is
// multiplied; the loads need no alignment, and the last chunk of a row is fetched as the 16 bytes that end with it and shifted into place.  64 x 4096 x 4096 6.2 us (17 MB: 3.4 at a copy's rate).
template <int DT, int MI, int NJ, int W>
__global__ __launch_bounds__(64 * W) void gemm_q8_small_kernel(const Q8Args g) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char small_lds[];
    constexpr int NL = 2 * (MI + NJ), NA = 2 * MI, STAGEB = NL * 1024;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
    const int l16 = lane % 16, g4 = lane / 16;
    const int tiles_m = (g.M + 16 * MI - 1) / (16 * MI);
    int product;
    const int t = tile_of_work_group(tiles_m * ((g.N + 16 * NJ - 1) / (16 * NJ)), 1, product);
    if (t < 0) return;
    const int m0 = (t % tiles_m) * 16 * MI, n0 = (t / tiles_m) * 16 * NJ;
    const int8_t *A = g.a + static_cast<int64_t>(m0) * g.lda, *B = g.b + static_cast<int64_t>(n0) * g.ldb;
    const int rows_a = min(16 * MI, g.M - m0), rows_b = min(16 * NJ, g.N - n0);
    const int ld_r = lane >> 3;
    unsigned char *st = small_lds + wave * STAGEB;

    int src[NL];      // the chunk of its row that a lane's load n fetches: the one that belongs at position lane & 7
    uint32_t off[NL]; // and where the row starts (rows past the end repeat the last one: they are not stored)
#pragma unroll
    for (int n = 0; n < NL; ++n) {
        const int row = 8 * (n < NA ? n : n - NA) + ld_r;
        src[n] = (lane & 7) ^ ((row >> 1) & 7);
        off[n] = n < NA ? static_cast<uint32_t>(min(row, rows_a - 1)) * g.lda : static_cast<uint32_t>(min(row, rows_b - 1)) * g.ldb;
    }
    uint4_t regs[NL];
    auto load = [&](int piece) { // (past the end of k: the row's end again)
#pragma unroll
        for (int n = 0; n < NL; ++n) regs[n] = q8_load_chunk((n < NA ? A : B) + (off[n] + static_cast<uint32_t>(min(128 * piece + 16 * src[n], g.K - 16))));
    };
    int4_t acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = int4_t{0, 0, 0, 0};
    const int pieces = (g.K + 127) / 128;
    load(wave);
#pragma unroll 1
    for (int p = wave; p < pieces; p += W) {
        if (128 * (p + 1) > g.K) {
#pragma unroll
            for (int n = 0; n < NL; ++n) regs[n] = q8_chunk_in_place(regs[n], 128 * p + 16 * src[n], g.K);
        }
#pragma unroll
        for (int n = 0; n < NL; ++n) *reinterpret_cast<uint4_t *>(st + n * 1024 + lane * 16) = regs[n];
        if (p + W < pieces) load(p + W);
        wave_lds_fence();
        uint4_t fa[2][MI], fb[2][NJ];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MI; ++i) fa[h][i] = *reinterpret_cast<const uint4_t *>(st + (16 * i + l16) * 128 + (((4 * h + g4) ^ ((l16 >> 1) & 7)) * 16));
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[h][j] = *reinterpret_cast<const uint4_t *>(st + MI * 2048 + (16 * j + l16) * 128 + (((4 * h + g4) ^ ((l16 >> 1) & 7)) * 16));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = q8_mfma(fb[h][j], fa[h][i], acc[i][j]);
        wave_lds_fence();
    }
    __syncthreads();
    small_finish<DT, MI, NJ, W>(g, acc, m0, n0, small_lds);
}

template <int DT, int MI, int NJ, int W> int launch_kernel(const Q8Args &g, hipStream_t s) {
    constexpr int stages = W * (MI + NJ) * 2048, sums = W * MI * NJ * 1024, lds = stages > sums ? stages : sums;
    const auto kernel = gemm_q8_small_kernel<DT, MI, NJ, W>;
    static const hipError_t configured = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    AXHIP_CHECK_HIP(configured);
    const int64_t tiles = static_cast<int64_t>((g.M + 16 * MI - 1) / (16 * MI)) * ((g.N + 16 * NJ - 1) / (16 * NJ));
    AXHIP_REQUIRE(launch_fits(tiles + 7, 64 * W), AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
    hipLaunchKernelGGL(kernel, dim3(tile_grid(tiles, 1)), dim3(64 * W), lds, s, g);
    return AXHIP_OK;
}
template <int DT, int MI, int NJ> int launch_waves(const Q8Args &g, int waves, hipStream_t s) { return waves == 8 ? launch_kernel<DT, MI, NJ, 8>(g, s) : launch_kernel<DT, MI, NJ, 4>(g, s); }
template <int DT> int launch_shape(const Q8Args &g, int shape, int waves, hipStream_t s) {
    switch (shape) {
    case SMALL_16x16: return launch_waves<DT, 1, 1>(g, waves, s);
    case SMALL_32x16: return launch_waves<DT, 2, 1>(g, waves, s);
    case SMALL_32x32: return launch_waves<DT, 2, 2>(g, waves, s);
    case SMALL_32x64: return launch_waves<DT, 2, 4>(g, waves, s);
    default: return launch_waves<DT, 4, 4>(g, waves, s);
    }
}
} // namespace

int launch_q8_small(const Q8Args &g, int dtype, int shape, int waves, hipStream_t s) {
    return dtype == AXHIP_DTYPE_F32 ? launch_shape<AXHIP_DTYPE_F32>(g, shape, waves, s) : dtype == AXHIP_DTYPE_F16 ? launch_shape<AXHIP_DTYPE_F16>(g, shape, waves, s) : launch_shape<AXHIP_DTYPE_BF16>(g, shape, waves, s);
}
} // namespace axhip
