// Large products of int8 rows: 256 x 256 tiles.
#include "gemm_q8_device.hpp"

namespace axhip {
namespace {

constexpr int BIG = 256, ROWB = 128, TILEB = BIG * ROWB; // rows and columns of a tile; bytes of an LDS row; 32 KiB per k-tile of A or B

// Work-group tile 256 x 256, k-tiles of 128, 8 wavefronts in a 2 x 4 layout, each owning 128 x 64 of C as 8 x 4 tiles of v_mfma_i32_16x16x64_i8: the
// schedule of the 16-bit kernel of this size, on the same bytes.  A and B k-tiles go L2 -> LDS directly into two 64 KiB buffers, one barrier per
// k-tile; a k-tile is two k-steps of 32 MFMAs.  The A fragments are single-buffered: the registers of fragment row i are refilled for the next
// k-step right behind the row's fourth MFMA; the B fragments are double-buffered.  Every LDS read and every global load sits between two MFMAs.  The barrier comes
// after the first fragment row of the second k-step: by then every wavefront has read the whole tile, so the buffer takes the tile after next and
// the reads turn to the next tile.
template <int DT>
__global__ __launch_bounds__(512, 1) void gemm_q8_big_kernel(const Q8Args g) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char big_lds[]; // A0 B0 A1 B1
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
    const int l16 = lane % 16, g4 = lane / 16;
    const int tiles_m = (g.M + BIG - 1) / BIG, tiles_n = (g.N + BIG - 1) / BIG;
    int product;
    const int t = tile_of_work_group(tiles_m * tiles_n, 1, product);
    if (t < 0) return;
    constexpr int GR = 4; // the tiles run down groups of 4 tile rows
    const int group = t / (GR * tiles_n), first_m = group * GR;
    const int gsz = min(GR, tiles_m - first_m);
    const int rem = t - group * GR * tiles_n;
    const int m0 = (first_m + rem % gsz) * BIG, n0 = (rem / gsz) * BIG;
    const int rows_a = min(BIG, g.M - m0), rows_b = min(BIG, g.N - n0);
    const int4_t arsrc = tile_rsrc(g.a + static_cast<int64_t>(m0) * g.lda, __builtin_amdgcn_readfirstlane((rows_a - 1) * g.lda + g.K));
    const int4_t brsrc = tile_rsrc(g.b + static_cast<int64_t>(n0) * g.ldb, __builtin_amdgcn_readfirstlane((rows_b - 1) * g.ldb + g.K));

    // L2 -> LDS: one wave-wide load moves 8 rows of 128 bytes; load n of wavefront w covers tile rows 64 n + 8 w + (lane >> 3); the lane fetches the
    // chunk that belongs at position lane & 7 of the swizzled row
    const int ld_r = 8 * wave + (lane >> 3), ld_c = (lane & 7) ^ ((ld_r >> 1) & 7);
    int a_voff[4], b_voff[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        a_voff[n] = (64 * n + ld_r) * g.lda + ld_c * 16;
        b_voff[n] = (64 * n + ld_r) * g.ldb + ld_c * 16;
    }
    const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(big_lds)) + 8 * wave * ROWB);
    auto load_one = [&](const int4_t &ar, const int4_t &br, int kt, int buf, int n) __attribute__((always_inline)) { // n: 0..3 of A, 4..7 of B
        if (n < 4) tile_load_to_lds(ar, lds_wave + buf * 2 * TILEB + n * 64 * ROWB, a_voff[n % 4], kt * ROWB);
        else tile_load_to_lds(br, lds_wave + buf * 2 * TILEB + TILEB + (n - 4) * 64 * ROWB, b_voff[n % 4], kt * ROWB);
    };

    const int wm = (wave / 4) * 128, wn = (wave % 4) * 64;
    Q8Scales<DT, 8> scales;
    scales.load(g, m0 + wm, n0 + wn, lane);
    int f_off[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) f_off[s] = l16 * ROWB + (((4 * s + g4) ^ ((l16 >> 1) & 7)) * 16);
    int4_t acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = int4_t{0, 0, 0, 0};
    uint4_t fa[8], fb[2][4];
    auto read_a = [&](int buf, int s, int i) __attribute__((always_inline)) { fa[i] = *reinterpret_cast<const uint4_t *>(big_lds + buf * 2 * TILEB + (wm + 16 * i) * ROWB + f_off[s]); };
    auto read_b = [&](int slot, int buf, int s, int j) __attribute__((always_inline)) {
        fb[slot][j] = *reinterpret_cast<const uint4_t *>(big_lds + buf * 2 * TILEB + TILEB + (wn + 16 * j) * ROWB + f_off[s]);
    };
    auto mfma = [&](int slot, int i, int j) __attribute__((always_inline)) { acc[i][j] = q8_mfma(fb[slot][j], fa[i], acc[i][j]); };
#define AXHIP_FENCE() __builtin_amdgcn_sched_barrier(0)

    const int nk = g.K / ROWB;
#pragma unroll
    for (int n = 0; n < 8; ++n) load_one(arsrc, brsrc, 0, 0, n);
    if (nk > 1) {
#pragma unroll
        for (int n = 0; n < 8; ++n) load_one(arsrc, brsrc, 1, 1, n);
        __builtin_amdgcn_s_waitcnt(0x0F78); // vmcnt(8): tile 0 has landed
    } else {
        __builtin_amdgcn_s_waitcnt(0x0F70); // vmcnt(0)
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) read_a(0, 0, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) read_b(0, 0, 0, j);
    for (int kt = 0; kt < nk; ++kt) {
        const int buf = kt & 1;
        // past the last tile the loads run on empty descriptors (every lane out of range: zeros into a buffer nobody reads, no memory traffic) rather
        // than behind eight branches
        const bool more = kt + 2 < nk;
        const int4_t ar = int4_t{arsrc.x, arsrc.y, more ? arsrc.z : 0, arsrc.w}, br = int4_t{brsrc.x, brsrc.y, more ? brsrc.z : 0, brsrc.w};
        AXHIP_FENCE();
        // k-step 0: B slot 0; the refills fetch k-step 1 of this tile
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mfma(0, i, j);
                AXHIP_FENCE();
                if (j == 2 && i < 4) {
                    read_b(1, buf, 1, i);
                    AXHIP_FENCE();
                }
                if (j == 3) {
                    read_a(buf, 1, i);
                    AXHIP_FENCE();
                }
            }
        // k-step 1: B slot 1; behind the barrier the refills fetch k-step 0 of the next tile (after the last tile: a harmless read of stale LDS) and
        // this tile's buffer takes the tile after next
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i == 1) {
                __builtin_amdgcn_s_waitcnt(0x0F70); // this wavefront's share of tile kt + 1 has landed
                __syncthreads();                    // ... everyone's has, and tile kt is no longer read
                AXHIP_FENCE();
                read_a(buf ^ 1, 0, 0);
                AXHIP_FENCE();
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mfma(1, i, j);
                AXHIP_FENCE();
                if (i >= 1) {
                    const int q = (i - 1) * 4 + j; // MFMAs since the barrier
                    if (q % 3 == 1 && q / 3 < 8) {
                        load_one(ar, br, kt + 2, buf, q / 3);
                        AXHIP_FENCE();
                    }
                    if (q % 2 == 0 && q >= 2 && q <= 8) {
                        read_b(0, buf ^ 1, 0, q / 2 - 1);
                        AXHIP_FENCE();
                    }
                    if (j == 3) {
                        read_a(buf ^ 1, 0, i);
                        AXHIP_FENCE();
                    }
                }
            }
        }
    }
#undef AXHIP_FENCE

    // the tile buffers become the staging area of the epilogue: no load of this work-group is still on its way into them (past the last tile they
    // write zeros), and every wavefront has its last fragments
    Q8Residual<DT, 4> res;
    res.load(g, m0 + wm, n0 + wn, lane);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    q8_store_pieces<DT, 8, 4>(g, acc, scales, res, m0 + wm, n0 + wn, lane, big_lds + wave * 16384);
}

template <int DT> int launch(const Q8Args &g, hipStream_t s) {
    constexpr int lds = 4 * TILEB;
    static const hipError_t configured = hipFuncSetAttribute(reinterpret_cast<const void *>(&gemm_q8_big_kernel<DT>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    AXHIP_CHECK_HIP(configured);
    const int64_t tiles = static_cast<int64_t>((g.M + BIG - 1) / BIG) * ((g.N + BIG - 1) / BIG);
    AXHIP_REQUIRE(launch_fits(tiles + 7, 512), AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
    hipLaunchKernelGGL(gemm_q8_big_kernel<DT>, dim3(tile_grid(tiles, 1)), dim3(512), lds, s, g);
    return AXHIP_OK;
}
} // namespace

int launch_q8_big(const Q8Args &g, int dtype, hipStream_t s) {
    return dtype == AXHIP_DTYPE_F32 ? launch<AXHIP_DTYPE_F32>(g, s) : dtype == AXHIP_DTYPE_F16 ? launch<AXHIP_DTYPE_F16>(g, s) : launch<AXHIP_DTYPE_BF16>(g, s);
}
} // namespace axhip
