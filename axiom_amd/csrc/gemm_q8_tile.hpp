// ------------------------------------------------------- middle-sized and large products of int8 rows
// C = A B^T, A [M, K], B [N, K].  Work-group tile TM x TN, k-tiles of TKB bytes in an S-stage ring in LDS; the schedule of the 16-bit tile
// kernel, whose LDS rows and fragments hold the same bytes: v_mfma_i32_16x16x64_i8 takes as many cycles for 64 k of int8 as the 16-bit form does for
// 32 k, and reads as many bytes.
//   * two wavefronts per SIMD, which split the k-tile: WK groups of wavefronts each own whole 16 MI x 64 blocks for a part of every k-tile, and
//     their sums (integers: the order does not matter) meet in LDS once, at the end.
//   * every LDS read and every tile load sits between two MFMAs (scheduling fences pin the order); A fragments are refilled behind their row's last
//     MFMA, B fragments are double-buffered.  The barrier sits after the first fragment row of a k-tile's last k-step: by then every wavefront has
//     read the whole tile, so its stage takes the tile S ahead, and the reads turn to the next tile.
//   * the 16-byte chunk index of an LDS row is XOR-ed by the row.
// DMA: tiles go L2 -> LDS directly (buffer_load ... lds).  Otherwise (rows off the 16-byte grid, K no whole chunks) through registers: unaligned
// 16-byte loads of one tile in flight while the previous is multiplied; the last chunk of a row is fetched as the 16 bytes that end with the row and
// shifted into place.
// What bounds it: 8192 x 4096 x 4096 + residual 118 - 133 us (2.07 - 2.33 POP/s, as the vendor's library): of a 256 x 256 tile's 3100 cycles per k-tile of 128 the matrix pipe is busy
// for 2048 and LDS as long.  Two work-groups per CU, deeper rings, 64-byte k-tiles, priorities of wavefronts and a residual fetched into L2 ahead changed nothing or cost 10 %.
// 1500 x 5120 x 1280 + GELU 17.6 - 18.9 us by card: one round of 240 work-groups, of which launch, first loads and epilogue are about 9 (0.6 of them the exponentials of GELU).
#pragma once
#include "gemm_q8_device.hpp"

#include <type_traits>

namespace axhip {
namespace {

template <int DT, bool DMA, int MI, int WM, int WN, int WK, int TKB, int S>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void gemm_q8_tile_kernel(const Q8Args g) {
    constexpr int NW = WM * WN * WK, TM = 16 * MI * WM, TN = 64 * WN;
    constexpr int KS = TKB / 64 / WK;         // k-steps of 64 per k-tile and wavefront
    constexpr int CH = TKB / 16;              // 16-byte chunks per LDS row
    constexpr int STAGEB = (TM + TN) * TKB, ABYTES = TM * TKB;
    constexpr int NLA = TM * TKB / 1024 / NW, NLB = TN * TKB / 1024 / NW, NL = NLA + NLB; // 1 KiB loads per wavefront and k-tile
    static_assert(KS >= 1 && NLA >= 1 && NLB >= 1 && MI >= 4 && MI % WK == 0, "tile");
    static_assert((NW * 64 / CH) % 16 == 0, "the XOR of a lane's row must not depend on the load");
    extern __shared__ __attribute__((aligned(1024))) unsigned char tile_lds[];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / WAVE), lane = tid % WAVE;
    const int l16 = lane % 16, g4 = lane / 16;
    const int wk = wave / (WM * WN), wt = wave % (WM * WN), wm = (wt / WN) * 16 * MI, wn = (wt % WN) * 64;

    // the tiles run down groups of GR tile rows, so that an XCD's L2 sees a compact block of C and each panel of A and B few times
    const int tiles_m = (g.M + TM - 1) / TM, tiles_n = (g.N + TN - 1) / TN;
    int product;
    const int t = tile_of_work_group(tiles_m * tiles_n, 1, product);
    if (t < 0) return;
    constexpr int GR = TM >= 128 ? 4 : 8;
    const int group = t / (GR * tiles_n), first_m = group * GR;
    const int gsz = min(GR, tiles_m - first_m);
    const int rem = t - group * GR * tiles_n;
    const int m0 = (first_m + rem % gsz) * TM, n0 = (rem / gsz) * TN;
    const int8_t *A = g.a + static_cast<int64_t>(m0) * g.lda, *B = g.b + static_cast<int64_t>(n0) * g.ldb;
    const int rows_a = min(TM, g.M - m0), rows_b = min(TN, g.N - n0);

    // row blocks that a wavefront finishes, and stages at a time (of eight in fp32 two: their residual's registers)
    constexpr int MB = MI / WK, MP = MB <= 4 ? MB : DT == AXHIP_DTYPE_F32 ? 2 : 4;
    Q8Scales<DT, MB> scales;
    scales.load(g, m0 + wm + wk * MB * 16, n0 + wn, lane);

    // ---- tile loads: load n of a wavefront moves chunks 64 (n NW + wave) + lane of the tile's LDS image
    const int ld_row = (wave * 64 + lane) / CH, ld_pos = lane % CH;
    auto swizzle = [](int row) { return TKB == 128 ? (row >> 1) & 7 : row & 15; };
    const int ld_src = ld_pos ^ swizzle(ld_row); // the chunk that belongs at this position
    constexpr int STEP = NW * 64 / CH;           // rows between a wavefront's consecutive loads
    constexpr int OUT_OF_RANGE = 0x7FFFFFF0;
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(tile_lds));
    const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(lds_base + wave * 1024);

    // DMA: offsets of this lane's chunks; a row past the tile's valid ones lies past the descriptor's extent
    const int4_t arsrc = tile_rsrc(A, (rows_a - 1) * g.lda + g.K), brsrc = tile_rsrc(B, (rows_b - 1) * g.ldb + g.K);
    int a_voff[NLA], b_voff[NLB];
    if constexpr (DMA) {
#pragma unroll
        for (int n = 0; n < NLA; ++n) a_voff[n] = (ld_row + n * STEP) * g.lda + ld_src * 16;
#pragma unroll
        for (int n = 0; n < NLB; ++n) b_voff[n] = (ld_row + n * STEP) * g.ldb + ld_src * 16;
    }
    auto dma_load = [&](int kt, int stage_off, int n) { // n: 0 .. NLA - 1 of A, then of B; past the last k-tile every lane is out of range
        const int k_left = g.K - kt * TKB, k_at = k_left > 0 ? kt * TKB : 0;
        const bool inside = 16 * ld_src < k_left;
        if (n < NLA) {
            tile_load_to_lds(arsrc, lds_wave + stage_off + n * NW * 1024, inside ? a_voff[n < NLA ? n : 0] : OUT_OF_RANGE, k_at);
        } else {
            const int nb = n - NLA < NLB ? n - NLA < 0 ? 0 : n - NLA : 0;
            tile_load_to_lds(brsrc, lds_wave + stage_off + ABYTES + nb * NW * 1024, inside ? b_voff[nb] : OUT_OF_RANGE, k_at);
        }
    };
    // through registers (rows past the tile's end repeat its last one: they are not stored)
    constexpr int R = DMA ? 1 : 4; // k-tiles in flight in registers
    uint4_t regs[R][NL];
    uint32_t r_off[NL];
    if constexpr (!DMA) {
#pragma unroll
        for (int n = 0; n < NLA; ++n) r_off[n] = static_cast<uint32_t>(min(ld_row + n * STEP, rows_a - 1)) * g.lda;
#pragma unroll
        for (int n = 0; n < NLB; ++n) r_off[NLA + n] = static_cast<uint32_t>(min(ld_row + n * STEP, rows_b - 1)) * g.ldb;
    }
    auto reg_load = [&](int set, int kt, int n) { // (past the last k-tile: the row's end again)
        regs[set][n] = q8_load_chunk((n < NLA ? A : B) + (r_off[n] + static_cast<uint32_t>(min(kt * TKB + 16 * ld_src, g.K - 16))));
    };
    auto chunk_at = [&](int stage_off, int n) { return reinterpret_cast<uint4_t *>(tile_lds + stage_off + (n < NLA ? n : n - NLA) * NW * 1024 + (n < NLA ? 0 : ABYTES) + wave * 1024 + lane * 16); };
    const int nk = (g.K + TKB - 1) / TKB;
    // (k-tiles past the last one, which the unrolled loop multiplies too, are zeros)
    auto reg_write = [&](int set, int kt, int stage_off, int n) { *chunk_at(stage_off, n) = kt < nk ? regs[set][n] : uint4_t{0, 0, 0, 0}; };
    // the last k-tile, where it reaches past the end of k: this lane's chunks, already in LDS, are put in place
    auto mend = [&](int kt, int stage_off) {
        if (!(kt == nk - 1 && nk * TKB > g.K)) return;
#pragma unroll
        for (int n = 0; n < NL; ++n) *chunk_at(stage_off, n) = q8_chunk_in_place(*chunk_at(stage_off, n), kt * TKB + 16 * ld_src, g.K);
    };

    // ---- fragment reads
    int fa_off[KS], fb_off[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const int chunk = ((4 * (wk * KS + s) + g4) ^ swizzle(l16)) * 16;
        fa_off[s] = (wm + l16) * TKB + chunk;
        fb_off[s] = ABYTES + (wn + l16) * TKB + chunk;
    }
    int4_t acc[MI][4];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = int4_t{0, 0, 0, 0};
    uint4_t fa[MI], fb[2][4];
    auto read_a = [&](int stage_off, int s, int i) { fa[i] = *reinterpret_cast<const uint4_t *>(tile_lds + stage_off + fa_off[s] + 16 * i * TKB); };
    auto read_b = [&](int slot, int stage_off, int s, int j) { fb[slot][j] = *reinterpret_cast<const uint4_t *>(tile_lds + stage_off + fb_off[s] + 16 * j * TKB); };
    auto mfma = [&](int slot, int i, int j) { acc[i][j] = q8_mfma(fb[slot][j], fa[i], acc[i][j]); };
#define AXHIP_FENCE() __builtin_amdgcn_sched_barrier(0)
    // s_waitcnt vmcnt(n) with the other counters left alone
#define AXHIP_VMCNT(n) __builtin_amdgcn_s_waitcnt(((n) & 0xF) | 0x0F70 | (((n) >> 4) << 14))
    static_assert(NL * (S - 1) < 64, "vmcnt is a 6-bit counter");
    if constexpr (DMA) {
#pragma unroll
        for (int st = 0; st < S; ++st)
#pragma unroll
            for (int n = 0; n < NL; ++n) dma_load(st, st * STAGEB, n);
        AXHIP_VMCNT(NL * (S - 1)); // tile 0 has landed
    } else {
        static_assert(DMA || (S == 2 && KS == 1 && R == 4), "through registers: two stages in LDS, four k-tiles in registers");
        // k-tile t travels in register set (t - 2) & 3; the first two go to LDS at once
#pragma unroll
        for (int t0 = 0; t0 < 4; ++t0)
            if (t0 < 2 || t0 < nk) {
#pragma unroll
                for (int n = 0; n < NL; ++n) reg_load((t0 + 2) & 3, t0, n);
            }
#pragma unroll
        for (int t0 = 0; t0 < 2; ++t0) {
#pragma unroll
            for (int n = 0; n < NL; ++n) reg_write(t0 + 2, t0, t0 * STAGEB, n);
            mend(t0, t0 * STAGEB);
            if (t0 + 4 < nk) {
#pragma unroll
                for (int n = 0; n < NL; ++n) reg_load(t0 + 2, t0 + 4, n);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i) read_a(0, 0, i);
#pragma unroll
    for (int j = 0; j < 4; ++j) read_b(0, 0, 0, j);

    int cur = 0; // offset of k-tile kt's stage
    auto tile = [&](auto phase_tag, auto last_tag, int kt) { // phase: kt modulo the unrolling; last (through registers): nothing left to load
        constexpr bool LAST = decltype(last_tag)::value;
        constexpr int P = decltype(phase_tag)::value & 1, SET = DMA ? 0 : decltype(phase_tag)::value % R; // set SET holds k-tile kt + 2
        const int next = cur + STAGEB == S * STAGEB ? 0 : cur + STAGEB;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            constexpr int SLOTS = (MI - 1) * 4; // MFMAs behind the barrier of the last k-step
            const int slot = (P + s) & 1;
            const bool last = s == KS - 1;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                if (last && i == 1) {
                    if constexpr (DMA) AXHIP_VMCNT(NL * (S - 2)); // this wavefront's share of tile kt + 1 has landed
                    __syncthreads();                              // ... everyone's has, and tile kt is no longer read
                    AXHIP_FENCE();
                    read_a(next, 0, 0);
                    AXHIP_FENCE();
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mfma(slot, i, j);
                    AXHIP_FENCE();
                    if (!last) {
                        if (j == 2 && i < 4) {
                            read_b(slot ^ 1, cur, s + 1, i);
                            AXHIP_FENCE();
                        }
                        if (j == 3) {
                            read_a(cur, s + 1, i);
                            AXHIP_FENCE();
                        }
                    } else if (i >= 1) {
                        const int q = (i - 1) * 4 + j;
                        constexpr int PERIOD = SLOTS / NL > 0 ? SLOTS / NL : 1;
                        if (q % 2 == 0 && q <= 6) {
                            read_b(slot ^ 1, next, 0, q / 2);
                            AXHIP_FENCE();
                        }
                        if (DMA && q % PERIOD == PERIOD - 1 && q / PERIOD < NL) {
                            dma_load(kt + S, cur, q / PERIOD);
                            AXHIP_FENCE();
                        }
                        if (!DMA && q % PERIOD == PERIOD - 1 && q / PERIOD < NL) {
                            reg_write(SET, kt + 2, cur, q / PERIOD);
                            AXHIP_FENCE();
                        }
                        if (j == 3) {
                            read_a(next, 0, i);
                            AXHIP_FENCE();
                        }
                    }
                }
            }
        }
        if constexpr (!DMA) {
            mend(kt + 2, cur);
            if constexpr (!LAST) {
#pragma unroll
                for (int n = 0; n < NL; ++n) reg_load(SET, kt + 2 + R, n);
            }
            AXHIP_FENCE();
        }
        cur = next;
    };
    if constexpr (!DMA) {
        // (no branch inside: the compiler would wait for every load in flight where the paths meet)
        auto four = [&](auto last_tag, int kt) {
            tile(std::integral_constant<int, 0>{}, last_tag, kt);
            tile(std::integral_constant<int, 1>{}, last_tag, kt + 1);
            tile(std::integral_constant<int, 2>{}, last_tag, kt + 2);
            tile(std::integral_constant<int, 3>{}, last_tag, kt + 3);
        };
        int kt = 0;
        for (; kt + 2 + R < nk; kt += 4) four(std::false_type{}, kt);
        for (; kt < nk; kt += 4) four(std::true_type{}, kt);
    } else if constexpr (KS % 2 == 0) {
        for (int kt = 0; kt < nk; ++kt) tile(std::integral_constant<int, 0>{}, std::false_type{}, kt);
    } else {
        for (int kt = 0; kt < nk; kt += 2) {
            tile(std::integral_constant<int, 0>{}, std::false_type{}, kt);
            if (kt + 1 < nk) tile(std::integral_constant<int, 1>{}, std::false_type{}, kt + 1);
        }
    }
#undef AXHIP_FENCE

    // ---- the WK groups' sums meet in LDS: group w finishes row blocks [w MB, (w + 1) MB) of its wavefront tile
    Q8Residual<DT, MP> res;
    res.load(g, m0 + wm + wk * MB * 16, n0 + wn, lane);
    AXHIP_VMCNT(0); // no load of this wavefront is still on its way into the ring
#undef AXHIP_VMCNT
    __syncthreads();
    int4_t own[MB][4];
    auto part = [&](int owner, int source, int i) -> unsigned char * { // 4 KiB: block i of `owner`, from `source` (!= owner)
        const int src = source - (source > owner ? 1 : 0);
        return tile_lds + ((((wt * WK + owner) * (WK - 1) + src) * MB + i) * 4096);
    };
    if constexpr (WK > 1) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int owner = i / MB;
            if (owner != wk) {
                unsigned char *p = part(owner, wk, i % MB);
#pragma unroll
                for (int j = 0; j < 4; ++j) *reinterpret_cast<int4_t *>(p + j * 1024 + lane * 16) = acc[i][j];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int w = 0; w < WK; ++w)
        if (wk == w) {
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) own[i][j] = acc[w * MB + i][j];
        }
    if constexpr (WK > 1) {
#pragma unroll
        for (int src = 0; src < WK - 1; ++src)
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                const unsigned char *p = tile_lds + ((((wt * WK + wk) * (WK - 1) + src) * MB + i) * 4096);
#pragma unroll
                for (int j = 0; j < 4; ++j) own[i][j] += *reinterpret_cast<const int4_t *>(p + j * 1024 + lane * 16);
            }
    }
    // (the blocks that a wavefront has just read are its staging area)
    unsigned char *stage = tile_lds + (WK > 1 ? (wt * WK + wk) * (WK - 1) * MB * 4096 : wave * MP * 4096);
    q8_store_pieces<DT, MB, MP>(g, own, scales, res, m0 + wm + wk * MB * 16, n0 + wn, lane, stage);
}

// bytes of LDS: the ring, or what the groups exchange at the end where that is more
template <int MI, int WM, int WN, int WK, int TKB, int S> constexpr size_t q8_tile_lds_bytes() {
    const size_t ring = size_t(S) * (16 * MI * WM + 64 * WN) * TKB;
    const size_t parts = WK > 1 ? size_t(WM * WN) * WK * (WK - 1) * (MI / WK) * 4096 : size_t(WM * WN) * (MI > 4 ? 4 : MI) * 4096;
    return ring > parts ? ring : parts;
}

template <int DT, bool DMA, int MI, int WM, int WN, int WK, int TKB, int S>
int launch_q8_tile_kernel(const Q8Args &g, hipStream_t s) {
    constexpr size_t lds = q8_tile_lds_bytes<MI, WM, WN, WK, TKB, S>();
    static_assert(lds <= 160 * 1024, "LDS of a CU");
    const auto kernel = gemm_q8_tile_kernel<DT, DMA, MI, WM, WN, WK, TKB, S>;
    static const hipError_t configured = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(lds));
    AXHIP_CHECK_HIP(configured);
    constexpr int TM = 16 * MI * WM, TN = 64 * WN;
    const int64_t tiles = static_cast<int64_t>((g.M + TM - 1) / TM) * ((g.N + TN - 1) / TN);
    AXHIP_REQUIRE(launch_fits(tiles + 7, 64 * WM * WN * WK), AXHIP_ERR_UNSUPPORTED, "axhip_gemm_q8: too many tiles");
    hipLaunchKernelGGL(kernel, dim3(tile_grid(tiles, 1)), dim3(64 * WM * WN * WK), lds, s, g);
    return AXHIP_OK;
}
template <int DT> int launch_q8_tile_as(const Q8Args &g, int tile, bool aligned, hipStream_t s) {
    if (!aligned) return launch_q8_tile_kernel<DT, false, 4, 2, 2, 2, 128, 2>(g, s);
    switch (tile) {
    case Q8_256x256: return launch_q8_tile_kernel<DT, true, 8, 2, 4, 1, 128, 2>(g, s);
    case Q8_256x128: return launch_q8_tile_kernel<DT, true, 8, 2, 2, 2, 128, 3>(g, s);
    case Q8_192x128: return launch_q8_tile_kernel<DT, true, 6, 2, 2, 2, 128, 3>(g, s);
    case Q8_128x128: return launch_q8_tile_kernel<DT, true, 4, 2, 2, 2, 128, 4>(g, s);
    case Q8_128x128_PAIR: return launch_q8_tile_kernel<DT, true, 4, 2, 2, 1, 128, 2>(g, s);
    default: return launch_q8_tile_kernel<DT, true, 4, 1, 2, 4, 256, 3>(g, s);
    }
}

} // namespace
} // namespace axhip
