// Device code shared by the kernels of int8 products.
#pragma once
#include "gemm_q8.hpp"
#include "gemm_skinny.hpp"
#include "gemm_tile_device.hpp"

namespace axhip {
namespace {

// int8 of any alignment
struct __attribute__((packed, aligned(1))) q8_chunk_t { uint4_t v; };
__device__ __forceinline__ uint4_t q8_load_chunk(const int8_t *p) { return reinterpret_cast<const q8_chunk_t *>(p)->v; }

// v: the 16 bytes of a row of n >= 16 bytes at byte min(at, n - 16).  What is left of [at, at + 16), in place, zeros behind it.
__device__ __forceinline__ uint4_t q8_chunk_in_place(uint4_t v, int at, int n) {
    const int drop = at - min(at, n - 16); // bytes in front of the chunk
    if (drop == 0) return v;
    if (drop >= 16) return uint4_t{0, 0, 0, 0};
    return __builtin_bit_cast(uint4_t, __builtin_bit_cast(unsigned __int128, v) >> (8 * drop));
}

// (B fragment) x (A fragment)^T on v_mfma_i32_16x16x64_i8: a lane's 16 bytes are 16 k of row lane % 16, from 16 (lane / 16) on -- the bytes that
// the 16-bit form of this instruction takes --, and it holds four consecutive columns of one row of C.
__device__ __forceinline__ int4_t q8_mfma(const uint4_t &fb, const uint4_t &fa, const int4_t &acc) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4_t, fb), __builtin_bit_cast(int4_t, fa), acc, 0, 0, 0);
}

// N sums of row `row` from column `col` on, of which columns [first, last) exist, to C: scales (scale_b's in sb, bias in b), residual, activation.
// Sums of up to 2^31 round to fp32 here, once; DT's rounding is the last.
template <int DT, int N>
__device__ __forceinline__ void q8_finish(const Q8Args &g, const int (&sum)[N], float sa, const float (&sb)[N], const float (&b)[N], int64_t at, int first, int last) {
    const bool whole = first == 0 && last == N;
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = __builtin_fmaf(static_cast<float>(sum[e]), sa * sb[e], b[e]);
    if (g.residual) {
        if (whole) {
            float r[N];
            load_vec<N, true>(g.residual, DT, at, r);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] += r[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e >= first && e < last) x[e] += Elem<DT>::load(g.residual, at + e);
        }
    }
    gemm_epilogue_all_as<DT != AXHIP_DTYPE_F32>(g.epilogue, x);
    if (whole) {
        store_vec<N, true>(g.c, DT, at, x);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e >= first && e < last) Elem<DT>::store(g.c, at + e, x[e]);
    }
}

// The wavefront's MB blocks of 16 x 64 sums -> C, through its own LDS (`stage`, 4 KiB per block), so that a lane holds eight consecutive columns of a
// row: whole 128-byte lines per store, and one short loop of code.
template <int DT, int MB>
__device__ __forceinline__ void q8_store_blocks(const Q8Args &g, const int4_t (&own)[MB][4], int m_base, int n_base, int lane, unsigned char *stage) {
    const int l16 = lane % 16, g4 = lane / 16;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<int4_t *>(stage + (16 * i + l16) * 256 + (((4 * j + g4) ^ l16) * 16)) = own[i][j];
    wave_lds_fence();
    const int q = lane & 7, col = n_base + 8 * q, last = min(8, g.N - col);
    if (last <= 0) return;
    float b[8], sb[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        sb[e] = e < last ? g.scale_b[col + e] : 0.0f;
        b[e] = g.bias && e < last ? Elem<DT>::load(g.bias, col + e) : 0.0f;
    }
#pragma unroll 1
    for (int r = lane >> 3; r < 16 * MB; r += 8) {
        const int row = m_base + r;
        if (row >= g.M) break;
        int sum[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int4_t v = *reinterpret_cast<const int4_t *>(stage + r * 256 + (((2 * q + h) ^ (r & 15)) * 16));
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[4 * h + e] = v[e];
        }
        q8_finish<DT, 8>(g, sum, g.scale_a[row], sb, b, static_cast<int64_t>(row) * g.ldc + col, 0, last);
    }
}

} // namespace
} // namespace axhip
