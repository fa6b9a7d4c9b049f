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

// A sum with its scales and bias.  Every kernel rounds here, in this order (the sum to fp32, the scales' product, the whole once), then adds the residual, so that a row's results
// have the same bits whichever kernel the other rows lead to.
__device__ __forceinline__ float q8_scaled(int sum, float sa, float sb, float bias) { return __builtin_fmaf(static_cast<float>(sum), sa * sb, bias); }

// x Phi(x) = max(x, 0) - z Phi(-z), z = |x|, for results of 16 bits, with Phi(-z) = 2^P(z): P is fitted to log2 Phi(-z) with all errors of one size, so that the left tail keeps its
// digits: within 2^-17.5 of itself for f16 (degree 7 up to 5.75, behind which no f16 is left but zero), 2^-12.8 for bf16 (degree 8 up to 13.1, where 2^P is below fp32's normal
// numbers and zero).  0 at -infinity.
template <int DT> __device__ __forceinline__ float q8_gelu16(float x) {
    constexpr float F16[] = {-1.82547734e-06f, 6.14397908e-05f, -0.000929487263f, 0.00850459774f, -0.0539548469f, -0.458468208f, -1.15125004f, -0.999995335f};
    constexpr float BF16[] = {2.78745644e-08f, -1.76587942e-06f, 4.82301422e-05f, -0.000750397564f, 0.00745485316f, -0.050910629f, -0.462621502f, -1.14912834f, -1.00017551f};
    const float z = fminf(fabsf(x), DT == AXHIP_DTYPE_F16 ? 5.75f : 13.1f);
    float p = DT == AXHIP_DTYPE_F16 ? F16[0] : BF16[0];
#pragma unroll
    for (int i = 1; i < (DT == AXHIP_DTYPE_F16 ? 8 : 9); ++i) p = __builtin_fmaf(p, z, DT == AXHIP_DTYPE_F16 ? F16[i < 8 ? i : 0] : BF16[i]);
    return __builtin_fmaf(-z, __builtin_amdgcn_exp2f(p), __builtin_elementwise_maximum(x, 0.0f));
}
// ... tanh within 2^-20 of itself: its series up to 1/4 (the next term is 3e-7 of the first), from there on by one exponential
__device__ __forceinline__ float q8_tanh16(float x) {
    const float s = x * x, far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + __expf(2.0f * x));
    const float near = x * __builtin_fmaf(s, __builtin_fmaf(s, __builtin_fmaf(s, -0.053968254f, 0.13333333f), -0.33333333f), 1.0f);
    return s < 0.0625f ? near : far;
}
// The activation of N values.  What is not a number stays so (v_maximum3_f32, where x > 0 ? x : 0 makes it a zero): a row with an infinity has scale NaN, and is not to
// leave a layer as zeros.
template <int DT, int N> __device__ __forceinline__ void q8_activation(int op, float (&x)[N]) {
    constexpr bool HALF = DT != AXHIP_DTYPE_F32;
    if (op == AXHIP_OP_RELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = __builtin_elementwise_maximum(x[e], 0.0f);
    } else if (HALF && op == AXHIP_OP_GELU) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = q8_gelu16<DT>(x[e]);
    } else if (HALF && op == AXHIP_OP_TANH) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = q8_tanh16(x[e]);
    } else {
        gemm_epilogue_all_as<HALF>(op, x);
    }
}

// N sums of a row, to C from `at` on, of which the first `last` exist: scales (scale_b's in sb, bias in b), residual, activation.
template <int DT, int N>
__device__ __forceinline__ void q8_finish(const Q8Args &g, const int (&sum)[N], float sa, const float (&sb)[N], const float (&b)[N], int64_t at, int last) {
    const bool whole = last == N;
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = q8_scaled(sum[e], sa, sb[e], b[e]);
    if (g.residual) {
        if (whole) {
            float r[N];
            load_vec<N, true>(g.residual, DT, at, r);
#pragma unroll
            for (int e = 0; e < N; ++e) x[e] += r[e];
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (e < last) x[e] += Elem<DT>::load(g.residual, at + e);
        }
    }
    q8_activation<DT>(g.epilogue, x);
    if (whole) {
        store_vec<N, true>(g.c, DT, at, x);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < last) Elem<DT>::store(g.c, at + e, x[e]);
    }
}

// What the epilogue of a wavefront's MB blocks of 16 x 64 needs of A's and B's rows, requested while the last products are still under way.
template <int DT, int MB> struct Q8Scales {
    float sa[MB], sb[4][4], b[4][4]; // as the sums lie: of rows 16 i + lane % 16, of columns 16 j + 4 (lane / 16) + e
    __device__ __forceinline__ void load(const Q8Args &g, int m_base, int n_base, int lane) {
#pragma unroll
        for (int i = 0; i < MB; ++i) sa[i] = g.scale_a[min(m_base + 16 * i + lane % 16, g.M - 1)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = n_base + 16 * j + 4 * (lane / 16);
            if (col + 4 <= g.N) {
                load_vec<4, true>(g.scale_b, AXHIP_DTYPE_F32, col, sb[j]);
                if (g.bias) load_vec<4, true>(g.bias, DT, col, b[j]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sb[j][e] = col + e < g.N ? g.scale_b[col + e] : 0.0f;
                    if (g.bias) b[j][e] = col + e < g.N ? Elem<DT>::load(g.bias, col + e) : 0.0f;
                }
            }
            if (!g.bias) {
#pragma unroll
                for (int e = 0; e < 4; ++e) b[j][e] = 0.0f;
            }
        }
    }
};

// The residual of a wavefront's MB blocks, as the lane that finishes it takes it: eight columns of rows lane / 8 + 8 n.
template <int DT, int MB> struct Q8Residual {
    static constexpr int V = DT == AXHIP_DTYPE_F32 ? 2 : 1; // 16-byte vectors
    uint4_t raw[2 * MB][V];
    __device__ __forceinline__ void load(const Q8Args &g, int m_base, int n_base, int lane) {
        constexpr int ES = DT == AXHIP_DTYPE_F32 ? 4 : 2;
        const int col = n_base + 8 * (lane & 7), last = min(8, g.N - col);
        if (!g.residual || last <= 0) return;
#pragma unroll
        for (int n = 0; n < 2 * MB; ++n) {
            const int64_t from = static_cast<int64_t>(min(m_base + (lane >> 3) + 8 * n, g.M - 1)) * g.ldc + col;
            const char *p = static_cast<const char *>(g.residual) + from * ES;
            if (last == 8) {
#pragma unroll
                for (int v = 0; v < V; ++v) raw[n][v] = reinterpret_cast<const uint4_unaligned_t *>(p + 16 * v)->v;
            } else {
#pragma unroll
                for (int v = 0; v < V; ++v) raw[n][v] = uint4_t{0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < last) {
                        if constexpr (V == 2) raw[n][e / 4][e % 4] = reinterpret_cast<const uint32_t *>(p)[e];
                        else raw[n][0][e / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(p)[e]) << (16 * (e % 2));
                    }
            }
        }
    }
    __device__ __forceinline__ float at(int n, int e) const {
        if constexpr (V == 2) return __uint_as_float(raw[n][e / 4][e % 4]);
        else if constexpr (DT == AXHIP_DTYPE_BF16) return bf16_bits_to_f32((raw[n][0][e / 2] >> (16 * (e % 2))) & 0xFFFFu);
        else return f16_bits_to_f32((raw[n][0][e / 2] >> (16 * (e % 2))) & 0xFFFFu);
    }
};

// Blocks first .. first + MP - 1 of the wavefront's sums of 16 x 64 -> C, through its own LDS (`stage`, 4 KiB per block), so that a lane holds eight consecutive columns of a
// row: whole 128-byte lines per store, and one short loop of code.  In that loop nothing is loaded from memory: scales and bias are taken
// on the way to LDS, and the residual (`res`, requested before the last products are over) is added to what lies there; then `behind` requests the next blocks' residual, which
// arrives while these are written (row by row, each waited for the one before: 8192 x 4096 x 128 with a residual took 60 us, 26 without).
template <int DT, int MB, int MP, class F>
__device__ __forceinline__ void q8_store_blocks(const Q8Args &g, const int4_t (&own)[MB][4], int first, const Q8Scales<DT, MB> &s, const Q8Residual<DT, MP> &res, int m_base, int n_base, int lane, unsigned char *stage, F behind) {
    const int l16 = lane % 16, g4 = lane / 16;
#pragma unroll
    for (int i = 0; i < MP; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float4_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = q8_scaled(own[first + i][j][e], s.sa[first + i], s.sb[j][e], s.b[j][e]);
            *reinterpret_cast<float4_t *>(stage + (16 * i + l16) * 256 + (((4 * j + g4) ^ l16) * 16)) = v;
        }
    wave_lds_fence();
    const int q = lane & 7, col = n_base + 8 * q, last = min(8, g.N - col);
    auto at = [&](int r, int h) { return reinterpret_cast<float4_t *>(stage + r * 256 + (((2 * q + h) ^ (r & 15)) * 16)); };
    if (g.residual && last > 0) {
#pragma unroll
        for (int n = 0; n < 2 * MP; ++n) {
            const int r = (lane >> 3) + 8 * n;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4_t v = *at(r, h);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += res.at(n, 4 * h + e);
                *at(r, h) = v;
            }
        }
    }
    behind();
    if (last <= 0) return;
#pragma unroll 1
    for (int r = lane >> 3; r < 16 * MP; r += 8) {
        const int row = m_base + r;
        if (row >= g.M) break;
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float4_t v = *at(r, h);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * h + e] = v[e];
        }
        q8_activation<DT>(g.epilogue, x);
        const int64_t to = static_cast<int64_t>(row) * g.ldc + col;
        if (last == 8) {
            store_vec<8, true>(g.c, DT, to, x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < last) Elem<DT>::store(g.c, to + e, x[e]);
        }
    }
}

// ... all MB blocks, MP staged at a time; `res`: the first ones' residual.
template <int DT, int MB, int MP>
__device__ __forceinline__ void q8_store_pieces(const Q8Args &g, const int4_t (&own)[MB][4], const Q8Scales<DT, MB> &s, Q8Residual<DT, MP> &res, int m_base, int n_base, int lane, unsigned char *stage) {
#pragma unroll
    for (int h = 0; h < MB / MP; ++h) {
        q8_store_blocks<DT, MB, MP>(g, own, MP * h, s, res, m_base + 16 * MP * h, n_base, lane, stage, [&]() __attribute__((always_inline)) {
            if (h + 1 < MB / MP) res.load(g, m_base + 16 * MP * (h + 1), n_base, lane);
        });
        wave_lds_fence();
    }
}

} // namespace
} // namespace axhip
