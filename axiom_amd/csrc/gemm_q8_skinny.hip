// Products of one or two int8 rows of x with a weight matrix: one read of the weights.
#include "gemm_q8_device.hpp"

namespace axhip {
namespace {

// The sums of P values (a power of two) over the wavefront, value i in the lanes [64 / P i, 64 / P (i + 1)): at each step that still has several
// values a lane hands half of them over and adds up the other half.
template <int P> __device__ __forceinline__ int q8_lane_sums(int (&v)[P], int lane) {
    auto step = [&](int p, int d) __attribute__((always_inline)) {
        if (p <= 1) {
            v[0] += __shfl_xor(v[0], d, WAVE);
            return;
        }
#pragma unroll
        for (int i = 0; i < p / 2; ++i) {
            const int mine = lane & d ? v[i + p / 2] : v[i], other = lane & d ? v[i] : v[i + p / 2];
            v[i] = mine + __shfl_xor(other, d, WAVE);
        }
    };
    step(P, 32);
    step(P / 2, 16);
    step(P / 4, 8);
    step(1, 4);
    step(1, 2);
    step(1, 1);
    return v[0];
}

// A wavefront owns R rows of W and walks k with its 64 lanes side by side, 1 KiB of a row per load; four products and their addition per instruction
// (v_dot4_i32_i8).  Rows may start anywhere; the chunk that K ends in is fetched as the 16 bytes that end with the row, with those in front of it
// cleared in x.  1 x 4096 x 4096 3.4 us back to back (16.8 MB from the caches), 4.7 with other weights in between.
template <int DT, int M, int R>
__global__ __launch_bounds__(256) void gemm_q8_skinny_kernel(const Q8Args a) {
    const int lane = threadIdx.x % 64;
    const int n0 = (static_cast<int>(blockIdx.x) * 4 + threadIdx.x / 64) * R;
    if (n0 >= a.N) return; // (whole wavefronts)
    constexpr int P = M * R; // sums of a wavefront: 1, 2 or 4
    // after the sums, lane 64 / P i finishes value i = m R + r; what it needs is requested before W is
    const int value = lane / (64 / P), n = n0 + value % R;
    const bool writes = lane % (64 / P) == 0 && n < a.N;
    const int64_t at = static_cast<int64_t>(value / R) * a.ldc + n;
    const float bias = writes && a.bias ? Elem<DT>::load(a.bias, n) : 0.0f, residual = writes && a.residual ? Elem<DT>::load(a.residual, at) : 0.0f;
    const float sa = writes ? a.scale_a[value / R] : 0.0f, sb = writes ? a.scale_b[n] : 0.0f;
    int acc[M][R] = {};
    const int8_t *wrow[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wrow[r] = a.b + static_cast<int64_t>(min(n0 + r, a.N - 1)) * a.ldb; // (rows past N: the last row again, not stored)
    constexpr int U = R == 1 ? 4 : 2; // k steps requested together
    for (int k0 = lane * 16; k0 < a.K; k0 += 1024 * U) {
        uint4_t wf[U][R], xf[U][M];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + 1024 * u, from = min(k, a.K - 16);
            const bool inside = k < a.K;
#pragma unroll
            for (int r = 0; r < R; ++r) wf[u][r] = inside ? q8_load_chunk(wrow[r] + from) : uint4_t{0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < M; ++m) xf[u][m] = inside ? q8_load_chunk(a.a + static_cast<int64_t>(m) * a.lda + from) : uint4_t{0, 0, 0, 0};
            if (inside && from != k) {
                const int drop = 8 * (k - from); // bits
#pragma unroll
                for (int m = 0; m < M; ++m) xf[u][m] = __builtin_bit_cast(uint4_t, __builtin_bit_cast(unsigned __int128, xf[u][m]) >> drop << drop);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][r] = __builtin_amdgcn_sdot4(static_cast<int>(wf[u][r][i]), static_cast<int>(xf[u][m][i]), acc[m][r], false);
    }
    int v[P];
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = acc[i / R][i % R];
    const int sum = q8_lane_sums<P>(v, lane);
    float x[1] = {q8_scaled(sum, sa, sb, bias) + residual};
    q8_activation<DT>(a.epilogue, x);
    if (writes) Elem<DT>::store(a.c, at, x[0]);
}

template <int DT, int M> void launch_rows(const Q8Args &g, int rows_per_wave, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>((g.N + 4 * rows_per_wave - 1) / (4 * rows_per_wave)));
    if (rows_per_wave == 2) hipLaunchKernelGGL((gemm_q8_skinny_kernel<DT, M, 2>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((gemm_q8_skinny_kernel<DT, M, 1>), grid, dim3(256), 0, s, g);
}
template <int DT> void launch_dtype(const Q8Args &g, int rows_per_wave, hipStream_t s) {
    if (g.M == 1) launch_rows<DT, 1>(g, rows_per_wave, s);
    else launch_rows<DT, 2>(g, rows_per_wave, s);
}
} // namespace

int launch_q8_skinny(const Q8Args &g, int dtype, int rows_per_wave, hipStream_t s) {
    if (dtype == AXHIP_DTYPE_F32) launch_dtype<AXHIP_DTYPE_F32>(g, rows_per_wave, s);
    else if (dtype == AXHIP_DTYPE_F16) launch_dtype<AXHIP_DTYPE_F16>(g, rows_per_wave, s);
    else launch_dtype<AXHIP_DTYPE_BF16>(g, rows_per_wave, s);
    return AXHIP_OK;
}
} // namespace axhip
