// Rows in 8 bits with a scale each: axhip_quantize_q8, and axhip_rms_norm_q8 with the residual's addition and the norm in the same pass.
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace axhip {
namespace {

struct RowsQ8Args {
    const void *x, *residual, *weight;
    void *sum;
    int8_t *q;
    float *scales;
    int64_t rows, ld_x, ld_residual, ld_sum, ld_q;
    int64_t cols;
    double inverse_cols;
    float eps;
    int blocks;
};

enum { QUANTIZE, NORM, NORM_RESIDUAL };

struct __attribute__((packed, aligned(1))) q8x8_unaligned_t { uint2_t v; };
struct __attribute__((packed, aligned(1))) q8x4_unaligned_t { uint32_t v; };

// What the rows' largest magnitude is kept in: products of two 16-bit floats are exact in fp32, those of two fp32 in fp64.
template <int DT, int MODE> using Product = std::conditional_t<DT == AXHIP_DTYPE_F32 && MODE != QUANTIZE, double, float>;

// Magnitudes compare as their bits do, and a NaN's are above an infinity's, which are above all others'.
__device__ __forceinline__ float larger(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }
__device__ __forceinline__ double larger(double a, double b) { return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b))); }
__device__ __forceinline__ float magnitude(float v) { return fabsf(v); }
__device__ __forceinline__ double magnitude(double v) { return fabs(v); }
__device__ __forceinline__ float wave_largest(float v) { return wave_all(v, [](float a, float b) { return larger(a, b); }); }
// wave_all of common.hpp in 64 bits
template <class F> __device__ __forceinline__ double wave_all64(double v, F combine) {
    auto low = [](double x) { return static_cast<uint32_t>(__double_as_longlong(x)); };
    auto high = [](double x) { return static_cast<uint32_t>(static_cast<uint64_t>(__double_as_longlong(x)) >> 32); };
    auto whole = [](uint32_t lo, uint32_t hi) { return __longlong_as_double(static_cast<long long>(static_cast<uint64_t>(hi) << 32 | lo)); };
    const auto lo32 = __builtin_amdgcn_permlane32_swap(low(v), low(v), false, false), hi32 = __builtin_amdgcn_permlane32_swap(high(v), high(v), false, false);
    v = combine(whole(lo32[0], hi32[0]), whole(lo32[1], hi32[1]));
    const auto lo16 = __builtin_amdgcn_permlane16_swap(low(v), low(v), false, false), hi16 = __builtin_amdgcn_permlane16_swap(high(v), high(v), false, false);
    v = combine(whole(lo16[0], hi16[0]), whole(lo16[1], hi16[1]));
    auto across = [&](auto control) __attribute__((always_inline)) { // (row_ror)
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(low(v)), decltype(control)::value, 0xF, 0xF, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(high(v)), decltype(control)::value, 0xF, 0xF, false);
        v = combine(v, whole(lo, hi));
    };
    across(std::integral_constant<int, 0x128>{});
    across(std::integral_constant<int, 0x124>{});
    across(std::integral_constant<int, 0x122>{});
    across(std::integral_constant<int, 0x121>{});
    return v;
}
__device__ __forceinline__ double wave_largest(double v) { return wave_all64(v, [](double a, double b) { return larger(a, b); }); }
__device__ __forceinline__ float sum_of_wave(float v) { return wave_sum(v); }
__device__ __forceinline__ double sum_of_wave(double v) { return wave_all64(v, [](double a, double b) { return a + b; }); }

// The sum of squares: those of f16 numbers lie within fp32's range, those of bf16 and fp32 ones from 2^-298 to 2^256.
__device__ __forceinline__ float add_square(float h, float sum) { return __builtin_fmaf(h, h, sum); }
__device__ __forceinline__ double add_square(float h, double sum) { return __builtin_fma(static_cast<double>(h), static_cast<double>(h), sum); }
template <int DT> using Squares = std::conditional_t<DT == AXHIP_DTYPE_F16, float, double>;

__device__ __forceinline__ float mantissa(float v, int &exponent) {
    exponent = __builtin_amdgcn_frexp_expf(v);
    return __builtin_amdgcn_frexp_mantf(v);
}
__device__ __forceinline__ float mantissa(double v, int &exponent) {
    exponent = __builtin_amdgcn_frexp_exp(v);
    return static_cast<float>(__builtin_amdgcn_frexp_mant(v));
}
// The row's scale: largest / 127, over the root of mean(h^2) + eps for a norm.  Mantissas in fp32, with their powers of two by themselves: neither the mean nor the largest need be an fp32 number,
// the scale alone.
template <int MODE, class Y, class S> __device__ __forceinline__ float scale_of(const RowsQ8Args &a, Y largest, S squares) {
    const float top = static_cast<float>(largest);
    if (!(__float_as_uint(top) < 0x7F800000u)) return __uint_as_float(0x7FC00000u);
    if (!(largest > 0)) return 0.0f;
    if constexpr (MODE == QUANTIZE) return top / 127.0f;
    const double mean = static_cast<double>(squares) * a.inverse_cols + static_cast<double>(a.eps);
    const int even = (__builtin_amdgcn_frexp_exp(mean) - 1) & ~1;
    int exponent;
    const float m = mantissa(largest, exponent);
    return __builtin_amdgcn_ldexpf(m * (1.0f / sqrtf(static_cast<float>(__builtin_amdgcn_ldexp(mean, -even)))) / 127.0f, exponent - even / 2);
}

// Products of two fp32 numbers may be as small as 2^-298: what a row of them is multiplied by (a power of two, exactly) so that 127 / a is an ordinary number.
__device__ __forceinline__ double bringing_up(double largest) { return largest > 0.0 ? __builtin_amdgcn_ldexp(1.0, -__builtin_amdgcn_frexp_exp(largest)) : 1.0; }

// E values -> E bytes.  127 y / a rounds to the nearest integer through the sum with 1.5 * 2^23, whose last bit is a one: the low byte of
// the sum is the integer.  The product with 127 / a is off by less than 3 * 2^-24 * 127 < 4e-5; where it lies that close to a half h (4 % of
// the wavefront's vectors), and where 127 / a would overflow (`tiny`), it is decided exactly.  Of y and a of 24 bits the quotient in 64 bits tells: it is the half itself or
// 2^-34 from it at least.  Products of two fp32 numbers have 48 bits and quotients as near as 2^-49, where steps are 2^-46: of them the sign of 127 y - h a decides, and where that is
// nothing the even integer is taken.  With s = h a to 53 bits, 127 y - s and h a - s are multiples of 2^-56 a and below 2^-14 a, so that two fused operations round neither.
template <int E, class Y> __device__ __forceinline__ void quantize(const Y (&y)[E], float inverse, Y largest, bool tiny, uint32_t (&w)[E / 4]) {
    constexpr float TO_INTEGER = 12582912.0f, NEAR_HALF = 0.49996f;
    uint32_t r[E];
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float v = static_cast<float>(y[e]), s = __builtin_fmaf(v, inverse, TO_INTEGER);
        off = fmaxf(off, fabsf(__builtin_fmaf(v, inverse, TO_INTEGER - s)));
        r[e] = __float_as_uint(s);
    }
    if (off > NEAR_HALF || (tiny && !std::is_same_v<Y, double>)) { // (products of fp32 numbers have been brought up)
        if constexpr (std::is_same_v<Y, double>) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float n = __uint_as_float(r[e]) - TO_INTEGER, from = __builtin_fmaf(static_cast<float>(y[e]), inverse, -n);
                const double half = n + __builtin_copysignf(0.5f, from), s = half * largest;
                const double left = __builtin_fma(127.0, y[e], -s) - __builtin_fma(half, largest, -s);
                const bool behind = (from > 0.0f) == (left > 0.0); // the half, as seen from n
                const bool moves = (fabsf(from) > NEAR_HALF) & (((left != 0.0) & behind) | ((left == 0.0) & static_cast<bool>(r[e] & 1u)));
                r[e] += moves ? (from > 0.0f ? 1u : ~0u) : 0u;
            }
        } else {
            for (int e = 0; e < E; ++e) {
                const int q = static_cast<int>(__builtin_rint(127.0 * static_cast<double>(y[e]) / static_cast<double>(largest)));
                r[e] = static_cast<uint32_t>(q);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(r[4 * i + 1], r[4 * i], 0x0C0C0400u), hi = __builtin_amdgcn_perm(r[4 * i + 3], r[4 * i + 2], 0x04000C0Cu);
        w[i] = lo | hi;
    }
}

// A chunk of E elements at `at`, of which `valid` are in the row (the others are zeros).
template <int DT, int E, bool UNALIGNED> __device__ __forceinline__ void load_chunk(const void *row, int64_t at, int64_t valid, float (&v)[E]) {
    if (valid >= E) {
        load_vec<E, UNALIGNED>(row, DT, at, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e < valid ? Elem<DT>::load(row, at + e) : 0.0f;
    }
}
template <int DT, int E, bool UNALIGNED> __device__ __forceinline__ void store_chunk(void *row, int64_t at, int64_t valid, const float (&v)[E]) {
    if (valid >= E) {
        store_vec<E, UNALIGNED>(row, DT, at, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < valid) Elem<DT>::store(row, at + e, v[e]);
    }
}
template <int E, bool UNALIGNED> __device__ __forceinline__ void store_bytes(int8_t *row, int64_t at, int64_t valid, const uint32_t (&w)[E / 4]) {
    if (valid >= E) {
        if constexpr (E == 8) {
            if constexpr (UNALIGNED) reinterpret_cast<q8x8_unaligned_t *>(row + at)->v = uint2_t{w[0], w[1]};
            else *reinterpret_cast<uint2_t *>(row + at) = uint2_t{w[0], w[1]};
        } else {
            if constexpr (UNALIGNED) reinterpret_cast<q8x4_unaligned_t *>(row + at)->v = w[0];
            else *reinterpret_cast<uint32_t *>(row + at) = w[0];
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < valid) row[at + e] = static_cast<int8_t>(w[e / 4] >> (8 * (e % 4)));
    }
}

// One chunk: h (after the residual's addition, rounded to DT), and y = h * weight.
template <int DT, int MODE, int E, bool UNALIGNED, class Y>
__device__ __forceinline__ void make_products(const RowsQ8Args &a, int64_t row, int64_t at, int64_t valid, float (&h)[E], Y (&y)[E]) {
    constexpr int64_t ES = DT == AXHIP_DTYPE_F32 ? 4 : 2;
    load_chunk<DT, E, UNALIGNED>(static_cast<const char *>(a.x) + row * a.ld_x * ES, at, valid, h);
    if constexpr (MODE == NORM_RESIDUAL) {
        float r[E];
        load_chunk<DT, E, UNALIGNED>(static_cast<const char *>(a.residual) + row * a.ld_residual * ES, at, valid, r);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float s = h[e] + r[e];
            if constexpr (DT == AXHIP_DTYPE_BF16) h[e] = bf16_bits_to_f32(f32_to_bf16_bits(s));
            else if constexpr (DT == AXHIP_DTYPE_F16) h[e] = f16_bits_to_f32(f32_to_f16_bits(s));
            else h[e] = s;
        }
        if (a.sum) store_chunk<DT, E, UNALIGNED>(static_cast<char *>(a.sum) + row * a.ld_sum * ES, at, valid, h);
    }
    if constexpr (MODE == QUANTIZE) {
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = h[e];
    } else {
        float w[E];
        if (a.weight) {
            load_chunk<DT, E, UNALIGNED>(a.weight, at, valid, w);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = 1.0f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = static_cast<Y>(h[e]) * static_cast<Y>(w[e]);
    }
}

// Bound by memory: one read of x (and the residual), one write of the integers (and the sum).  bf16 8192 x 4096 with a residual and the sum 47.8 us (235 MB, 4.9 TB/s, 96 % of what a
// copy reaches; squares in 64 bits take 0.6 of them), fp32 4096 x 4096 14.6 (84 MB, partly from the caches); one row of 1280 takes 3.1 - 3.6 us, a launch.
// A row to G threads, in their registers (IT chunks of 16 bytes each), so that x is read once.  1 / sqrt(mean(h^2) + eps) is the same factor in y
// and in max |y|: it cancels in the integers and shows in the scale alone, so the integers wait for one maximum, not for a norm and then
// a maximum.
template <int DT, int MODE, int G, int IT, bool UNALIGNED>
__global__ __launch_bounds__(G < 256 ? 256 : G) void rows_q8_kernel(const RowsQ8Args a) {
    using Y = Product<DT, MODE>;
    using S = Squares<DT>;
    constexpr int E = DT == AXHIP_DTYPE_F32 ? 4 : 8, ROWS = G < 256 ? 256 / G : 1, WAVES = G / WAVE;
    __shared__ Y s_largest[2][WAVES > 1 ? WAVES : 1];
    __shared__ S s_squares[2][WAVES > 1 ? WAVES : 1];
    const int lane = threadIdx.x % G, wave = threadIdx.x / WAVE;
    int turn = 0;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / G; row < a.rows; row += static_cast<int64_t>(a.blocks) * ROWS, turn ^= 1) {
        Y y[IT][E], largest = 0;
        S squares = 0;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int64_t at = static_cast<int64_t>(i * G + lane) * E;
            if (at < a.cols) {
                float h[E];
                make_products<DT, MODE, E, UNALIGNED>(a, row, at, a.cols - at, h, y[i]);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    largest = larger(largest, magnitude(y[i][e]));
                    if constexpr (MODE != QUANTIZE) squares = add_square(h[e], squares);
                }
            }
        }
        largest = wave_largest(largest);
        if constexpr (MODE != QUANTIZE) squares = sum_of_wave(squares);
        if constexpr (WAVES > 1) {
            if (threadIdx.x % WAVE == 0) {
                s_largest[turn][wave] = largest;
                if constexpr (MODE != QUANTIZE) s_squares[turn][wave] = squares;
            }
            __syncthreads(); // (the next row uses the other set, and meets here before this one is written again)
            largest = s_largest[turn][0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) largest = larger(largest, s_largest[turn][w]);
        }
        const float top = static_cast<float>(largest);
        const bool finite = __float_as_uint(top) < 0x7F800000u, tiny = top < 1e-30f;
        if (lane == 0) { // (here, not behind the integers: nothing of it takes registers there)
            if constexpr (MODE != QUANTIZE && WAVES > 1)
                for (int w = 1; w < WAVES; ++w) squares += s_squares[turn][w]; // (lane 0 is of wavefront 0)
            a.scales[row] = scale_of<MODE>(a, largest, squares);
        }
        float inverse = tiny ? 0.0f : 127.0f / top;
        if constexpr (std::is_same_v<Y, double>) {
            if (tiny) {
                const double up = bringing_up(largest);
                largest *= up;
                inverse = 127.0f / static_cast<float>(largest);
#pragma unroll
                for (int i = 0; i < IT; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) y[i][e] *= up;
            }
        }
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int64_t at = static_cast<int64_t>(i * G + lane) * E;
            if (at < a.cols) {
                uint32_t w[E / 4] = {};
                if (finite && largest > 0) quantize<E, Y>(y[i], inverse, largest, tiny, w);
                store_bytes<E, UNALIGNED>(a.q + row * a.ld_q, at, a.cols - at, w);
            }
        }
    }
}

// Rows longer than the registers of 1024 threads: the same in two sweeps, the second of which forms the products again (from the sum where there is one: it may lie where x or the
// residual did).
template <int DT, int MODE>
__global__ __launch_bounds__(1024) void rows_q8_long_kernel(const RowsQ8Args a) {
    using Y = Product<DT, MODE>;
    using S = Squares<DT>;
    constexpr int E = DT == AXHIP_DTYPE_F32 ? 4 : 8;
    __shared__ Y s_largest[16];
    __shared__ S s_squares[16];
    for (int64_t row = blockIdx.x; row < a.rows; row += a.blocks) {
        Y largest = 0;
        S squares = 0;
        for (int64_t at = threadIdx.x * E; at < a.cols; at += 1024 * E) {
            float h[E];
            Y y[E];
            make_products<DT, MODE, E, true>(a, row, at, a.cols - at, h, y);
            S part = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                largest = larger(largest, magnitude(y[e]));
                if constexpr (MODE != QUANTIZE) part = add_square(h[e], part);
            }
            squares += part;
        }
        largest = wave_largest(largest);
        if constexpr (MODE != QUANTIZE) squares = sum_of_wave(squares);
        __syncthreads();
        if (threadIdx.x % WAVE == 0) {
            s_largest[threadIdx.x / WAVE] = largest;
            s_squares[threadIdx.x / WAVE] = squares;
        }
        __syncthreads();
        largest = s_largest[0];
        squares = s_squares[0];
        for (int w = 1; w < 16; ++w) {
            largest = larger(largest, s_largest[w]);
            squares += s_squares[w];
        }
        if (threadIdx.x == 0) a.scales[row] = scale_of<MODE>(a, largest, squares);
        const float top = static_cast<float>(largest);
        const bool finite = __float_as_uint(top) < 0x7F800000u, tiny = top < 1e-30f;
        float inverse = tiny ? 0.0f : 127.0f / top;
        Y up = 1;
        if constexpr (std::is_same_v<Y, double>) {
            if (tiny) {
                up = bringing_up(largest);
                largest *= up;
                inverse = 127.0f / static_cast<float>(largest);
            }
        }
        RowsQ8Args again = a;
        if (MODE == NORM_RESIDUAL && a.sum) {
            again.x = a.sum;
            again.ld_x = a.ld_sum;
        }
        again.sum = nullptr;
        for (int64_t at = threadIdx.x * E; at < a.cols; at += 1024 * E) {
            float h[E];
            Y y[E];
            if (MODE == NORM_RESIDUAL && a.sum) make_products<DT, MODE == QUANTIZE ? QUANTIZE : NORM, E, true>(again, row, at, a.cols - at, h, y);
            else make_products<DT, MODE, E, true>(again, row, at, a.cols - at, h, y);
            uint32_t w[E / 4] = {};
            if constexpr (std::is_same_v<Y, double>) {
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] *= up;
            }
            if (finite && largest > 0) quantize<E, Y>(y, inverse, largest, tiny, w);
            store_bytes<E, true>(a.q + row * a.ld_q, at, a.cols - at, w);
        }
    }
}

template <int DT, int MODE, int G, int IT> void launch_plan(RowsQ8Args a, bool aligned, hipStream_t s) {
    constexpr int ROWS = G < 256 ? 256 / G : 1, THREADS = G < 256 ? 256 : G;
    a.blocks = static_cast<int>(std::min<int64_t>((a.rows + ROWS - 1) / ROWS, 1 << 20));
    if (aligned) hipLaunchKernelGGL((rows_q8_kernel<DT, MODE, G, IT, false>), dim3(a.blocks), dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((rows_q8_kernel<DT, MODE, G, IT, true>), dim3(a.blocks), dim3(THREADS), 0, s, a);
}
template <int DT, int MODE> void launch_mode(RowsQ8Args a, bool aligned, hipStream_t s) {
    constexpr int E = DT == AXHIP_DTYPE_F32 ? 4 : 8;
    const int64_t chunks = (a.cols + E - 1) / E;
    if (chunks <= 64) return launch_plan<DT, MODE, 64, 1>(a, aligned, s);
    if (chunks <= 128) return launch_plan<DT, MODE, 64, 2>(a, aligned, s);
    if (chunks <= 256) return launch_plan<DT, MODE, 256, 1>(a, aligned, s);
    if (chunks <= 512) return launch_plan<DT, MODE, 256, 2>(a, aligned, s);
    if (chunks <= 1024) return launch_plan<DT, MODE, 256, 4>(a, aligned, s);
    if (chunks <= 2048) return launch_plan<DT, MODE, 256, 8>(a, aligned, s);
    if (chunks <= 8192) return launch_plan<DT, MODE, 1024, 8>(a, aligned, s);
    a.blocks = static_cast<int>(std::min<int64_t>(a.rows, 1 << 20));
    hipLaunchKernelGGL((rows_q8_long_kernel<DT, MODE>), dim3(a.blocks), dim3(1024), 0, s, a);
}
template <int MODE> void launch_dtype(const RowsQ8Args &a, int dtype, bool aligned, hipStream_t s) {
    if (dtype == AXHIP_DTYPE_F32) launch_mode<AXHIP_DTYPE_F32, MODE>(a, aligned, s);
    else if (dtype == AXHIP_DTYPE_F16) launch_mode<AXHIP_DTYPE_F16, MODE>(a, aligned, s);
    else launch_mode<AXHIP_DTYPE_BF16, MODE>(a, aligned, s);
}

int rows_q8(const char *who, int mode, const void *x, const void *residual, const void *weight, void *sum, int8_t *q, float *scales, const AxhipRowsQ8Params *params, void *stream) {
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "%s: params is NULL", who);
    const AxhipRowsQ8Params &p = *params;
    AXHIP_REQUIRE(valid_dtype(p.dtype), AXHIP_ERR_INVALID_ARG, "%s: bad dtype %d", who, p.dtype);
    constexpr int64_t SIDE = int64_t(1) << 40;
    AXHIP_REQUIRE(p.rows >= 0 && p.cols >= 0 && p.rows < SIDE && p.cols < SIDE, AXHIP_ERR_INVALID_ARG, "%s: bad extent", who);
    AXHIP_REQUIRE(p.ld_x >= p.cols && p.ld_q >= p.cols && (!residual || p.ld_residual >= p.cols) && (!sum || p.ld_sum >= p.cols), AXHIP_ERR_INVALID_ARG,
                  "%s: rows overlap (a leading dimension is below cols)", who);
    AXHIP_REQUIRE(!sum || residual, AXHIP_ERR_INVALID_ARG, "%s: a sum without a residual", who);
    AXHIP_REQUIRE(sum != x || !sum || p.ld_sum == p.ld_x, AXHIP_ERR_INVALID_ARG, "%s: a sum in x's place needs its leading dimension", who);
    AXHIP_REQUIRE(sum != residual || !sum || p.ld_sum == p.ld_residual, AXHIP_ERR_INVALID_ARG, "%s: a sum in the residual's place needs its leading dimension", who);
    AXHIP_REQUIRE(mode == QUANTIZE || (p.eps >= 0.0f && p.eps <= 3.4e38f), AXHIP_ERR_INVALID_ARG, "%s: bad eps", who);
    if (p.rows == 0) return AXHIP_OK;
    AXHIP_REQUIRE(scales && (p.cols == 0 || (x && q)), AXHIP_ERR_INVALID_ARG, "%s: NULL buffer", who);
    const uintptr_t unit = dtype_size(p.dtype) - 1;
    AXHIP_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(sum)) & unit) == 0 &&
                      (reinterpret_cast<uintptr_t>(scales) & 3u) == 0,
                  AXHIP_ERR_INVALID_ARG, "%s: a buffer is not aligned to its elements", who);
    int rc = ensure_init();
    if (rc) return rc;
    const int64_t e = p.dtype == AXHIP_DTYPE_F32 ? 4 : 8;
    const bool aligned = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(sum)) & 15u) == 0 &&
                         reinterpret_cast<uintptr_t>(q) % e == 0 && (p.ld_x | p.ld_q | (residual ? p.ld_residual : 0) | (sum ? p.ld_sum : 0)) % e == 0;
    const RowsQ8Args a{x, residual, weight, sum, q, scales, p.rows, p.ld_x, p.ld_residual, p.ld_sum, p.ld_q, p.cols, 1.0 / static_cast<double>(p.cols), p.eps, 0};
    hipStream_t s = resolve_stream(stream);
    if (mode == QUANTIZE) launch_dtype<QUANTIZE>(a, p.dtype, aligned, s);
    else if (!residual) launch_dtype<NORM>(a, p.dtype, aligned, s);
    else launch_dtype<NORM_RESIDUAL>(a, p.dtype, aligned, s);
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}
} // namespace
} // namespace axhip

extern "C" int axhip_quantize_q8(const void *x, int8_t *q, float *scales, const AxhipRowsQ8Params *params, void *stream) {
    return axhip::rows_q8("axhip_quantize_q8", axhip::QUANTIZE, x, nullptr, nullptr, nullptr, q, scales, params, stream);
}
extern "C" int axhip_rms_norm_q8(const void *x, const void *residual, const void *weight, void *sum, int8_t *q, float *scales, const AxhipRowsQ8Params *params, void *stream) {
    return axhip::rows_q8("axhip_rms_norm_q8", axhip::NORM, x, residual, weight, sum, q, scales, params, stream);
}
