// Sampling: the kernel.
#pragma once
#include "sample.hpp"

#include <type_traits>
#include <utility>

namespace axhip {
namespace {

// A work-group of 1024 threads to a row, which it holds in registers where it fits (IT steps of eight elements a lane).  A filter keeps a prefix of the order "larger
// logit first, equal ones by index", and where it ends is found by what lies in front (numbers of logits, or sums of weights).  The draw is the same search in
// the order of the indexes.  Weights are integers, multiples of 2^-43 of the largest, of which 2^20 fit 64 bits: sums do not depend on the order in which
// atomics arrive.  Three ways, by what is asked of the row:
//   * top_k up to SMALL_K (and short rows): of the threads' 1024 largest logits the k-th largest is a bound that at least k logits reach, and hardly more do (of k = 512, 1024 ln 2 = 710 where
//     they lie anywhere; a larger k would often leave more than there are threads).  On a steep row, where fewer than k weigh anything, the list is all that do.  An entry to a thread, they are
//     sorted by the order, and then those that are kept by index (a list of more than there are threads, of equal logits or near ones, goes the other ways).
//   * other 16-bit rows: all 65535 values are counted in LDS (128 KiB), and every filter is answered by the counts: one weight for each value that occurs
//     instead of one for each logit.  The draw takes weights from a table of the values that are kept.  Counts are 16 bits wide; if one overflows, the sum of all shows
//     it and the row goes the third way.
//   * other fp32 rows: a histogram of 2048 bins that are linear in the logit, from the largest to 31 temperatures below it, from where on weights round to zero (bins by the
//     bits of the float hold most logits in a few dozen bins, on which a wavefront's atomics wait for each other).  The logits in the bin in which a filter ends go to a list
//     in LDS if they fit, where the cut is found.  (Lists of all that is kept, for the draw, and weights formed of what is kept alone took as long as a pass over the row.)
// What bounds it: few rows the chain of dependent passes and barriers (fp32 1 x 51865, top_k: 8.9 us, of which 3 are the launch; bf16 64 x 51865, top_k, top_p and min_p: 15.2);
// 256 rows a CU's own work on its row.  bf16 256 x 128256, top_p, 49 us: 8 loading (at HBM's rate), 2 the largest, 11 counting (LDS atomics: a wavefront's 64 random banks take 12
// cycles), 5 the blocks' weights (64-bit operations), 3 the cut, 8 the draw's table look-ups, 3 the step it falls in.  (Rows of more than 65536 are held in 64 registers of a thread's 128, and a thread spills 44 bytes,
// f16 36.)  fp32, the same rows: without filters 61, top_k 45, top_p 129: a pass over the row takes
// 35 to 45, 200 cycles of a SIMD for each vector of 64 weights, half of them 64-bit operations.
constexpr int THREADS = 1024, WAVES = THREADS / WAVE, E = 8; // elements of a lane's vector
constexpr int STEP = WAVE * E;                               // consecutive elements of a wavefront's step
constexpr int BINS = 2048, FEW = 128;
constexpr int FEW_LOGITS = 1024, SMALL_K = 512;
constexpr int LIST = 16384;
constexpr int BLOCK = 64, BLOCKS = 65536 / BLOCK; // 16-bit values are summed up by blocks
static_assert(MOST_VOCAB <= int64_t(BINS) * STEP, "a bin for a step");
constexpr uint64_t ONE = uint64_t(1) << 43, MARK = uint64_t(1) << 53;
constexpr double REACH = 31.0; // temperatures: exp(-31) is below half of 2^-43

struct SampleShared {
    uint64_t bins[BINS];
    uint64_t block_mass[BLOCKS];
    uint64_t few_place[FEW], few_value[FEW];
    uint64_t scratch[WAVES + 2], other_scratch[WAVES];
    uint64_t pow2[32]; // 2^43 2^(i / 32), less i in the place to which scaled_weight adds it
    float top[WAVES];
    uint32_t where[WAVES], few, inside;
    union {
        uint64_t list[LIST];
        uint32_t counts[32768]; // two values to a word
        uint64_t weights[LIST];
    };
};
static_assert(sizeof(SampleShared) <= 160 * 1024, "LDS of a CU");

// ---- sums over a wavefront's lanes in 64 bits
template <int CTRL, int ROWS = 0xF> __device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v)), CTRL, ROWS, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v >> 32)), CTRL, ROWS, 0xF, false);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t sum16(uint64_t v) { // over rows of 16 lanes
    v += dpp64<0x128>(v); // row_ror:8, 4, 2, 1
    v += dpp64<0x124>(v);
    v += dpp64<0x122>(v);
    return v + dpp64<0x121>(v);
}
__device__ __forceinline__ uint64_t sum32(uint64_t v) { // over halves
    v = sum16(v);
    const auto lo = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(v), static_cast<uint32_t>(v), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(v >> 32), static_cast<uint32_t>(v >> 32), false, false);
    return (static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + (static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}
// x's sum in the first half's lanes, y's in the second's
__device__ __forceinline__ uint64_t sums_of_two(uint64_t x, uint64_t y) {
    const auto lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(x), static_cast<uint32_t>(y), false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y >> 32), false, false);
    return sum32((static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + (static_cast<uint64_t>(hi[1]) << 32 | lo[1]));
}
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
    v = sum32(v);
    const auto lo = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(v), static_cast<uint32_t>(v), false, false);
    const auto hi = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(v >> 32), static_cast<uint32_t>(v >> 32), false, false);
    return (static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + (static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}
__device__ __forceinline__ uint64_t wave_upto64(uint64_t v) { // of the lanes up to this one
    v += dpp64<0x111>(v); // row_shr:1, 2, 4, 8
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    v += dpp64<0x142, 0xA>(v); // the row in front, to rows 1 and 3
    return v + dpp64<0x143, 0xC>(v); // the first half, to the second
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v >> 32)), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(v)), lane));
}
// The sums of P values (a power of two from 2 to 16), value i in lanes [64 / P i, 64 / P (i + 1)): at each step a lane hands half of them over and adds up the other half.
template <int P> __device__ __forceinline__ uint64_t sums_of_many(uint64_t (&v)[P], int lane) {
    static_assert(P == 2 || P == 4 || P == 8 || P == 16, "a power of two");
    auto halve = [&](int p, auto swap) __attribute__((always_inline)) { // (swap(x, y): x's low and y's low lanes, x's high and y's high)
#pragma unroll
        for (int i = 0; i < (p > 1 ? p / 2 : 1); ++i) {
            const uint64_t x = v[i], y = v[p > 1 ? i + p / 2 : i];
            const auto lo = swap(static_cast<uint32_t>(x), static_cast<uint32_t>(y)), hi = swap(static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y >> 32));
            v[i] = (static_cast<uint64_t>(hi[0]) << 32 | lo[0]) + (static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
        }
    };
    auto step = [&](int p, int d, auto from) __attribute__((always_inline)) { // (from(x): x of the lane d away)
        if (p <= 1) {
            v[0] += from(v[0]);
            return;
        }
#pragma unroll
        for (int i = 0; i < p / 2; ++i) {
            const uint64_t mine = lane & d ? v[i + p / 2] : v[i], other = lane & d ? v[i] : v[i + p / 2];
            v[i] = mine + from(other);
        }
    };
    halve(P, [](uint32_t x, uint32_t y) { return __builtin_amdgcn_permlane32_swap(x, y, false, false); });
    halve(P / 2, [](uint32_t x, uint32_t y) { return __builtin_amdgcn_permlane16_swap(x, y, false, false); });
    step(P / 4, 8, [](uint64_t x) { return dpp64<0x128>(x); }); // (row_ror:8)
    step(P / 8, 4, [](uint64_t x) { return __shfl_xor(x, 4, WAVE); });
    v[0] += dpp64<0x4E>(v[0]); // (quad_perm: 2 and 1 apart)
    return v[0] + dpp64<0xB1>(v[0]);
}
template <int N, class F, int... I> __device__ __forceinline__ void unrolled_as(F f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F> __device__ __forceinline__ void unrolled(F f) { unrolled_as<N>(f, std::make_integer_sequence<int, N>{}); }
__device__ __forceinline__ uint32_t lanes_in_front(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0)); }
// A counter's old value; lane by lane (the compiler makes a sum over the wavefront of additions to one address, which is the longer way for the few lanes that come here)
__device__ __forceinline__ uint32_t take_from(uint32_t &counter, uint32_t n) {
    uint32_t offset = 0;
    asm volatile("" : "+v"(offset));
    return atomicAdd(&counter + offset, n);
}
__device__ __forceinline__ void add_to_bin(uint64_t &bin, uint64_t v) { atomicAdd(reinterpret_cast<unsigned long long *>(&bin), static_cast<unsigned long long>(v)); }

// ---- the order: smaller numbers first.  Larger logits (-0 is +0), and of equal ones smaller indexes.
__device__ __forceinline__ uint64_t order_of(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return static_cast<uint64_t>(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu) << 20 | i;
}
__device__ __forceinline__ float logit_of(uint64_t order) {
    const uint32_t b = static_cast<uint32_t>(order >> 20);
    return __uint_as_float(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu);
}
__device__ __forceinline__ uint32_t index_of(uint64_t order) { return static_cast<uint32_t>(order) & 0xFFFFFu; }

// The same of two 16-bit logits at a time: 0x7FFF - h of a positive one, h - 1 of a negative one (so that -0 has the number of +0).
typedef uint16_t pair_t __attribute__((ext_vector_type(2)));
typedef int16_t signed_pair_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ pair_t orders_of(uint32_t w) {
    const signed_pair_t sign = __builtin_bit_cast(signed_pair_t, w) >> static_cast<int16_t>(15); // -1 or 0
    const uint32_t m = ~__builtin_bit_cast(uint32_t, sign) & 0x7FFF7FFFu;
    return __builtin_bit_cast(pair_t, w ^ m) + __builtin_bit_cast(pair_t, sign);
}
__device__ __forceinline__ uint32_t order_of16(uint32_t h) { return orders_of(h)[0]; }
template <int DT> constexpr uint32_t INFINITY16 = DT == AXHIP_DTYPE_BF16 ? 0x7F80u : 0x7C00u;
template <int DT> constexpr uint32_t FIRST_ORDER = 0x7FFFu ^ INFINITY16<DT>;                                    // of infinity,
template <int DT> constexpr uint32_t DRAWN_ORDERS = (0x8000u | INFINITY16<DT>) - 1 - FIRST_ORDER<DT>;          // and how many there are before -infinity and the NaNs
template <int DT> __device__ __forceinline__ float logit_of16(uint32_t order) {
    const uint32_t h = order <= 0x7FFFu ? order ^ 0x7FFFu : order + 1;
    return DT == AXHIP_DTYPE_BF16 ? bf16_bits_to_f32(h) : f16_bits_to_f32(h);
}

template <int DT> struct Step { uint4_t v[DT == AXHIP_DTYPE_F32 ? 2 : 1]; };
template <int DT> __device__ __forceinline__ float element(const Step<DT> &s, int e) {
    if constexpr (DT == AXHIP_DTYPE_F32) return __uint_as_float(s.v[e / 4][e % 4]);
    else if constexpr (DT == AXHIP_DTYPE_BF16) return e % 2 ? __uint_as_float(s.v[0][e / 2] & 0xFFFF0000u) : __uint_as_float(s.v[0][e / 2] << 16);
    else return f16_bits_to_f32((s.v[0][e / 2] >> (16 * (e % 2))) & 0xFFFFu);
}

template <int DT> struct Row {
    const char *logits;
    int vocab;
    float top = 0.0f;      // the largest logit
    double base = 0.0;     // ... or the largest finite number
    double rate = 0.0;     // log2(e) / temperature
    float floor = 0.0f;    // from here on weights may be more than nothing
    float lowest = 0.0f, highest = 0.0f; // finite bounds of what powers are formed of
    const uint64_t *pow2 = nullptr;
    uint64_t last = ~0ull; // kept: up to this one in the order (the one of last_index among the logits that equal last_logit),
    float last_logit = -__builtin_inff();
    uint32_t last_index = 0;
    double least = 0.0; // and with at least this weight

    __device__ __forceinline__ Step<DT> load(int step) const {
        constexpr int ES = DT == AXHIP_DTYPE_F32 ? 4 : 2;
        const int at = step * STEP + static_cast<int>(threadIdx.x % WAVE) * E;
        Step<DT> s;
        if (at + E <= vocab) {
#pragma unroll
            for (int i = 0; i < ES / 2; ++i) s.v[i] = reinterpret_cast<const uint4_unaligned_t *>(logits + static_cast<int64_t>(at) * ES + 16 * i)->v;
        } else { // (past the end: NaN, which is never drawn)
#pragma unroll
            for (int i = 0; i < ES / 2; ++i) s.v[i] = uint4_t{~0u, ~0u, ~0u, ~0u};
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (at + e < vocab) {
                    if constexpr (ES == 4) s.v[e / 4][e % 4] = reinterpret_cast<const uint32_t *>(logits)[at + e];
                    else s.v[0][e / 2] = e % 2 ? (s.v[0][e / 2] & 0xFFFFu) | static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(logits)[at + e]) << 16
                                              : (s.v[0][e / 2] & 0xFFFF0000u) | reinterpret_cast<const uint16_t *>(logits)[at + e];
                }
        }
        return s;
    }
    __device__ __forceinline__ int steps() const { return (vocab + STEP - 1) / STEP; }

    // log2 of the weight, 0 at most and -90 at least: logits below the floor count as the floor (NaN too), an infinite one as the largest finite number.
    __device__ __forceinline__ double power(float v) const { return (static_cast<double>(__builtin_amdgcn_fmed3f(v, lowest, highest)) - base) * rate; }
    // exp((v - top) / temperature) in multiples of 2^-43: 2^z with z = i / 32 + r, |r| <= 1/64: 2^(i / 32) from a table in LDS (of 64 banks: no two lanes wait for each
    // other), with the power of two put into its exponent, and five terms of 2^r, which leave less than 3e-15 of the weight.  (Operations of 64 bits take a wavefront eight
    // cycles, others four: eleven terms and no table took a fifth longer.)
    __device__ __forceinline__ double scaled_weight(double z) const {
        constexpr double SPLIT = 211106232532992.0; // 1.5 * 2^47: its last bit is 1/32
        const double t = z + SPLIT, r = z - (t - SPLIT);
        const uint32_t i = static_cast<uint32_t>(__double_as_longlong(t));
        const uint64_t power_of_two = pow2[i & 31] + (static_cast<uint64_t>(i << 15) << 32);
        double p = 0.0013333558146428443;
        p = __builtin_fma(r, p, 0.009618129107628477);
        p = __builtin_fma(r, p, 0.05550410866482158);
        p = __builtin_fma(r, p, 0.2402265069591007);
        p = __builtin_fma(r, p, 0.6931471805599453);
        p = __builtin_fma(r, p, 1.0);
        return __longlong_as_double(static_cast<long long>(power_of_two)) * p;
    }
    static __device__ __forceinline__ uint64_t integer(double w) {
        constexpr double TO_INTEGER = 4503599627370496.0; // 2^52: the integer is what its last bits say
        return static_cast<uint64_t>(__double_as_longlong(w + TO_INTEGER)) & ((uint64_t(1) << 52) - 1);
    }
    // (formed for all lanes, eight chains at a time, whether or not a lane's is used: behind a branch each would wait for the one before)
    static __device__ __forceinline__ uint64_t formed(uint64_t x) {
        uint32_t lo = static_cast<uint32_t>(x), hi = static_cast<uint32_t>(x >> 32);
        asm("" : "+v"(lo), "+v"(hi));
        return static_cast<uint64_t>(hi) << 32 | lo;
    }
    __device__ __forceinline__ uint64_t mass(float v) const { return integer(scaled_weight(power(v))); }
    // ... 0 below min_p, and of what is not kept
    __device__ __forceinline__ uint64_t mass_of_least(float v, bool kept = true) const {
        const double w = scaled_weight(power(v));
        return integer(kept && w >= least ? w : 0.0);
    }
    // bins of the power, BINS to REACH temperatures; the last one holds everything from there on
    __device__ __forceinline__ uint32_t bin_of_power(double z) const {
        constexpr double PER_POWER = (BINS - 1) / (REACH * 1.4426950408889634), TO_INTEGER = 4503599627370496.0;
        return min(static_cast<uint32_t>(__double_as_longlong(__builtin_fma(z, -PER_POWER, TO_INTEGER))), static_cast<uint32_t>(BINS - 1));
    }
    __device__ __forceinline__ uint32_t bin_of(float v) const { return bin_of_power(power(v)); }
    // Below every logit of bins up to `bin` (-inf where rounding leaves nothing to say).
    __device__ __forceinline__ float below(int bin) const {
        const double edge = base - (bin + 2) * (REACH * 1.4426950408889634 / (BINS - 1)) / rate;
        const float low = static_cast<float>(edge) - fabsf(static_cast<float>(edge)) * 1e-6f;
        return low > -3e38f ? low : -3.402823466e38f;
    }
    // The smallest float of bins up to `bin`, not below `from` (by a whole wavefront: in each round its lanes look at 64 places of what is left)
    __device__ __forceinline__ float smallest_up_to(int bin, float from) const {
        auto key_of = [](float v) { return __float_as_uint(v) ^ (__float_as_uint(v) & 0x80000000u ? ~0u : 0x80000000u); };
        auto float_of = [](uint32_t key) { return __uint_as_float(key ^ (key & 0x80000000u ? 0x80000000u : ~0u)); };
        uint32_t lo = key_of(from), hi = key_of(top); // (the largest logit's bin is the first)
        while (lo < hi) {
            const uint32_t at = lo + static_cast<uint32_t>(static_cast<uint64_t>(hi - lo) * (threadIdx.x % WAVE) / WAVE);
            const uint64_t reached = __ballot(static_cast<int>(bin_of(float_of(at))) <= bin);
            const int first = reached ? __builtin_ctzll(reached) : WAVE; // (they are in order: from this one on)
            const uint32_t at_first = __builtin_amdgcn_readlane(at, first % WAVE), in_front = __builtin_amdgcn_readlane(at, (first + WAVE - 1) % WAVE);
            if (first == 0) hi = lo;
            else {
                lo = in_front + 1;
                if (first < WAVE) hi = at_first;
            }
        }
        return float_of(lo);
    }
    __device__ __forceinline__ void keep_up_to(uint64_t order) {
        last = order;
        last_logit = logit_of(order);
        last_index = index_of(order);
    }
    __device__ __forceinline__ bool counts(float v, uint32_t i) const { return v >= floor && (v > last_logit || (v == last_logit && i <= last_index)); }
};

// ---- All of these are called by the whole work-group, and their answers are every thread's.
__device__ __forceinline__ void clear_bins(SampleShared &sh) {
    sh.bins[threadIdx.x] = 0;
    sh.bins[threadIdx.x + THREADS] = 0;
    __syncthreads();
}
__device__ __forceinline__ uint64_t sum_of_all(SampleShared &sh, uint64_t v) {
    v = wave_sum64(v);
    if (threadIdx.x % WAVE == 0) sh.other_scratch[threadIdx.x / WAVE] = v;
    __syncthreads();
    v = sum16(sh.other_scratch[threadIdx.x % WAVES]);
    __syncthreads();
    return v;
}
// (behind a barrier behind the additions to the bins)
__device__ __forceinline__ uint64_t sum_of_bins(SampleShared &sh) { return sum_of_all(sh, sh.bins[threadIdx.x] + sh.bins[threadIdx.x + THREADS]); }
// The first bin at which the running sum, `before` in front, exceeds `than`, and the sum in front of it; -1 if none does.
__device__ __forceinline__ int find_bin(SampleShared &sh, uint64_t before, uint64_t than, uint64_t &in_front) {
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
    const uint64_t v0 = sh.bins[2 * t], v1 = sh.bins[2 * t + 1], upto = wave_upto64(v0 + v1);
    if (lane == WAVE - 1) sh.scratch[wave] = upto;
    if (t == 0) sh.scratch[WAVES] = ~0ull;
    __syncthreads();
    const uint64_t others = sum16(lane % WAVES < wave ? sh.scratch[lane % WAVES] : 0);
    const uint64_t all = before + others + upto, mine = all - v0 - v1;
    if (all > than && mine <= than) {
        sh.scratch[WAVES] = mine + v0 > than ? 2 * t : 2 * t + 1;
        sh.scratch[WAVES + 1] = mine + v0 > than ? mine : mine + v0;
    }
    __syncthreads();
    const int bin = static_cast<int>(sh.scratch[WAVES]);
    in_front = sh.scratch[WAVES + 1];
    __syncthreads();
    return bin;
}
__device__ __forceinline__ void smallest_and_largest(SampleShared &sh, uint64_t &lo, uint64_t &hi) {
#pragma unroll
    for (int d = 32; d; d /= 2) {
        const uint64_t l = __shfl_xor(lo, d, WAVE), h = __shfl_xor(hi, d, WAVE);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
    }
    if (threadIdx.x % WAVE == 0) {
        sh.scratch[threadIdx.x / WAVE] = lo;
        sh.other_scratch[threadIdx.x / WAVE] = hi;
    }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) {
        lo = sh.scratch[w] < lo ? sh.scratch[w] : lo;
        hi = sh.other_scratch[w] > hi ? sh.other_scratch[w] : hi;
    }
    __syncthreads();
}

// The number of the lane D away (D a power of two).
template <int D> __device__ __forceinline__ uint64_t lane_across(uint64_t v, int lane) {
    if constexpr (D == 1) return dpp64<0xB1>(v); // (quad_perm)
    else if constexpr (D == 2) return dpp64<0x4E>(v);
    else if constexpr (D == 4) return dpp64<0x1B>(dpp64<0x141>(v)); // (7 away, 3 away)
    else if constexpr (D == 8) return dpp64<0x128>(v);
    else {
        const uint32_t low = static_cast<uint32_t>(v), high = static_cast<uint32_t>(v >> 32);
        const auto lo = D == 16 ? __builtin_amdgcn_permlane16_swap(low, low, false, false) : __builtin_amdgcn_permlane32_swap(low, low, false, false);
        const auto hi = D == 16 ? __builtin_amdgcn_permlane16_swap(high, high, false, false) : __builtin_amdgcn_permlane32_swap(high, high, false, false);
        return lane & D ? static_cast<uint64_t>(hi[0]) << 32 | lo[0] : static_cast<uint64_t>(hi[1]) << 32 | lo[1];
    }
}
// Numbers, one to a thread of the first `waves` wavefronts (a power of two), the smallest to the first thread and so on: a bitonic sort, by exchanges between lanes where they are of
// one wavefront and through LDS (`room`, two numbers a thread) where not.  Called by the whole work-group.
__device__ __forceinline__ uint64_t sorted(uint64_t *room, uint64_t v, int waves) {
    const int t = threadIdx.x, lane = t % WAVE;
    auto keep = [&](uint64_t other, int d, bool up) __attribute__((always_inline)) { v = (other < v) == (up == ((t & d) == 0)) ? other : v; };
    auto within = [&](auto from, bool up) __attribute__((always_inline)) { // distances from `from` down
        constexpr int D = decltype(from)::value;
        if constexpr (D >= 32) keep(lane_across<32>(v, lane), 32, up);
        if constexpr (D >= 16) keep(lane_across<16>(v, lane), 16, up);
        if constexpr (D >= 8) keep(lane_across<8>(v, lane), 8, up);
        if constexpr (D >= 4) keep(lane_across<4>(v, lane), 4, up);
        if constexpr (D >= 2) keep(lane_across<2>(v, lane), 2, up);
        keep(lane_across<1>(v, lane), 1, up);
    };
    const bool mine = t < waves * WAVE;
    if (mine) {
        within(std::integral_constant<int, 1>{}, (t & 2) == 0);
        within(std::integral_constant<int, 2>{}, (t & 4) == 0);
        within(std::integral_constant<int, 4>{}, (t & 8) == 0);
        within(std::integral_constant<int, 8>{}, (t & 16) == 0);
        within(std::integral_constant<int, 16>{}, (t & 32) == 0);
        within(std::integral_constant<int, 32>{}, (t & 64) == 0 || waves == 1);
    }
    int half = 0;
    for (int size = 2 * WAVE; size <= waves * WAVE; size *= 2) {
        const bool up = (t & size) == 0 || size == waves * WAVE;
        for (int d = size / 2; d >= WAVE; d /= 2, half ^= THREADS) {
            if (mine) room[half + t] = v;
            __syncthreads(); // (the numbers of the step before last have been read)
            if (mine) keep(room[half + (t ^ d)], d, up);
        }
        if (mine) within(std::integral_constant<int, 32>{}, up);
    }
    __syncthreads();
    return v;
}
// The sum of the threads in front of this one, and of all.
__device__ __forceinline__ uint64_t sum_in_front(SampleShared &sh, uint64_t v, uint64_t &total) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    const uint64_t upto = wave_upto64(v);
    if (lane == WAVE - 1) sh.scratch[wave] = upto;
    __syncthreads();
    const uint64_t other = sh.scratch[lane % WAVES];
    total = sum16(other);
    const uint64_t front = sum16(lane % WAVES < wave ? other : 0) + upto - v;
    __syncthreads();
    return front;
}

// Of the elements that `all(f)` hands to f(place, value()), those with places in [lo, hi]: the place at which the running sum of values, by place and with `before` in
// front, exceeds than(sum of them all) -- hi if it never does.  Places are unique, values may be 0.  `count`: how many they are at most.
template <class Than, class All> __device__ __forceinline__ uint64_t find_place(SampleShared &sh, uint64_t lo, uint64_t hi, uint64_t before, int count, Than than_of, All all) {
    uint64_t than = 0;
    for (bool first = true; lo < hi; first = false) {
        // (each round leaves a bin, at most 1 / 2047 of the places, or fewer than FEW elements)
        const double rate = (BINS - 0.5) / (static_cast<double>(hi - lo) + 1.0);
        auto bin_of = [&](uint64_t place) { return static_cast<int>(static_cast<double>(place - lo) * rate); };
        const bool all_few = first && count <= FEW;
        int bin = 0;
        if (threadIdx.x == 0) sh.few = 0;
        if (!all_few) {
            clear_bins(sh);
            all([&](uint64_t place, auto value) __attribute__((always_inline)) {
                if (place >= lo && place <= hi) {
                    const uint64_t v = value();
                    if (v) add_to_bin(sh.bins[bin_of(place)], v);
                }
            });
            __syncthreads();
            if (first) than = than_of([&] { return sum_of_bins(sh); });
            bin = find_bin(sh, before, than, before);
            if (bin < 0) return hi;
        } else {
            __syncthreads();
        }
        uint64_t l = ~0ull, h = 0;
        all([&](uint64_t place, auto value) __attribute__((always_inline)) {
            if (place >= lo && place <= hi && (all_few || bin_of(place) == bin)) {
                const uint64_t v = value();
                if (v) {
                    const uint32_t at = take_from(sh.few, 1);
                    if (at < FEW) {
                        sh.few_place[at] = place;
                        sh.few_value[at] = v;
                    }
                    l = place < l ? place : l;
                    h = place > h ? place : h;
                }
            }
        });
        __syncthreads();
        const int n = static_cast<int>(sh.few);
        if (n <= FEW) {
            if (all_few) than = than_of([&] { return sum_of_all(sh, static_cast<int>(threadIdx.x) < n ? sh.few_value[threadIdx.x] : 0); });
            if (threadIdx.x == 0) sh.scratch[WAVES] = hi;
            __syncthreads();
            if (static_cast<int>(threadIdx.x) < n) {
                const uint64_t mine = sh.few_place[threadIdx.x];
                uint64_t front = before;
                for (int i = 0; i < n; ++i) front += sh.few_place[i] < mine ? sh.few_value[i] : 0;
                if (front <= than && front + sh.few_value[threadIdx.x] > than) sh.scratch[WAVES] = mine;
            }
            __syncthreads();
            lo = sh.scratch[WAVES];
            __syncthreads();
            return lo;
        }
        smallest_and_largest(sh, l, h);
        lo = l;
        hi = h;
    }
    return lo;
}

template <int DT, int IT> __global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char sample_lds[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(sample_lds);
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
    const int64_t row = blockIdx.x;
    constexpr int64_t ES = DT == AXHIP_DTYPE_F32 ? 4 : 2;
    Row<DT> r{static_cast<const char *>(a.logits) + row * a.ld * ES, a.vocab};
    const int steps = r.steps();
    Step<DT> held[IT > 0 ? IT : 1];
#pragma unroll
    for (int i = 0; i < IT; ++i)
        if (i * WAVES + wave < steps) held[i] = r.load(i * WAVES + wave);
    // f(vectors, index of the first, step) for the wavefront's steps, from memory with the next ones' loads in flight
    auto each_step_of_memory = [&](auto f) __attribute__((always_inline)) {
        constexpr int AHEAD = 2; // (sets of registers of their own: moved from one to the next, every load would be waited for)
        Step<DT> next[AHEAD];
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) next[d] = r.load(min(wave + d * WAVES, steps - 1));
#pragma unroll 1
        for (int step = wave; step < steps; step += AHEAD * WAVES) {
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) {
                if (step + d * WAVES < steps) f(next[d], static_cast<uint32_t>((step + d * WAVES) * STEP + lane * E), step + d * WAVES);
                next[d] = r.load(min(step + (d + AHEAD) * WAVES, steps - 1));
            }
        }
    };
    // ... from the registers, for passes of few instructions.  (The compiler is not to see that a later pass forms the same numbers of the same vectors: it would keep them all.)
    auto each_step_at = [&](auto f) __attribute__((always_inline)) { // f(vectors, index of the first, their place in `held`)
        int first = lane * E;
        unrolled<IT>([&](auto place) __attribute__((always_inline)) {
            constexpr int i = decltype(place)::value;
            const int step = i * WAVES + wave;
            Step<DT> s = held[i];
#pragma unroll
            for (int v = 0; v < ES / 2; ++v)
#pragma unroll
                for (int w = 0; w < 4; ++w) asm volatile("" : "+v"(s.v[v][w]));
            asm volatile("" : "+v"(first));
            if (step < steps) f(s, static_cast<uint32_t>(step * STEP + first), place);
        });
    };
    auto each_step = [&](auto f) __attribute__((always_inline)) {
        if constexpr (IT > 0) each_step_at([&](const Step<DT> &s, uint32_t at, auto place) __attribute__((always_inline)) { f(s, at, decltype(place)::value * WAVES + wave); });
        else each_step_of_memory(f);
    };
    auto each_of = [&](auto steps_of, auto f) __attribute__((always_inline)) { // f(logit, index)
        steps_of([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < E; ++e) f(element<DT>(s, e), at + e);
        });
    };

    float temperature = a.temperature ? a.temperature[row] : a.all_temperature;
    temperature = temperature > 1e30f ? 1e30f : temperature;
    const float p = a.top_p ? a.top_p[row] : a.all_top_p, m = a.min_p ? a.min_p[row] : a.all_min_p, u = a.u[row];
    const int32_t asked = a.top_k ? a.top_k[row] : a.all_top_k, k = asked > 0 && asked < a.vocab ? asked : 0;
    if (t == 0) sh.inside = 0;
    if (t < 32) sh.pow2[t] = static_cast<uint64_t>(__double_as_longlong(exp2(43.0 + t * (1.0 / 32.0)))) - (uint64_t(t) << 47); // (a barrier before they are used)
    r.pow2 = sh.pow2;
    sh.bins[t] = 0;
    sh.bins[t + THREADS] = 0;

    // kept by top_p: those with less than p of the sum in front of them, so up to the one at which the running sum reaches p of it
    auto than_of_p = [&](auto total) __attribute__((always_inline)) {
        const double reach = static_cast<double>(p) * static_cast<double>(total());
        return reach > 1.0 ? static_cast<uint64_t>(__builtin_ceil(reach)) - 1 : uint64_t(0);
    };
    auto than_of_u = [&](uint64_t total) __attribute__((always_inline)) {
        const double reach = u > 0.0f ? static_cast<double>(u) * static_cast<double>(total) : 0.0;
        return reach < static_cast<double>(total - 1) ? static_cast<uint64_t>(reach) : total - 1;
    };
    auto answer = [&](uint32_t index, uint64_t mass, uint64_t total) {
        a.tokens[row] = static_cast<int64_t>(index);
        if (a.probs) a.probs[row] = static_cast<float>(static_cast<double>(mass) / static_cast<double>(total));
    };

    // ---- the largest logit
    float mine = -__builtin_inff(); // of this thread's
    each_of(each_step, [&](float v, uint32_t) { mine = fmaxf(mine, v); });
    float top = wave_max(mine);
    if (lane == 0) sh.top[wave] = top;
    __syncthreads();
    top = sh.top[lane % WAVES];
    top = wave_max(top);
    if (top == -__builtin_inff() || !(temperature > 0.0f)) { // (the same in every thread)
        uint32_t first = ~0u;
        if (top != -__builtin_inff()) each_of(each_step_of_memory, [&](float v, uint32_t i) { first = v == top ? min(first, i) : first; });
#pragma unroll
        for (int d = 32; d; d /= 2) first = min(first, static_cast<uint32_t>(__shfl_xor(first, d, WAVE)));
        if (lane == 0) sh.where[wave] = first;
        __syncthreads();
        for (int w = 0; w < WAVES; ++w) first = min(first, sh.where[w]);
        if (t == 0) {
            a.tokens[row] = first == ~0u ? -1 : static_cast<int64_t>(first);
            if (a.probs) a.probs[row] = first == ~0u ? 0.0f : 1.0f;
        }
        return;
    }
    constexpr float LARGEST = 3.402823466e38f;
    r.top = top;
    r.base = static_cast<double>(fminf(top, LARGEST));
    r.rate = 1.4426950408889634 / static_cast<double>(temperature);
    r.floor = fmaxf(top - static_cast<float>(REACH) * temperature, -LARGEST); // (NaN, of an infinite logit and temperature: everything finite)
    if (top > LARGEST) r.floor = top;                                         // (only its equals)
    r.lowest = fminf(r.floor, LARGEST);
    r.highest = fminf(top, LARGEST);
    const double least = m > 0.0f ? (m < 1.0f ? static_cast<double>(m) : 1.0) * static_cast<double>(ONE) : 0.0;
    r.least = least;

    // Those for which `taken(logit, index)` holds to the list (as many as it has room for); how many there are.
    auto gather = [&](auto taken) __attribute__((always_inline)) {
        each_step_of_memory([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
            uint64_t lanes[E];
            uint32_t n = 0, before = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                lanes[e] = __ballot(taken(element<DT>(s, e), at + e));
                n += __builtin_popcountll(lanes[e]);
            }
            if (n == 0) return;
            if (lane == 0) before = take_from(sh.inside, n);
            before = __builtin_amdgcn_readfirstlane(before);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t to = before + lanes_in_front(lanes[e]);
                if ((lanes[e] >> lane & 1) && to < LIST) sh.list[to] = order_of(element<DT>(s, e), at + e);
                before += __builtin_popcountll(lanes[e]);
            }
        });
        __syncthreads();
        const int n = static_cast<int>(sh.inside);
        __syncthreads();
        if (t == 0) sh.inside = 0;
        return n;
    };

    // ================ top_k of a few, short rows: a list of little more than what is kept
    if ((k && k <= SMALL_K) || a.vocab <= FEW_LOGITS) {
        float low = r.floor;
        if (a.vocab > FEW_LOGITS) { // (the bins are clear: a barrier ago)
            if (a.vocab >= THREADS * E) {
                if (mine >= r.floor) add_to_bin(sh.bins[r.bin_of(mine)], 1);
            } else { // (too few threads have any: all logits)
                each_of(each_step_of_memory, [&](float v, uint32_t) {
                    if (v >= r.floor) add_to_bin(sh.bins[r.bin_of(v)], 1);
                });
            }
            __syncthreads();
            uint64_t in_front;
            const int bin = find_bin(sh, 0, static_cast<uint64_t>(k - 1), in_front);
            if (bin >= 0 && bin < BINS - 1) low = fmaxf(low, r.below(bin)); // (or there are fewer than k that weigh anything: all of them)
        }
        // each wavefront's to a part of the list of its own
        constexpr uint32_t PART = LIST / WAVES;
        uint32_t own = 0;
        each_step([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
            float largest = element<DT>(s, 0);
#pragma unroll
            for (int e = 1; e < E; ++e) largest = fmaxf(largest, element<DT>(s, e));
            if (__ballot(largest >= low) == 0) return;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float v = element<DT>(s, e);
                const uint64_t taken = __ballot(v >= low);
                if (taken == 0) continue;
                const uint32_t to = own + lanes_in_front(taken);
                if (v >= low && to < PART) sh.list[wave * PART + to] = order_of(v, at + e);
                own += __builtin_popcountll(taken);
            }
        });
        if (lane == 0) sh.where[wave] = own;
        __syncthreads();
        uint32_t in_front = 0, n = 0;
        for (int w = 0; w < WAVES; ++w) {
            in_front += w < wave ? sh.where[w] : 0;
            n += sh.where[w];
        }
        if (n <= THREADS) { // an entry to a thread
            uint64_t *const entries = sh.bins;
            for (uint32_t i = lane; i < own; i += WAVE) entries[in_front + i] = sh.list[wave * PART + i];
            __syncthreads();
            uint64_t o = static_cast<uint32_t>(t) < n ? entries[t] : ~0ull, total;
            int waves = 1;
            while (waves * WAVE < static_cast<int>(n)) waves *= 2;
            if (k || p < 1.0f) o = sorted(sh.list, o, waves);
            // (in their order: what lies in front of an entry is what the threads in front hold)
            bool kept = static_cast<uint32_t>(t) < n && (k == 0 || t < k);
            const float v = logit_of(o);
            if (p < 1.0f) {
                const uint64_t front = sum_in_front(sh, kept ? r.mass(v) : 0, total);
                kept = kept && front <= than_of_p([&] { return total; });
            }
            // by index, with their weights: 20 and 44 bits
            static_assert(MOST_VOCAB <= int64_t(1) << 20 && ONE < uint64_t(1) << 44, "one number for both");
            const uint64_t mass = kept ? r.mass_of_least(v) : 0;
            const uint64_t drawn = sorted(sh.list, mass ? static_cast<uint64_t>(index_of(o)) << 44 | mass : ~0ull, waves);
            const uint64_t x = drawn != ~0ull ? drawn & ((uint64_t(1) << 44) - 1) : 0;
            const uint64_t front = sum_in_front(sh, x, total), than = than_of_u(total);
            if (front <= than && front + x > than) answer(static_cast<uint32_t>(drawn >> 44), x, total);
            return;
        }
        __syncthreads(); // (many equal ones: the other ways)
    }

    // The draw by the sums of the wavefronts' steps, and then within one.  masses(vectors, index of the first, sums): of a lane's eight, MARK for a logit of which only the first
    // `ties` are kept, with the weight `of_tie` each.
    auto draw_by_steps = [&](auto in_registers, uint64_t of_tie, uint32_t ties, auto masses) __attribute__((always_inline)) {
        constexpr bool HELD = decltype(in_registers)::value;
        clear_bins(sh);
        if constexpr (HELD && IT > 0) { // (weights of a step are 2^52 at most, marks 512)
            constexpr int N = IT > 0 ? IT : 2;
            uint64_t sums[N];
#pragma unroll
            for (int i = 0; i < N; ++i) sums[i] = 0;
            each_step_at([&](const Step<DT> &s, uint32_t at, auto place) __attribute__((always_inline)) {
                uint64_t x[E];
                masses(s, at, x);
#pragma unroll
                for (int e = 0; e < E; ++e) sums[place.value] += x[e];
            });
            const uint64_t sum = sums_of_many<N>(sums, lane);
            const int step = lane / (WAVE / N) * WAVES + wave;
            if (lane % (WAVE / N) == 0 && step < steps) sh.bins[step] = sum;
        } else {
            each_step_of_memory([&](const Step<DT> &s, uint32_t at, int step) __attribute__((always_inline)) {
                uint64_t x[E], sum = 0;
                masses(s, at, x);
#pragma unroll
                for (int e = 0; e < E; ++e) sum += x[e];
                sum = wave_sum64(sum);
                if (lane == 0) sh.bins[step] = sum;
            });
        }
        __syncthreads();
        uint64_t marks_in_front = 0; // of the step that is looked for
        if (of_tie) { // marks -> the weights of those that are kept
            const uint64_t b0 = sh.bins[2 * t], b1 = sh.bins[2 * t + 1], m0 = b0 / MARK, m1 = b1 / MARK, upto = wave_upto64(m0 + m1);
            if (lane == WAVE - 1) sh.scratch[wave] = upto;
            __syncthreads();
            const uint64_t in_front = sum16(lane % WAVES < wave ? sh.scratch[lane % WAVES] : 0) + upto - m0 - m1;
            auto kept = [&](uint64_t before, uint64_t marks) { return before >= ties ? uint64_t(0) : min(marks, ties - before); };
            sh.bins[2 * t] = b0 % MARK + kept(in_front, m0) * of_tie;
            sh.bins[2 * t + 1] = b1 % MARK + kept(in_front + m0, m1) * of_tie;
            sh.block_mass[t] = in_front; // (in front of step 2 t; the other's are m0 more, whose steps are looked at again)
            __syncthreads();
        }
        const uint64_t total = sum_of_bins(sh), than = than_of_u(total);
        uint64_t front;
        const int step = max(find_bin(sh, 0, than, front), 0); // (the largest logit's weight is there, and `than` is below the sum)
        if (wave == 0) {
            const uint32_t at = static_cast<uint32_t>(step * STEP + lane * E);
            uint64_t x[E], own = 0;
            if (of_tie) {
                marks_in_front = sh.block_mass[step / 2];
                if (step % 2) {
                    masses(r.load(step - 1), at - STEP, x);
#pragma unroll
                    for (int e = 0; e < E; ++e) own += x[e] / MARK;
                    marks_in_front += wave_sum64(own);
                }
            }
            masses(r.load(step), at, x);
            if (of_tie) {
                own = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) own += x[e] / MARK;
                uint64_t before = marks_in_front + wave_upto64(own) - own;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (x[e] == MARK) x[e] = before++ < ties ? of_tie : 0;
            }
            own = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) own += x[e];
            const uint64_t upto = front + wave_upto64(own);
            front = upto - own;
            if (upto > than && front <= than) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (front <= than && front + x[e] > than) answer(at + e, x[e], total);
                    front += x[e];
                }
            }
        }
    };

    // ================ 16-bit logits: counts of their values
    if (DT != AXHIP_DTYPE_F32) {
        const bool filtered = k || p < 1.0f; // (else there is nothing to count)
        // The count of order o is a half of word o % 32768 (values next to each other lie in different banks).
        auto count_at = [&](uint32_t order) { return (sh.counts[order & 0x7FFFu] >> (order >> 15 << 4)) & 0xFFFFu; };
        if (filtered)
            for (int i = t; i < 8192; i += THREADS) reinterpret_cast<uint4_t *>(sh.counts)[i] = uint4_t{0, 0, 0, 0};
        clear_bins(sh); // (and a barrier)
        uint32_t drawn = 0;
        if (filtered)
            each_step([&](const Step<DT> &s, uint32_t, int) __attribute__((always_inline)) {
                // (most steps hold nothing that is never drawn: no look at every logit)
                pair_t farthest = pair_t{0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) farthest = __builtin_elementwise_max(farthest, orders_of(s.v[0][i]) - static_cast<uint16_t>(FIRST_ORDER<DT>));
                const bool whole = max(farthest[0], farthest[1]) < DRAWN_ORDERS<DT>;
                const bool all_whole = __ballot(!whole) == 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t orders = __builtin_bit_cast(uint32_t, orders_of(s.v[0][i])), halves = orders >> 11 & 0x00100010u; // 16 for counts in the upper half
                    uint32_t *const first = &sh.counts[orders & 0x7FFFu], *const second = &sh.counts[orders >> 16 & 0x7FFFu];
                    const uint32_t one = 1u << (halves & 31u), other = 1u << (halves >> 16);
                    if (all_whole) {
                        atomicAdd(first, one);
                        atomicAdd(second, other);
                    } else {
                        const pair_t at = __builtin_bit_cast(pair_t, orders) - static_cast<uint16_t>(FIRST_ORDER<DT>);
                        if (at[0] < DRAWN_ORDERS<DT>) {
                            ++drawn;
                            atomicAdd(first, one);
                        }
                        if (at[1] < DRAWN_ORDERS<DT>) {
                            ++drawn;
                            atomicAdd(second, other);
                        }
                    }
                }
                if (all_whole) drawn += E;
            });
        __syncthreads();
        // f(counts of the lane's value in block j and in block j + BLOCKS / 2, its order in the first) where either has any, a sum for each block; the others' sums are 0
        auto sum_blocks = [&](auto f) __attribute__((always_inline)) {
            constexpr int TOGETHER = 8;
#pragma unroll 1
            for (int j0 = wave; j0 < BLOCKS / 2; j0 += WAVES * TOGETHER) {
                uint32_t w[TOGETHER];
#pragma unroll
                for (int i = 0; i < TOGETHER; ++i) w[i] = sh.counts[BLOCK * (j0 + WAVES * i) + lane];
#pragma unroll 1
                for (int i = 0; i < TOGETHER; ++i) {
                    uint32_t pair = w[0];
#pragma unroll
                    for (int d = 0; d + 1 < TOGETHER; ++d) w[d] = w[d + 1];
                    if (__ballot(pair != 0) == 0) continue;
                    const int j = j0 + WAVES * i;
                    uint64_t of_first, of_second;
                    f(pair & 0xFFFFu, pair >> 16, static_cast<uint32_t>(BLOCK * j + lane), of_first, of_second);
                    const uint64_t sum = sums_of_two(of_first, of_second);
                    if (lane % 32 == 0) sh.bins[lane ? j + BLOCKS / 2 : j] = sum;
                }
            }
        };
        static_assert(BLOCKS / 2 % (WAVES * 8) == 0 && BLOCK == WAVE && BLOCKS <= BINS, "whole rounds, a value to a lane, and a bin for a block");
        uint32_t counted = 0;
        auto weight_of = [&](uint32_t order) __attribute__((always_inline)) { // (nothing below the floor: an infinite largest logit's is itself)
            const float v = logit_of16<DT>(order);
            return v >= r.floor ? r.mass_of_least(v) : uint64_t(0);
        };
        auto masses_of = [&](uint32_t last, uint32_t ties) __attribute__((always_inline)) {
            return [&r, last, ties](uint32_t order, uint32_t count) __attribute__((always_inline)) {
                const uint32_t c = order < last ? count : order == last ? min(count, ties) : 0u;
                const float v = logit_of16<DT>(order);
                return c && v >= r.floor ? c * r.mass(v) : uint64_t(0);
            };
        };
        if (k) {
            sum_blocks([&](uint32_t c0, uint32_t c1, uint32_t, uint64_t &first, uint64_t &second) __attribute__((always_inline)) {
                first = c0;
                second = c1;
                counted += c0 + c1;
            });
        } else if (p < 1.0f) { // (what the blocks weigh, at once)
            sum_blocks([&, mass_of = masses_of(~0u, 0)](uint32_t c0, uint32_t c1, uint32_t order, uint64_t &first, uint64_t &second) __attribute__((always_inline)) {
                first = mass_of(order, c0);
                second = mass_of(order + 32768, c1);
                counted += c0 + c1;
            });
        }
        if (sum_of_all(sh, uint64_t(drawn) - counted) == 0) { // (a count that overflowed takes 65535 or 65536 from the sum)
            // the first value of `block` at which the running sum exceeds `than`, and the sum in front of it
            auto find_value = [&](int block, uint64_t front, uint64_t than, uint64_t own, uint64_t &in_front) __attribute__((always_inline)) {
                const uint64_t upto = front + wave_upto64(own);
                const int first = __builtin_ctzll(__ballot(upto > than) | uint64_t(1) << 63);
                in_front = lane_of(upto - own, first);
                return static_cast<uint32_t>(block * BLOCK + first);
            };
            const uint32_t first = order_of16(DT == AXHIP_DTYPE_BF16 ? f32_to_bf16_bits(top) : f32_to_f16_bits(top)); // the largest's
            uint64_t front, in_front;
            const uint32_t lowest = order_of16(DT == AXHIP_DTYPE_BF16 ? f32_to_bf16_bits(r.floor) : f32_to_f16_bits(r.floor)) + 1; // (the floor, rounded)
            uint32_t last = min(lowest, FIRST_ORDER<DT> + DRAWN_ORDERS<DT> - 1), ties = ~0u; // kept: orders up to `last`, and of that one so many, by index
            if (k) {
                const uint64_t than = static_cast<uint64_t>(k - 1);
                const int block = find_bin(sh, 0, than, front);
                if (block >= 0) {
                    last = find_value(block, front, than, count_at(block * BLOCK + lane), in_front);
                    ties = static_cast<uint32_t>(than - in_front) + 1;
                }
            }
            if (p < 1.0f) {
                const auto kept_mass = masses_of(last, ties);
                if (k) {
                    clear_bins(sh);
                    sum_blocks([&](uint32_t c0, uint32_t c1, uint32_t order, uint64_t &first, uint64_t &second) __attribute__((always_inline)) {
                        first = kept_mass(order, c0);
                        second = kept_mass(order + 32768, c1);
                    });
                    __syncthreads();
                }
                const uint64_t than = than_of_p([&] { return sum_of_bins(sh); });
                const int block = find_bin(sh, 0, than, front);
                if (block >= 0) {
                    if (wave == 0) { // (operations of 64 bits, for all wavefronts)
                        const uint32_t order = block * BLOCK + lane;
                        last = find_value(block, front, than, kept_mass(order, count_at(order)), in_front);
                        const uint64_t each_of_them = r.mass(logit_of16<DT>(last)), reached = than - in_front;
                        ties = static_cast<uint32_t>(static_cast<double>(reached) / static_cast<double>(each_of_them)); // (to within one)
                        if (ties * each_of_them > reached) --ties;
                        else if ((ties + 1) * each_of_them <= reached) ++ties;
                        ++ties;
                        if (lane == 0) sh.other_scratch[0] = uint64_t(ties) << 32 | last;
                    }
                    __syncthreads();
                    last = static_cast<uint32_t>(sh.other_scratch[0]);
                    ties = static_cast<uint32_t>(sh.other_scratch[0] >> 32);
                }
            }
            // Of the last value only the first `ties` by index are kept: its logits carry no weight but a mark, and their share is added when the steps' numbers of
            // marks are known.
            const uint64_t of_last = filtered && ties < count_at(last) ? weight_of(last) : 0;
            const bool in_part = of_last != 0; // (those that weigh nothing need no marks)
            const uint32_t values = last - first + 1;
            __syncthreads(); // (the counts make room for the weights)
            // (weights of logits between two small ones of either sign are the same to an eighth of an integer, and are taken as one: one entry of the table for all of them, which lets it
            // reach negative bfloat16 logits)
            uint32_t zone = values, gap = 0; // entries zone .. zone + gap are one
            if (DT == AXHIP_DTYPE_BF16 && values >= LIST) {
                const uint32_t small = order_of16(f32_to_bf16_bits(temperature * 7.105427357601002e-15f)); // 2^-47 temperatures
                const uint32_t end = 0xFFFEu - small;                                                                       // ... and as much below zero
                if (small > first && end < last) {
                    zone = small - first;
                    gap = end - small;
                }
            }
            const uint32_t entries = values - gap;
            // of two logits, `values` where they are not kept (orders in front of the first, of NaNs, come out beyond it)
            auto place_of = [&](uint32_t w) __attribute__((always_inline)) {
                return __builtin_elementwise_min(orders_of(w) - static_cast<uint16_t>(first), pair_t{static_cast<uint16_t>(values), static_cast<uint16_t>(values)});
            };
            if (entries < LIST) {
                for (uint32_t i = t; i <= entries; i += THREADS)
                    sh.weights[i] = i == entries ? 0 : in_part && i == entries - 1 ? MARK : weight_of(first + (i > zone ? i + gap : i));
                if (gap == 0) {
                    draw_by_steps(std::true_type{}, of_last, ties, [&](const Step<DT> &s, uint32_t, uint64_t(&x)[E]) __attribute__((always_inline)) { // (a barrier in front of the loop)
#pragma unroll
                        for (int e = 0; e < E; ++e) x[e] = sh.weights[place_of(s.v[0][e / 2])[e % 2]];
                    });
                } else {
                    draw_by_steps(std::true_type{}, of_last, ties, [&](const Step<DT> &s, uint32_t, uint64_t(&x)[E]) __attribute__((always_inline)) {
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const uint32_t i = place_of(s.v[0][e / 2])[e % 2];
                            x[e] = sh.weights[i <= zone ? i : i - min(i - zone, gap)];
                        }
                    });
                }
            } else {
                draw_by_steps(std::false_type{}, of_last, ties, [&](const Step<DT> &s, uint32_t, uint64_t(&x)[E]) __attribute__((always_inline)) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t i = place_of(s.v[0][e / 2])[e % 2];
                        const float v = element<DT>(s, e);
                        const bool marked = in_part && i == values - 1;
                        x[e] = r.formed(r.mass_of_least(v, v >= r.floor && i < values && !marked));
                        if (marked) x[e] = MARK;
                    }
                });
            }
            return;
        }
        __syncthreads(); // (the list takes the counts' place)
    }

    // ================ other fp32 rows, and 16-bit ones with more than 65535 equal logits
    // Keeps what is kept up to where the running sum of value(logit, power) exceeds than(sum of all).
    auto cut = [&](auto value, auto than_of) __attribute__((always_inline)) {
        auto value_of = [&](float v) __attribute__((always_inline)) { return value(r.power(v)); };
        clear_bins(sh);
        each_step_of_memory([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
            uint64_t x[E];
            uint32_t bins[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const double z = r.power(element<DT>(s, e));
                x[e] = r.formed(value(z));
                bins[e] = r.bin_of_power(z);
                asm("" : "+v"(bins[e]));
            }
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (r.counts(element<DT>(s, e), at + e)) add_to_bin(sh.bins[bins[e]], x[e]);
        });
        __syncthreads();
        const uint64_t than = than_of([&] { return sum_of_bins(sh); });
        uint64_t before;
        const int bin = find_bin(sh, 0, than, before);
        if (bin < 0 || bin == BINS - 1) return; // (all are kept, or all that weigh anything)
        // where the bins up to this one end, and those in front of it: two comparisons for each logit instead of its bin
        if (wave < 2) {
            const float edge = r.smallest_up_to(bin - wave, r.floor);
            if (lane == 0) sh.top[wave] = edge;
        }
        __syncthreads();
        const float inside_from = sh.top[0], front_from = bin ? sh.top[1] : __builtin_nanf("");
        auto inside = [&](float v, uint32_t i) __attribute__((always_inline)) { return v >= inside_from && !(v >= front_from) && r.counts(v, i); };
        const int n = gather(inside);
        const uint64_t first = order_of(r.top, 0), behind = r.last < (uint64_t(1) << 52) ? r.last : (uint64_t(1) << 52) - 1;
        auto known = [&](auto) { return than; };
        if (n <= LIST) {
            r.keep_up_to(find_place(sh, first, behind, before, n, known, [&](auto f) __attribute__((always_inline)) {
                for (int i = t; i < n; i += THREADS) {
                    const uint64_t o = sh.list[i];
                    f(o, [&] { return value_of(logit_of(o)); });
                }
            }));
        } else {
            r.keep_up_to(find_place(sh, first, behind, before, n, known, [&](auto f) __attribute__((always_inline)) {
                each_of(each_step_of_memory, [&](float v, uint32_t i) {
                    if (inside(v, i)) f(order_of(v, i), [&] { return value_of(v); });
                });
            }));
        }
    };
    if (k) cut([](double) { return uint64_t(1); }, [&](auto) { return static_cast<uint64_t>(k - 1); });
    if (p < 1.0f) cut([&](double z) { return r.integer(r.scaled_weight(z)); }, than_of_p);

    draw_by_steps(std::false_type{}, 0, 0, [&](const Step<DT> &s, uint32_t at, uint64_t(&x)[E]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = element<DT>(s, e);
            x[e] = r.formed(r.mass_of_least(v, r.counts(v, at + e)));
        }
    });
}

template <int DT, int IT> int launch(const SampleArgs &a, int64_t rows, hipStream_t s) {
    const auto kernel = sample_kernel<DT, IT>;
    static const hipError_t configured = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(SampleShared));
    AXHIP_CHECK_HIP(configured);
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(rows)), dim3(THREADS), sizeof(SampleShared), s, a);
    return AXHIP_OK;
}
// Registers for a row: 64 of a thread's 128 (65536 fp32 or 131072 16-bit logits).
template <int DT> int launch(const SampleArgs &a, int64_t rows, hipStream_t s) {
    const int held = (a.vocab + STEP * WAVES - 1) / (STEP * WAVES);
    if (held <= 2) return launch<DT, 2>(a, rows, s);
    if (held <= 4) return launch<DT, 4>(a, rows, s);
    if (held <= 8) return launch<DT, 8>(a, rows, s);
    if constexpr (DT != AXHIP_DTYPE_F32)
        if (held <= 16) return launch<DT, 16>(a, rows, s);
    return launch<DT, 0>(a, rows, s);
}

} // namespace
} // namespace axhip
