// A token from each row of logits: axhip_sample.
#include "common.hpp"

namespace axhip {
namespace {

struct SampleArgs {
    const void *logits;
    int64_t *tokens;
    float *probs;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    int64_t ld;
    int vocab;
};

// A work-group of 1024 threads to a row.  No sorting: a filter keeps a prefix of the order "larger logit first, equal ones by index", and where it ends is found by
// histograms of what lies in front (numbers of logits, or sums of weights).  The draw is the same search in the order of the indexes.
//   * Weights are integers, multiples of 2^-43 of the largest, of which 2^20 fit 64 bits: sums do not depend on the order in which atomics arrive.
//   * 16-bit logits: all 65535 values are counted in LDS (128 KiB), in the pass that finds the largest, and every filter is answered by the counts: one weight for
//     each value that occurs instead of one for each logit.  The draw takes weights from a table of the values that are kept.  Counts are 16 bits wide; if one
//     overflows, the sum of all shows it and the row goes the other way.
//   * fp32 logits: the histogram's bins are linear in the logit, from the largest to 31 temperatures below it, from where on weights round to zero (bins by the bits of
//     the float hold most logits in a few dozen bins, on which a wavefront's atomics wait for each other).  All logits in the bin in which a filter ends, or in front
//     of it, go to a list in LDS if they fit, and everything after happens there: a row is read three times (its maximum, the histogram, the list).
constexpr int THREADS = 1024, WAVES = THREADS / WAVE, E = 8; // elements of a lane's vector
constexpr int STEP = WAVE * E;                               // consecutive elements of a wavefront's step
constexpr int BINS = 2048, FEW = 128;
constexpr int LIST = 16384, FRONT = 12288; // of which this many for what lies in front of the bin
constexpr int BLOCK = 64, BLOCKS = 65536 / BLOCK; // 16-bit values are summed up by blocks
constexpr int64_t MOST_VOCAB = 1 << 20; // BINS steps
constexpr uint64_t ONE = uint64_t(1) << 43;
constexpr float REACH = 31.0f; // temperatures: exp(-31) is below half of 2^-43

struct SampleShared {
    uint64_t bins[BINS];
    uint64_t block_mass[BLOCKS];
    uint32_t block_count[BLOCKS];
    uint64_t few_place[FEW], few_value[FEW];
    uint64_t scratch[WAVES + 2], other_scratch[WAVES];
    float top[WAVES];
    uint32_t where[WAVES], few, front, inside;
    union {
        uint64_t list[LIST];
        uint32_t counts[32768]; // two values to a word
        uint64_t weights[LIST];
        uint32_t ties[32768];
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
__device__ __forceinline__ uint32_t orders_of_pair(uint32_t w) {
    const uint32_t sign = (w >> 15) & 0x00010001u;
    return (w ^ 0x7FFF7FFFu ^ ((sign << 15) - sign)) - sign;
}
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
    float top;             // the largest logit
    double rate;           // log2(e) / temperature
    float bin_rate;        // bins per unit of the logit
    uint64_t last = ~0ull; // kept: up to this one in the order,
    double least = 0.0;    // and with at least this weight

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
    // f(vectors, index of the first, step) for the wavefront's steps, the next ones' loads in flight
    template <class F> __device__ __forceinline__ void each_step(F f) const {
        const int n = steps(), first = threadIdx.x / WAVE;
        if (first >= n) return;
        Step<DT> next = load(first);
#pragma unroll 1
        for (int step = first; step < n; step += WAVES) {
            const Step<DT> s = next;
            if (step + WAVES < n) next = load(step + WAVES);
            f(s, static_cast<uint32_t>(step * STEP) + threadIdx.x % WAVE * E, step);
        }
    }
    template <class F> __device__ __forceinline__ void each(F f) const { // f(logit, index)
        each_step([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < E; ++e) f(element<DT>(s, e), at + e);
        });
    }

    // exp((v - top) / temperature) in multiples of 2^-43: 2^z with z = i + r, |r| <= 1/2, by a polynomial through the Chebyshev points of 2^r, off by less than 5e-15 of the weight (2^-53 takes a
    // degree more; a table of 2^(i / 256) and four terms waited longer for LDS than the six terms more take).
    __device__ __forceinline__ double scaled_weight(float v) const {
        constexpr double SPLIT = 6755399441055744.0; // 1.5 * 2^52: its last bit is 1
        double z = (static_cast<double>(v) - static_cast<double>(top)) * rate;
        z = fmax(z, -64.0); // (NaN, of an infinity against an infinite temperature or a finite logit, too)
        const double t = z + SPLIT, r = z - (t - SPLIT);
        const uint32_t i = static_cast<uint32_t>(__double_as_longlong(t));
        double p = 6.422412339320131e-09;
        p = __builtin_fma(r, p, 1.02053706737851e-07);
        p = __builtin_fma(r, p, 1.3219110032865315e-06);
        p = __builtin_fma(r, p, 1.5252674086943783e-05);
        p = __builtin_fma(r, p, 0.00015403523472909156);
        p = __builtin_fma(r, p, 0.0013333558203519715);
        p = __builtin_fma(r, p, 0.00961812911264106);
        p = __builtin_fma(r, p, 0.05550410866458426);
        p = __builtin_fma(r, p, 0.2402265069589931);
        p = __builtin_fma(r, p, 0.6931471805599488);
        p = __builtin_fma(r, p, 1.0);
        return __longlong_as_double(__double_as_longlong(p) + (static_cast<long long>(static_cast<uint64_t>(i + 43u) << 52)));
    }
    __device__ __forceinline__ uint64_t mass(float v) const {
        if (v == top) return ONE;
        constexpr double TO_INTEGER = 4503599627370496.0; // 2^52: the integer is what its last bits say
        const double w = scaled_weight(v);
        return w >= least ? static_cast<uint64_t>(__double_as_longlong(w + TO_INTEGER)) & ((uint64_t(1) << 52) - 1) : 0;
    }
    __device__ __forceinline__ uint32_t bin_of(float v) const {
        return static_cast<uint32_t>(fminf(fmaxf((top - v) * bin_rate, 0.0f), static_cast<float>(BINS - 1))); // (inf - inf, NaN: bin 0)
    }
    __device__ __forceinline__ bool counts(float v, uint32_t i) const { return v > -__builtin_inff() && (last == ~0ull || order_of(v, i) <= last); }
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
                    const uint32_t at = atomicAdd(&sh.few, 1u);
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

template <int DT> __global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char sample_lds[];
    SampleShared &sh = *reinterpret_cast<SampleShared *>(sample_lds);
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
    const int64_t row = blockIdx.x;
    constexpr int64_t ES = DT == AXHIP_DTYPE_F32 ? 4 : 2;
    Row<DT> r{static_cast<const char *>(a.logits) + row * a.ld * ES, a.vocab, 0.0f, 0.0, 0.0f, ~0ull, 0.0};
    const float temperature = a.temperature ? a.temperature[row] : 1.0f, p = a.top_p ? a.top_p[row] : 1.0f, m = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
    const int32_t k = a.top_k && a.top_k[row] > 0 && a.top_k[row] < a.vocab ? a.top_k[row] : 0;
    if (t == 0) sh.front = sh.inside = 0;

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
    auto nothing_or_first = [&](bool nothing, auto is_top) __attribute__((always_inline)) {
        uint32_t first = ~0u;
        if (!nothing) r.each([&](float v, uint32_t i) { first = is_top(v) ? min(first, i) : first; });
#pragma unroll
        for (int d = 32; d; d /= 2) first = min(first, static_cast<uint32_t>(__shfl_xor(first, d, WAVE)));
        if (lane == 0) sh.where[wave] = first;
        __syncthreads();
        for (int w = 0; w < WAVES; ++w) first = min(first, sh.where[w]);
        if (t == 0) {
            a.tokens[row] = first == ~0u ? -1 : static_cast<int64_t>(first);
            if (a.probs) a.probs[row] = first == ~0u ? 0.0f : 1.0f;
        }
    };
    auto set_temperature = [&]() __attribute__((always_inline)) {
        r.rate = 1.4426950408889634 / static_cast<double>(temperature);
        r.bin_rate = static_cast<float>(BINS - 1) / (REACH * temperature);
        if (m > 0.0f) r.least = (m < 1.0f ? static_cast<double>(m) : 1.0) * static_cast<double>(ONE);
    };
    // The draw by the sums of the wavefronts' steps, and then within one.  masses(vectors, index of the first, sums): of a lane's eight.
    auto draw_by_steps = [&](auto masses) __attribute__((always_inline)) {
        clear_bins(sh);
        r.each_step([&](const Step<DT> &s, uint32_t at, int step) __attribute__((always_inline)) {
            uint64_t x[E], sum = 0;
            masses(s, at, x);
#pragma unroll
            for (int e = 0; e < E; ++e) sum += x[e];
            sum = wave_sum64(sum);
            if (lane == 0) sh.bins[step] = sum;
        });
        __syncthreads();
        const uint64_t total = sum_of_bins(sh), than = than_of_u(total);
        uint64_t front;
        const int step = find_bin(sh, 0, than, front);
        if (wave == 0) {
            const uint32_t at = static_cast<uint32_t>(step * STEP + lane * E);
            uint64_t x[E], mine = 0;
            masses(r.load(step), at, x);
#pragma unroll
            for (int e = 0; e < E; ++e) mine += x[e];
            const uint64_t upto = front + wave_upto64(mine);
            front = upto - mine;
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
    if constexpr (DT != AXHIP_DTYPE_F32) {
        auto count_at = [&](uint32_t order) { return (sh.counts[order >> 1] >> (16 * (order & 1))) & 0xFFFFu; };
        for (int i = t; i < 8192; i += THREADS) reinterpret_cast<uint4_t *>(sh.counts)[i] = uint4_t{0, 0, 0, 0};
        __syncthreads();
        uint32_t drawn = 0;
        r.each_step([&](const Step<DT> &s, uint32_t, int) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t pair = orders_of_pair(s.v[0][i]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t order = h ? pair >> 16 : pair & 0xFFFFu;
                    if (order - FIRST_ORDER<DT> < DRAWN_ORDERS<DT>) {
                        ++drawn;
                        atomicAdd(&sh.counts[order >> 1], 1u << (16 * (order & 1)));
                    }
                }
            }
        });
        drawn = static_cast<uint32_t>(sum_of_all(sh, drawn)); // (a barrier behind the counts)
        // sums of blocks of 64 values, 128 values to a wavefront at a time
        auto each_block_pair = [&](auto f) __attribute__((always_inline)) { // f(block, count of value 2 l, of value 2 l + 1, the first's order): by the lanes of a half
            for (int j = wave; j < BLOCKS / 2; j += WAVES) {
                const uint32_t w = sh.counts[64 * j + lane];
                f(2 * j + lane / 32, w & 0xFFFFu, w >> 16, static_cast<uint32_t>(128 * j + 2 * lane), __ballot(w != 0) != 0);
            }
        };
        each_block_pair([&](int block, uint32_t c0, uint32_t c1, uint32_t, bool any) __attribute__((always_inline)) {
            const uint32_t sum = any ? static_cast<uint32_t>(sum32(c0 + c1)) : 0;
            if (lane % 32 == 0) {
                sh.block_count[block] = sum;
                sh.bins[block] = sum;
                sh.bins[BLOCKS + block] = 0;
            }
        });
        __syncthreads();
        const uint64_t counted = sum_of_bins(sh);
        if (drawn == 0) return nothing_or_first(true, [](float) { return false; });
        if (counted == drawn) { // (a count that overflowed takes 65535 or 65536 from the sum)
            static_assert(BLOCK == WAVE && 2 * BLOCKS == BINS, "a value to a lane, and bins for counts with as many zeros");
            // the first value of `block` at which the running sum exceeds `than`, and the sum in front of it
            auto find_value = [&](int block, uint64_t front, uint64_t than, uint64_t mine, uint64_t &in_front) __attribute__((always_inline)) {
                const uint64_t upto = front + wave_upto64(mine);
                const int first = __builtin_ctzll(__ballot(upto > than) | uint64_t(1) << 63);
                in_front = lane_of(upto - mine, first);
                return static_cast<uint32_t>(block * BLOCK + first);
            };
            uint64_t front, in_front;
            int block = find_bin(sh, 0, 0, front);
            const uint32_t first = find_value(block, front, 0, count_at(block * BLOCK + lane), in_front);
            r.top = logit_of16<DT>(first);
            if (!(temperature > 0.0f)) return nothing_or_first(false, [&](float v) { return v == r.top; });
            set_temperature();
            uint32_t last = FIRST_ORDER<DT> + DRAWN_ORDERS<DT> - 1, ties = ~0u; // kept: orders up to `last`, and of that one so many, by index
            if (k) {
                const uint64_t than = static_cast<uint64_t>(k - 1);
                block = find_bin(sh, 0, than, front);
                if (block >= 0) {
                    last = find_value(block, front, than, count_at(block * BLOCK + lane), in_front);
                    ties = static_cast<uint32_t>(than - in_front) + 1;
                }
            }
            if (p < 1.0f) {
                auto kept_count = [&](uint32_t order) __attribute__((always_inline)) { return order < last ? count_at(order) : order == last ? min(count_at(order), ties) : 0u; };
                auto kept_mass = [&](uint32_t order) __attribute__((always_inline)) {
                    const uint32_t c = kept_count(order);
                    return c ? c * r.mass(logit_of16<DT>(order)) : uint64_t(0);
                };
                const double least = r.least;
                r.least = 0.0; // (top_p's sum is taken before min_p)
                each_block_pair([&](int b, uint32_t, uint32_t, uint32_t order, bool any) __attribute__((always_inline)) {
                    const uint64_t sum = any ? sum32(kept_mass(order) + kept_mass(order + 1)) : 0;
                    if (lane % 32 == 0) sh.bins[b] = sum;
                });
                __syncthreads();
                const uint64_t than = than_of_p([&] { return sum_of_bins(sh); });
                block = find_bin(sh, 0, than, front);
                if (block >= 0) {
                    const uint32_t order = block * BLOCK + lane;
                    last = find_value(block, front, than, kept_mass(order), in_front);
                    ties = static_cast<uint32_t>((than - in_front) / r.mass(logit_of16<DT>(last))) + 1;
                }
                r.least = least;
            }
            uint32_t last_index = ~0u; // of order `last`
            const uint32_t equal = count_at(last);
            const bool in_part = ties < equal;
            __syncthreads(); // (the counts make room for the indexes of the last value, then for the weights)
            if (in_part) {
                r.each_step([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t pair = orders_of_pair(s.v[0][i]);
                        if ((pair & 0xFFFFu) == last) {
                            const uint32_t n = atomicAdd(&sh.inside, 1u);
                            if (n < 32768) sh.ties[n] = at + 2 * i;
                        }
                        if (pair >> 16 == last) {
                            const uint32_t n = atomicAdd(&sh.inside, 1u);
                            if (n < 32768) sh.ties[n] = at + 2 * i + 1;
                        }
                    }
                });
                __syncthreads();
                const int n = static_cast<int>(sh.inside);
                auto one = [] { return uint64_t(1); };
                auto than = [&](auto) { return static_cast<uint64_t>(ties - 1); };
                if (n <= 32768) {
                    last_index = static_cast<uint32_t>(find_place(sh, 0, static_cast<uint64_t>(a.vocab - 1), 0, n, than, [&](auto f) __attribute__((always_inline)) {
                        for (int i = t; i < n; i += THREADS) f(sh.ties[i], one);
                    }));
                } else {
                    const float v0 = logit_of16<DT>(last);
                    last_index = static_cast<uint32_t>(find_place(sh, 0, static_cast<uint64_t>(a.vocab - 1), 0, n, than, [&](auto f) __attribute__((always_inline)) {
                        r.each([&](float v, uint32_t i) {
                            if (v == v0) f(i, one);
                        });
                    }));
                }
                __syncthreads();
            }
            const uint32_t values = last - first + 1;
            if (values <= LIST) {
                for (uint32_t i = t; i < values; i += THREADS) sh.weights[i] = r.mass(logit_of16<DT>(first + i));
                draw_by_steps([&](const Step<DT> &s, uint32_t at, uint64_t(&x)[E]) __attribute__((always_inline)) { // (a barrier in front of the loop)
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t pair = orders_of_pair(s.v[0][e / 2]), i = (e % 2 ? pair >> 16 : pair & 0xFFFFu) - first;
                        x[e] = i < values ? sh.weights[i] : 0;
                        if (in_part && i == values - 1 && at + e > last_index) x[e] = 0;
                    }
                });
            } else {
                draw_by_steps([&](const Step<DT> &s, uint32_t at, uint64_t(&x)[E]) __attribute__((always_inline)) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const uint32_t pair = orders_of_pair(s.v[0][e / 2]), i = (e % 2 ? pair >> 16 : pair & 0xFFFFu) - first;
                        x[e] = i < values && !(in_part && i == values - 1 && at + e > last_index) ? r.mass(element<DT>(s, e)) : 0;
                    }
                });
            }
            return;
        }
        __syncthreads(); // (the list takes the counts' place)
    }

    // ================ fp32 logits, and 16-bit rows with more than 65535 equal ones
    float top = -__builtin_inff();
    r.each([&](float v, uint32_t) { top = fmaxf(top, v); });
    top = wave_max(top);
    if (lane == 0) sh.top[wave] = top;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sh.top[w]);
    r.top = top;
    if (top == -__builtin_inff() || !(temperature > 0.0f)) return nothing_or_first(top == -__builtin_inff(), [&](float v) { return v == top; });
    set_temperature();
    const double least = r.least;
    r.least = 0.0;

    // `listed`: the list holds all that is kept: `front` in front of the bin in which the filter ended, `inside` of it.
    bool listed = false;
    int front = 0, inside = 0;
    auto each_listed = [&](auto f) __attribute__((always_inline)) {
        for (int i = t; i < front + inside; i += THREADS) f(sh.list[i < front ? i : FRONT + i - front]);
    };
    // Keeps what is kept up to where the running sum of value(logit) exceeds than(sum of all).
    auto cut = [&](auto value, auto than_of) __attribute__((always_inline)) {
        if (listed) {
            r.last = find_place(sh, order_of(r.top, 0), r.last, 0, front + inside, than_of, [&](auto f) __attribute__((always_inline)) { each_listed([&](uint64_t o) { f(o, [&] { return value(logit_of(o)); }); }); });
            return;
        }
        clear_bins(sh);
        r.each([&](float v, uint32_t i) {
            if (r.counts(v, i)) {
                const uint64_t x = value(v);
                if (x) add_to_bin(sh.bins[r.bin_of(v)], x);
            }
        });
        __syncthreads();
        const uint64_t than = than_of([&] { return sum_of_bins(sh); });
        uint64_t before;
        const int bin = find_bin(sh, 0, than, before);
        if (bin < 0 || bin == BINS - 1) return; // (all are kept, or all that weigh anything)
        const float lowest = r.top - static_cast<float>(bin + 2) / r.bin_rate; // (below every logit of the bin; -inf or NaN where that cannot be said)
        const bool quick = lowest > -3e38f;
        r.each_step([&](const Step<DT> &s, uint32_t at, int) __attribute__((always_inline)) {
            // what the lane has of either kind, one addition for the wavefront, and places by what the lanes in front have
            uint32_t kinds = 0; // two bits an element: 1 in front, 2 inside
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float v = element<DT>(s, e);
                if (quick ? v >= lowest : true) {
                    const uint32_t b = r.bin_of(v);
                    if (b <= static_cast<uint32_t>(bin) && r.counts(v, at + e)) kinds |= (b == static_cast<uint32_t>(bin) ? 2u : 1u) << (2 * e);
                }
            }
            if (__ballot(kinds != 0) == 0) return;
            const uint32_t mine = __builtin_popcount(kinds & 0x5555u) | static_cast<uint32_t>(__builtin_popcount(kinds & 0xAAAAu)) << 16;
            const uint32_t upto = static_cast<uint32_t>(wave_upto64(mine)), all = __builtin_amdgcn_readlane(upto, WAVE - 1);
            uint32_t f0 = 0, i0 = 0;
            if (lane == 0) {
                f0 = atomicAdd(&sh.front, all & 0xFFFFu);
                i0 = atomicAdd(&sh.inside, all >> 16);
            }
            uint32_t f = __builtin_amdgcn_readfirstlane(f0) + ((upto - mine) & 0xFFFFu), i = __builtin_amdgcn_readfirstlane(i0) + ((upto - mine) >> 16);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t kind = (kinds >> (2 * e)) & 3u;
                if (kind == 1 && f++ < FRONT) sh.list[f - 1] = order_of(element<DT>(s, e), at + e);
                if (kind == 2 && i++ < LIST - FRONT) sh.list[FRONT + i - 1] = order_of(element<DT>(s, e), at + e);
            }
        });
        __syncthreads();
        front = static_cast<int>(sh.front);
        inside = static_cast<int>(sh.inside);
        __syncthreads();
        if (t == 0) sh.front = sh.inside = 0;
        listed = front <= FRONT && inside <= LIST - FRONT;
        const uint64_t first = order_of(r.top, 0), behind = r.last < (uint64_t(1) << 52) ? r.last : (uint64_t(1) << 52) - 1;
        auto known = [&](auto) { return than; };
        if (inside <= LIST - FRONT) {
            const int n = inside;
            r.last = find_place(sh, first, behind, before, n, known, [&](auto f) __attribute__((always_inline)) {
                for (int i = t; i < n; i += THREADS) {
                    const uint64_t o = sh.list[FRONT + i];
                    f(o, [&] { return value(logit_of(o)); });
                }
            });
        } else {
            r.last = find_place(sh, first, behind, before, inside, known, [&](auto f) __attribute__((always_inline)) {
                r.each([&](float v, uint32_t i) {
                    if (v > -__builtin_inff() && r.bin_of(v) == static_cast<uint32_t>(bin)) f(order_of(v, i), [&] { return value(v); });
                });
            });
        }
    };
    if (k) cut([](float) { return uint64_t(1); }, [&](auto) { return static_cast<uint64_t>(k - 1); });
    if (p < 1.0f) cut([&](float v) { return r.mass(v); }, than_of_p);
    r.least = least;

    if (listed) {
        uint64_t total = 0;
        const uint64_t at = find_place(sh, 0, static_cast<uint64_t>(a.vocab), 0, front + inside, [&](auto sum) { return than_of_u(total = sum()); }, [&](auto f) __attribute__((always_inline)) {
            each_listed([&](uint64_t o) { f(index_of(o), [&] { return o <= r.last ? r.mass(logit_of(o)) : uint64_t(0); }); });
        });
        each_listed([&](uint64_t o) {
            if (index_of(o) == at && o <= r.last) answer(static_cast<uint32_t>(at), r.mass(logit_of(o)), total);
        });
        return;
    }
    draw_by_steps([&](const Step<DT> &s, uint32_t at, uint64_t(&x)[E]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = element<DT>(s, e);
            x[e] = r.counts(v, at + e) ? r.mass(v) : 0;
        }
    });
}

template <int DT> int launch(const SampleArgs &a, int64_t rows, hipStream_t s) {
    static const hipError_t configured = hipFuncSetAttribute(reinterpret_cast<const void *>(&sample_kernel<DT>), hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(SampleShared));
    AXHIP_CHECK_HIP(configured);
    hipLaunchKernelGGL(sample_kernel<DT>, dim3(static_cast<unsigned>(rows)), dim3(THREADS), sizeof(SampleShared), s, a);
    return AXHIP_OK;
}

int sample(const void *logits, int64_t *tokens, float *probs, const AxhipSampleParams *params, void *, size_t, void *stream) {
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_sample: params is NULL");
    const AxhipSampleParams &p = *params;
    AXHIP_REQUIRE(valid_dtype(p.dtype), AXHIP_ERR_INVALID_ARG, "axhip_sample: bad dtype %d", p.dtype);
    AXHIP_REQUIRE(p.rows >= 0 && p.rows < (int64_t(1) << 22), AXHIP_ERR_INVALID_ARG, "axhip_sample: bad number of rows");
    AXHIP_REQUIRE(p.vocab > 0, AXHIP_ERR_INVALID_ARG, "axhip_sample: an empty vocabulary");
    AXHIP_REQUIRE(p.vocab <= MOST_VOCAB, AXHIP_ERR_UNSUPPORTED, "axhip_sample: a vocabulary of %lld (up to %lld)", static_cast<long long>(p.vocab), static_cast<long long>(MOST_VOCAB));
    AXHIP_REQUIRE(p.ld >= p.vocab && p.ld < (int64_t(1) << 40), AXHIP_ERR_INVALID_ARG, "axhip_sample: bad leading dimension");
    if (p.rows == 0) return AXHIP_OK;
    AXHIP_REQUIRE(logits && tokens && p.u, AXHIP_ERR_INVALID_ARG, "axhip_sample: NULL buffer");
    AXHIP_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype_size(p.dtype) - 1)) == 0 && (reinterpret_cast<uintptr_t>(tokens) & 7u) == 0 &&
                      ((reinterpret_cast<uintptr_t>(probs) | reinterpret_cast<uintptr_t>(p.temperature) | reinterpret_cast<uintptr_t>(p.top_k) | reinterpret_cast<uintptr_t>(p.top_p) |
                        reinterpret_cast<uintptr_t>(p.min_p) | reinterpret_cast<uintptr_t>(p.u)) & 3u) == 0,
                  AXHIP_ERR_INVALID_ARG, "axhip_sample: a buffer is not aligned to its elements");
    int rc = ensure_init();
    if (rc) return rc;
    hipStream_t s = resolve_stream(stream);
    const SampleArgs a{logits, tokens, probs, p.temperature, p.top_k, p.top_p, p.min_p, p.u, p.ld, static_cast<int>(p.vocab)};
    rc = p.dtype == AXHIP_DTYPE_F32 ? launch<AXHIP_DTYPE_F32>(a, p.rows, s) : p.dtype == AXHIP_DTYPE_F16 ? launch<AXHIP_DTYPE_F16>(a, p.rows, s) : launch<AXHIP_DTYPE_BF16>(a, p.rows, s);
    if (rc) return rc;
    AXHIP_CHECK_HIP(hipGetLastError());
    return AXHIP_OK;
}
} // namespace
} // namespace axhip
using namespace axhip;

extern "C" size_t axhip_sample_workspace_bytes(const AxhipSampleParams *) { return 0; }
extern "C" int axhip_sample(const void *logits, int64_t *tokens, float *probs, const AxhipSampleParams *params, void *stream) {
    return sample(logits, tokens, probs, params, nullptr, 0, stream);
}
extern "C" int axhip_sample_ws(const void *logits, int64_t *tokens, float *probs, const AxhipSampleParams *params, void *workspace, size_t workspace_bytes, void *stream) {
    return sample(logits, tokens, probs, params, workspace, workspace_bytes, stream);
}
