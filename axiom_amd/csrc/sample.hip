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
// a histogram of what lies in front (numbers of logits, or sums of weights), then another one of the bin in which it ends, until one logit is left.  The draw is the
// same search in the order of the indexes.
//   * Weights are integers, multiples of 2^-43 of the largest, of which 2^20 fit 64 bits: sums do not depend on the order in which atomics arrive.
//   * The first histogram's bins are linear in the logit, from the largest to 31 temperatures below it, from where on weights round to
//     zero: bins by the bits of the float hold most logits in a few dozen bins, on which a wavefront's atomics wait for each other.
//   * Once the bin is known, all logits in it or in front of it go to a list in LDS if they fit (LIST of them), and everything after happens there: a row is read three
//     times (its maximum, the histogram, the list), twice more for each further filter and the draw where the list does not hold what is kept.
constexpr int THREADS = 1024, WAVES = THREADS / WAVE, E = 8; // elements of a lane's vector
constexpr int STEP = WAVE * E;                               // consecutive elements of a wavefront's step
constexpr int BINS = 2048, LIST = 16384;
constexpr int64_t MOST_VOCAB = 1 << 20; // BINS steps
constexpr uint64_t ONE = uint64_t(1) << 43;
constexpr float REACH = 31.0f; // temperatures: exp(-31) is below half of 2^-43

struct SampleShared {
    uint64_t bins[BINS];
    double pow2[256]; // 2^(i / 256)
    uint64_t scratch[WAVES + 2], lowest[WAVES], highest[WAVES];
    float top[WAVES];
    uint32_t where[WAVES];
    uint32_t length;
    uint64_t list[LIST];
};

// The order: smaller numbers first.  Larger logits (-0 is +0), and of equal ones smaller indexes.
__device__ __forceinline__ uint64_t order_of(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return static_cast<uint64_t>(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu) << 20 | i;
}
__device__ __forceinline__ float logit_of(uint64_t order) {
    const uint32_t b = static_cast<uint32_t>(order >> 20);
    return __uint_as_float(b & 0x80000000u ? b : ~b & 0x7FFFFFFFu);
}
__device__ __forceinline__ uint32_t index_of(uint64_t order) { return static_cast<uint32_t>(order) & 0xFFFFFu; }

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
    SampleShared &sh;

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
    // f(logit, index) of the wavefront's elements, the next step's loads in flight
    template <class F, class G> __device__ __forceinline__ void each(F f, G behind) const {
        const int n = steps(), first = threadIdx.x / WAVE;
        if (first >= n) return;
        Step<DT> next = load(first);
#pragma unroll 1
        for (int step = first; step < n; step += WAVES) {
            const Step<DT> s = next;
            if (step + WAVES < n) next = load(step + WAVES);
            const uint32_t at = static_cast<uint32_t>(step * STEP) + threadIdx.x % WAVE * E;
#pragma unroll
            for (int e = 0; e < E; ++e) f(element<DT>(s, e), at + e);
            behind(step);
        }
    }
    template <class F> __device__ __forceinline__ void each(F f) const {
        each(f, [](int) {});
    }

    // exp((v - top) / temperature) in multiples of 2^-43.  2^z with z = i / 256 + r, |r| <= 2^-9: 2^(i / 256) from the table, with the power of two put into its
    // exponent, times the four terms of 2^r that 2^-53 leaves.
    __device__ __forceinline__ double scaled_weight(float v) const {
        constexpr double SPLIT = 1.5 * 17592186044416.0; // 1.5 * 2^44: its last bit is 2^-8
        double z = (static_cast<double>(v) - static_cast<double>(top)) * rate;
        z = fmax(z, -64.0); // (NaN, of an infinity against an infinite temperature or a finite logit, too)
        const double t = z + SPLIT, r = z - (t - SPLIT);
        const int i = static_cast<int>(static_cast<uint32_t>(__double_as_longlong(t)));
        const uint64_t power = static_cast<uint64_t>(__double_as_longlong(sh.pow2[i & 255])) + (static_cast<uint64_t>(static_cast<uint32_t>((i >> 8) + 43)) << 52);
        double p = __builtin_fma(r, 0.009618129107628477, 0.055504108664821576);
        p = __builtin_fma(r, p, 0.24022650695910072);
        p = __builtin_fma(r, p, 0.6931471805599453) * r;
        const double w = __longlong_as_double(static_cast<long long>(power));
        return __builtin_fma(w, p, w);
    }
    __device__ __forceinline__ uint64_t mass(float v) const {
        if (v == top) return ONE;
        constexpr double TO_INTEGER = 4503599627370496.0; // 2^52: the integer is what its last bits say
        const double w = scaled_weight(v);
        return w >= least ? static_cast<uint64_t>(__double_as_longlong(w + TO_INTEGER)) & ((uint64_t(1) << 52) - 1) : 0;
    }
    __device__ __forceinline__ uint32_t bin_of(float v) const {
        return static_cast<uint32_t>(fminf(fmaxf((top - v) * bin_rate, 0.0f), static_cast<float>(BINS - 1))); // (inf - inf: bin 0)
    }
    __device__ __forceinline__ bool counts(float v, uint32_t i) const { return v > -__builtin_inff() && order_of(v, i) <= last; }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v += __shfl_xor(v, d, WAVE);
    return v;
}
__device__ __forceinline__ void add_to_bin(uint64_t &bin, uint64_t v) { atomicAdd(reinterpret_cast<unsigned long long *>(&bin), static_cast<unsigned long long>(v)); }

// All of these are called by the whole work-group, and their answers are every thread's.
__device__ __forceinline__ void clear_bins(SampleShared &sh) {
    sh.bins[threadIdx.x] = 0;
    sh.bins[threadIdx.x + THREADS] = 0;
    __syncthreads();
}
// (call after a barrier behind the bins' additions)
__device__ __forceinline__ uint64_t sum_of_bins(SampleShared &sh) {
    const uint64_t v = wave_sum64(sh.bins[threadIdx.x] + sh.bins[threadIdx.x + THREADS]);
    if (threadIdx.x % WAVE == 0) sh.scratch[threadIdx.x / WAVE] = v;
    __syncthreads();
    uint64_t sum = 0;
    for (int w = 0; w < WAVES; ++w) sum += sh.scratch[w];
    __syncthreads();
    return sum;
}
// The first bin at which the running sum, `before` in front, exceeds `than`, and the sum in front of it; -1 if none does.
__device__ __forceinline__ int find_bin(SampleShared &sh, uint64_t before, uint64_t than, uint64_t &in_front) {
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
    const uint64_t v0 = sh.bins[2 * t], v1 = sh.bins[2 * t + 1];
    uint64_t upto = v0 + v1;
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
        const uint64_t other = __shfl_up(upto, d, WAVE);
        if (lane >= d) upto += other;
    }
    if (lane == WAVE - 1) sh.scratch[wave] = upto;
    if (t == 0) sh.scratch[WAVES] = ~0ull;
    __syncthreads();
    uint64_t first = before;
    for (int w = 0; w < wave; ++w) first += sh.scratch[w];
    const uint64_t all = first + upto, mine = all - v0 - v1;
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
        sh.lowest[threadIdx.x / WAVE] = lo;
        sh.highest[threadIdx.x / WAVE] = hi;
    }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) {
        lo = sh.lowest[w] < lo ? sh.lowest[w] : lo;
        hi = sh.highest[w] > hi ? sh.highest[w] : hi;
    }
    __syncthreads();
}

// Of the elements that `all(f)` hands to f(place, value()), those with places in [lo, hi]: the place at which the running sum of values, by place and with `before` in
// front, exceeds `than`.  (It does: the caller has seen the sums.  Places are unique, values may be 0.)
template <class All> __device__ __forceinline__ uint64_t find_place(SampleShared &sh, uint64_t lo, uint64_t hi, uint64_t before, uint64_t than, All all) {
    while (lo < hi) {
        const double rate = (BINS - 0.5) / (static_cast<double>(hi - lo) + 1.0);
        auto bin_of = [&](uint64_t place) { return static_cast<int>(static_cast<double>(place - lo) * rate); };
        clear_bins(sh);
        all([&](uint64_t place, auto value) __attribute__((always_inline)) {
            if (place >= lo && place <= hi) {
                const uint64_t v = value();
                if (v) add_to_bin(sh.bins[bin_of(place)], v);
            }
        });
        __syncthreads();
        const int bin = find_bin(sh, before, than, before);
        uint64_t l = ~0ull, h = 0;
        all([&](uint64_t place, auto value) __attribute__((always_inline)) {
            if (place >= lo && place <= hi && bin_of(place) == bin && value()) {
                l = place < l ? place : l;
                h = place > h ? place : h;
            }
        });
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
    Row<DT> r{static_cast<const char *>(a.logits) + row * a.ld * ES, a.vocab, 0.0f, 0.0, 0.0f, ~0ull, 0.0, sh};
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;

    // ---- the largest logit
    float top = -__builtin_inff();
    r.each([&](float v, uint32_t) { top = fmaxf(top, v); });
    top = wave_max(top);
    if (lane == 0) sh.top[wave] = top;
    if (t < 256) sh.pow2[t] = exp2(t * (1.0 / 256.0));
    if (t == 0) sh.length = 0;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sh.top[w]);
    r.top = top;
    if (top == -__builtin_inff() || !(temperature > 0.0f)) { // (the same in every thread)
        uint32_t first = ~0u;
        if (top != -__builtin_inff()) r.each([&](float v, uint32_t i) { first = v == top ? min(first, i) : first; });
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
    r.rate = 1.4426950408889634 / static_cast<double>(temperature);
    r.bin_rate = static_cast<float>(BINS - 1) / (REACH * temperature);

    // ---- the filters.  `listed`: the list holds all that is kept, and n is its length.
    bool listed = false;
    int n = 0;
    auto each_listed = [&](auto f) __attribute__((always_inline)) {
        for (int i = t; i < n; i += THREADS) f(sh.list[i]);
    };
    // Keeps what is kept up to where the running sum of value(logit) exceeds than(sum of all).
    auto cut = [&](auto value, auto than_of) __attribute__((always_inline)) {
        uint64_t before = 0, lo = ~0ull, hi = 0;
        if (!listed) {
            clear_bins(sh);
            r.each([&](float v, uint32_t i) {
                if (r.counts(v, i)) {
                    const uint64_t x = value(v);
                    if (x) add_to_bin(sh.bins[r.bin_of(v)], x);
                }
            });
            __syncthreads();
            const uint64_t than = than_of(sum_of_bins(sh));
            const int bin = find_bin(sh, 0, than, before);
            if (bin < 0 || bin == BINS - 1) return; // (all are kept, or all that weigh anything)
            r.each([&](float v, uint32_t i) {
                const bool mine = r.counts(v, i) && r.bin_of(v) <= static_cast<uint32_t>(bin);
                const uint64_t mask = __ballot(mine);
                if (mask) {
                    uint32_t at = 0;
                    if (lane == 0) at = atomicAdd(&sh.length, static_cast<uint32_t>(__popcll(mask)));
                    at = __builtin_amdgcn_readfirstlane(at) + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0));
                    if (mine && at < LIST) sh.list[at] = order_of(v, i);
                }
                if (mine && r.bin_of(v) == static_cast<uint32_t>(bin)) {
                    const uint64_t o = order_of(v, i);
                    lo = o < lo ? o : lo;
                    hi = o > hi ? o : hi;
                }
            });
            __syncthreads();
            n = static_cast<int>(sh.length);
            listed = n <= LIST;
            smallest_and_largest(sh, lo, hi);
            if (t == 0) sh.length = 0; // (read above in front of a barrier)
            if (listed) r.last = find_place(sh, lo, hi, before, than, [&](auto f) __attribute__((always_inline)) { each_listed([&](uint64_t o) { f(o, [&] { return value(logit_of(o)); }); }); });
            else r.last = find_place(sh, lo, hi, before, than, [&](auto f) __attribute__((always_inline)) { r.each([&](float v, uint32_t i) { if (v > -__builtin_inff()) f(order_of(v, i), [&] { return value(v); }); }); });
        } else {
            clear_bins(sh);
            uint64_t sum = 0;
            each_listed([&](uint64_t o) {
                if (o <= r.last) {
                    sum += value(logit_of(o));
                    lo = o < lo ? o : lo;
                    hi = o > hi ? o : hi;
                }
            });
            add_to_bin(sh.bins[wave], sum);
            __syncthreads();
            const uint64_t total = sum_of_bins(sh), than = than_of(total);
            smallest_and_largest(sh, lo, hi);
            if (than >= total) return;
            r.last = find_place(sh, lo, hi, 0, than, [&](auto f) __attribute__((always_inline)) { each_listed([&](uint64_t o) { f(o, [&] { return value(logit_of(o)); }); }); });
        }
    };
    const int32_t k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < a.vocab) cut([](float) { return uint64_t(1); }, [&](uint64_t) { return static_cast<uint64_t>(k - 1); });
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
        // kept: those with less than p of the sum in front of them, so up to the one at which the running sum reaches p of it
        cut([&](float v) { return r.mass(v); }, [&](uint64_t total) {
            const double reach = static_cast<double>(p) * static_cast<double>(total);
            return reach > 1.0 ? static_cast<uint64_t>(__builtin_ceil(reach)) - 1 : uint64_t(0);
        });
    }
    const float m = a.min_p ? a.min_p[row] : 0.0f;
    if (m > 0.0f) r.least = (m < 1.0f ? static_cast<double>(m) : 1.0) * static_cast<double>(ONE);

    // ---- the draw, by index: in the list, or by the sums of the wavefronts' steps and then within one
    const double u = static_cast<double>(a.u[row]);
    auto than_of = [&](uint64_t total) {
        const double reach = u > 0.0 ? u * static_cast<double>(total) : 0.0;
        return reach < static_cast<double>(total - 1) ? static_cast<uint64_t>(reach) : total - 1;
    };
    auto answer = [&](uint32_t index, uint64_t mass, uint64_t total) {
        a.tokens[row] = static_cast<int64_t>(index);
        if (a.probs) a.probs[row] = static_cast<float>(static_cast<double>(mass) / static_cast<double>(total));
    };
    clear_bins(sh);
    if (listed) {
        uint64_t sum = 0;
        each_listed([&](uint64_t o) { sum += o <= r.last ? r.mass(logit_of(o)) : 0; });
        add_to_bin(sh.bins[wave], sum);
        __syncthreads();
        const uint64_t total = sum_of_bins(sh);
        const uint64_t at = find_place(sh, 0, static_cast<uint64_t>(a.vocab - 1), 0, than_of(total), [&](auto f) __attribute__((always_inline)) {
            each_listed([&](uint64_t o) { f(index_of(o), [&] { return o <= r.last ? r.mass(logit_of(o)) : uint64_t(0); }); });
        });
        each_listed([&](uint64_t o) {
            if (index_of(o) == at && o <= r.last) answer(static_cast<uint32_t>(at), r.mass(logit_of(o)), total);
        });
        return;
    }
    uint64_t sum = 0;
    r.each([&](float v, uint32_t i) { if (r.counts(v, i)) sum += r.mass(v); }, [&](int step) {
        const uint64_t s = wave_sum64(sum);
        if (lane == 0) sh.bins[step] = s;
        sum = 0;
    });
    __syncthreads();
    const uint64_t total = sum_of_bins(sh), than = than_of(total);
    uint64_t in_front;
    const int step = find_bin(sh, 0, than, in_front);
    if (wave == 0) {
        const Step<DT> s = r.load(step);
        const uint32_t at = static_cast<uint32_t>(step * STEP + lane * E);
        uint64_t masses[E], mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float v = element<DT>(s, e);
            mine += masses[e] = r.counts(v, at + e) ? r.mass(v) : 0;
        }
        uint64_t upto = mine;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const uint64_t other = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto += other;
        }
        upto += in_front;
        uint64_t front = upto - mine;
        if (upto > than && front <= than) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (front <= than && front + masses[e] > than) answer(at + e, masses[e], total);
                front += masses[e];
            }
        }
    }
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
