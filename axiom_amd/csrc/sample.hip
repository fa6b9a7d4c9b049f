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
    int64_t rows, ld;
    int vocab;
};

constexpr int THREADS = 1024, WAVES = THREADS / WAVE, E = 8; // elements of a lane's vector
constexpr int BINS = 2048;                                   // of a step of the searches: 11 bits
constexpr int STEP = WAVE * E;                               // consecutive elements of a wavefront's step
constexpr int64_t MOST_VOCAB = 1 << 20;                      // BINS steps; and 2^20 weights of 2^43 fit 64 bits
constexpr double ONE = 8796093022208.0;                      // 2^43: the weight of the largest logit

// Floats in the order of their unsigned keys; -0 is +0 (equal logits are ties).  0: nothing (NaN; -inf has 0x007FFFFF).
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t KEY_MINUS_INF = 0x007FFFFFu;
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); }

struct Row {
    const void *logits; // of the row
    int vocab;
    float top;          // the largest logit
    double per_unit;    // 1 / temperature
    // what is kept: keys above `key`, and of those equal to it the indexes up to `index`; and weights of at least `least`
    uint32_t key, index;
    double least;
    __device__ double weight(uint32_t k) const {
        const float v = of_key(k);
        return v == top ? 1.0 : exp((static_cast<double>(v) - static_cast<double>(top)) * per_unit);
    }
    __device__ bool first_ones(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= index); }
    // in multiples of 2^-43, 0 where the element is not kept
    __device__ uint64_t mass(uint32_t k, uint32_t i) const {
        if (k <= KEY_MINUS_INF || !first_ones(k, i)) return 0;
        const double w = weight(k);
        return w >= least ? static_cast<uint64_t>(__builtin_rint(w * ONE)) : 0; // (NaN, of an infinite temperature: 0)
    }
};

template <int DT, class F> __device__ __forceinline__ void each_step(const Row &r, int step, F f) {
    const int at = step * STEP + (threadIdx.x % WAVE) * E;
    float v[E];
    if (at + E <= r.vocab) {
        load_vec<E, true>(r.logits, DT, at, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = at + e < r.vocab ? Elem<DT>::load(r.logits, at + e) : __uint_as_float(0x7FC00000u);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f(key_of(v[e]), static_cast<uint32_t>(at + e));
}
template <int DT, class F> __device__ __forceinline__ void each(const Row &r, F f) {
    const int steps = (r.vocab + STEP - 1) / STEP;
    for (int step = threadIdx.x / WAVE; step < steps; step += WAVES) each_step<DT>(r, step, f);
}

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
    for (int d = 32; d; d /= 2) v += __shfl_xor(v, d, WAVE);
    return v;
}

// s[0 .. BINS) -> the first bin, counted from `from_above` ? the top : the bottom, at which the running sum (with `before` in front) exceeds
// `than`, and the sum in front of it.  Every thread gets the answer; the last bin with anything where none does.
__device__ void find_bin(uint64_t *s, uint64_t *scratch, bool from_above, uint64_t before, uint64_t than, int &bin, uint64_t &in_front) {
    static_assert(BINS == 2 * THREADS, "two bins a thread");
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
    const int b0 = from_above ? BINS - 1 - 2 * t : 2 * t, b1 = from_above ? b0 - 1 : b0 + 1;
    const uint64_t v0 = s[b0], v1 = s[b1];
    uint64_t upto = v0 + v1;
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
        const uint64_t other = __shfl_up(upto, d, WAVE);
        if (lane >= d) upto += other;
    }
    if (lane == WAVE - 1) scratch[wave] = upto;
    if (t == 0) scratch[WAVES] = ~0ull;
    __syncthreads();
    uint64_t first = before;
    for (int w = 0; w < wave; ++w) first += scratch[w];
    const uint64_t all = first + upto, mine = all - v0 - v1;
    if (all > than && mine <= than) scratch[WAVES] = static_cast<uint64_t>(mine + v0 > than ? b0 : b1), scratch[WAVES + 1] = mine + v0 > than ? mine : mine + v0;
    __syncthreads();
    bin = static_cast<int>(scratch[WAVES]);
    in_front = scratch[WAVES + 1];
    __syncthreads();
}

template <int DT>
__global__ __launch_bounds__(THREADS) void sample_kernel(const SampleArgs a) {
    __shared__ uint64_t s_bins[BINS], s_scratch[WAVES + 2];
    __shared__ uint32_t s_key[WAVES], s_index[WAVES];
    const int t = threadIdx.x, lane = t % WAVE, wave = t / WAVE;
    const int64_t row = blockIdx.x;
    constexpr int64_t ES = DT == AXHIP_DTYPE_F32 ? 4 : 2;
    Row r;
    r.logits = static_cast<const char *>(a.logits) + row * a.ld * ES;
    r.vocab = a.vocab;
    const float temperature = a.temperature ? a.temperature[row] : 1.0f;

    // the largest logit and where it stands first
    uint32_t best = 0, where = 0;
    each<DT>(r, [&](uint32_t k, uint32_t i) {
        if (k > best) { best = k; where = i; } // (a thread meets its indexes in order)
    });
#pragma unroll
    for (int d = 32; d; d /= 2) {
        const uint32_t k = __shfl_xor(best, d, WAVE), i = __shfl_xor(where, d, WAVE);
        if (k > best || (k == best && i < where)) { best = k; where = i; }
    }
    if (lane == 0) { s_key[wave] = best; s_index[wave] = where; }
    __syncthreads();
    for (int w = 0; w < WAVES; ++w)
        if (s_key[w] > best || (s_key[w] == best && s_index[w] < where)) { best = s_key[w]; where = s_index[w]; }
    if (best <= KEY_MINUS_INF || !(temperature > 0.0f)) { // (the same in every thread)
        if (t == 0) {
            a.tokens[row] = best <= KEY_MINUS_INF ? -1 : static_cast<int64_t>(where);
            if (a.probs) a.probs[row] = best <= KEY_MINUS_INF ? 0.0f : 1.0f;
        }
        return;
    }
    r.top = of_key(best);
    r.per_unit = 1.0 / static_cast<double>(temperature);
    r.key = 0;
    r.index = 0xFFFFFFFFu;
    r.least = 0.0;

    // The element at which the running sum of `value`, in the order larger key first, equal ones by index, exceeds `than`: from then on kept up to it.
    auto cut = [&](auto value, uint64_t than) {
        uint32_t prefix = 0;
        uint64_t before = 0;
        int bin;
        bool alone = false;
        constexpr int SHIFTS[3] = {21, 10, 0}, BITS[3] = {11, 11, 10};
        for (int level = 0; level < 3; ++level) {
            for (int b = t; b < BINS; b += THREADS) s_bins[b] = 0;
            __syncthreads();
            const int shift = SHIFTS[level], done = shift + BITS[level];
            each<DT>(r, [&](uint32_t k, uint32_t i) {
                if (level > 0 && (k >> done) != prefix) return;
                const uint64_t v = value(k, i);
                if (v) atomicAdd(reinterpret_cast<unsigned long long *>(&s_bins[(k >> shift) & ((1u << BITS[level]) - 1)]), static_cast<unsigned long long>(v));
            });
            __syncthreads();
            uint64_t in_front;
            find_bin(s_bins, s_scratch, true, before, than, bin, in_front);
            if (bin < 0) return; // (nothing reaches it: all are kept)
            before = in_front;
            prefix = (prefix << BITS[level]) | static_cast<uint32_t>(bin);
        }
        (void)alone;
        uint32_t place = 0;
        for (int level = 0; level < 2; ++level) {
            for (int b = t; b < BINS; b += THREADS) s_bins[b] = 0;
            __syncthreads();
            each<DT>(r, [&](uint32_t k, uint32_t i) {
                if (k != prefix || (level == 1 && (i >> 10) != place)) return;
                const uint64_t v = value(k, i);
                if (v) atomicAdd(reinterpret_cast<unsigned long long *>(&s_bins[level == 0 ? i >> 10 : i & 1023]), static_cast<unsigned long long>(v));
            });
            __syncthreads();
            uint64_t in_front;
            find_bin(s_bins, s_scratch, false, before, than, bin, in_front);
            if (bin < 0) return;
            before = in_front;
            place = level == 0 ? static_cast<uint32_t>(bin) : (place << 10) | static_cast<uint32_t>(bin);
        }
        r.key = prefix;
        r.index = place;
    };

    const int32_t k = a.top_k ? a.top_k[row] : 0;
    if (k > 0 && k < a.vocab) cut([](uint32_t, uint32_t) { return uint64_t(1); }, static_cast<uint64_t>(k - 1));
    auto total_mass = [&]() -> uint64_t {
        uint64_t sum = 0;
        each<DT>(r, [&](uint32_t key, uint32_t i) { sum += r.mass(key, i); });
        sum = wave_sum64(sum);
        __syncthreads();
        if (lane == 0) s_scratch[wave] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < WAVES; ++w) sum += s_scratch[w];
        __syncthreads();
        return sum;
    };
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
        // kept: those with less than p of the mass in front of them, so up to the one at which the running sum reaches p of it
        const double reach = static_cast<double>(p) * static_cast<double>(total_mass());
        cut([&](uint32_t key, uint32_t i) { return r.mass(key, i); }, reach > 1.0 ? static_cast<uint64_t>(__builtin_ceil(reach)) - 1 : 0);
    }
    const float m = a.min_p ? a.min_p[row] : 0.0f;
    if (m > 0.0f) r.least = m < 1.0f ? static_cast<double>(m) : 1.0;

    // the draw: the sums of the wavefronts' steps, then the step's own
    for (int b = t; b < BINS; b += THREADS) s_bins[b] = 0;
    __syncthreads();
    const int steps = (r.vocab + STEP - 1) / STEP;
    for (int step = wave; step < steps; step += WAVES) {
        uint64_t sum = 0;
        each_step<DT>(r, step, [&](uint32_t key, uint32_t i) { sum += r.mass(key, i); });
        sum = wave_sum64(sum);
        if (lane == 0) s_bins[step] = sum;
    }
    __syncthreads();
    uint64_t total = 0;
    for (int b = t; b < BINS; b += THREADS) total += s_bins[b];
    total = wave_sum64(total);
    if (lane == 0) s_scratch[wave] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < WAVES; ++w) total += s_scratch[w];
    __syncthreads();
    const double u = static_cast<double>(a.u[row]);
    const double reach = u > 0.0 ? u * static_cast<double>(total) : 0.0;
    const uint64_t than = reach < static_cast<double>(total - 1) ? static_cast<uint64_t>(reach) : total - 1;
    int step;
    uint64_t in_front;
    find_bin(s_bins, s_scratch, false, 0, than, step, in_front);
    if (wave == 0) {
        uint64_t masses[E], sum = 0;
        int n = 0;
        each_step<DT>(r, step, [&](uint32_t key, uint32_t i) { sum += masses[n++] = r.mass(key, i); });
        uint64_t upto = sum;
#pragma unroll
        for (int d = 1; d < WAVE; d *= 2) {
            const uint64_t other = __shfl_up(upto, d, WAVE);
            if (lane >= d) upto += other;
        }
        upto += in_front;
        uint64_t mine = upto - sum;
        if (upto > than && mine <= than) {
            for (int e = 0; e < E; ++e) {
                if (mine + masses[e] > than) {
                    a.tokens[row] = static_cast<int64_t>(step) * STEP + lane * E + e;
                    if (a.probs) a.probs[row] = static_cast<float>(static_cast<double>(masses[e]) / static_cast<double>(total));
                    break;
                }
                mine += masses[e];
            }
        }
    }
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
    const SampleArgs a{logits, tokens, probs, p.temperature, p.top_k, p.top_p, p.min_p, p.u, p.rows, p.ld, static_cast<int>(p.vocab)};
    const dim3 grid(static_cast<unsigned>(p.rows));
    if (p.dtype == AXHIP_DTYPE_F32) hipLaunchKernelGGL((sample_kernel<AXHIP_DTYPE_F32>), grid, dim3(THREADS), 0, s, a);
    else if (p.dtype == AXHIP_DTYPE_F16) hipLaunchKernelGGL((sample_kernel<AXHIP_DTYPE_F16>), grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((sample_kernel<AXHIP_DTYPE_BF16>), grid, dim3(THREADS), 0, s, a);
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
