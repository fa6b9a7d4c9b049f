// Shared by sample.hip and the sample_*.hip translation units (one for each type of logits).
#pragma once
#include "common.hpp"

namespace axhip {

struct SampleArgs {
    const void *logits;
    int64_t *tokens;
    float *probs;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p, *min_p, *u;
    int64_t ld;
    int vocab;
    int32_t all_top_k; // where there is no array
    float all_temperature, all_top_p, all_min_p;
};

constexpr int64_t MOST_VOCAB = 1 << 20;

int launch_sample_f32(const SampleArgs &a, int64_t rows, hipStream_t s);
int launch_sample_f16(const SampleArgs &a, int64_t rows, hipStream_t s);
int launch_sample_bf16(const SampleArgs &a, int64_t rows, hipStream_t s);

} // namespace axhip
