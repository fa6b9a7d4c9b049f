// A token from each row of logits: axhip_sample.
#include "sample.hpp"

namespace axhip {
namespace {

int sample(const void *logits, int64_t *tokens, float *probs, const AxhipSampleParams *params, void *, size_t, void *stream) {
    AXHIP_REQUIRE(params != nullptr, AXHIP_ERR_INVALID_ARG, "axhip_sample: params is NULL");
    const AxhipSampleParams &p = *params;
    AXHIP_REQUIRE(valid_dtype(p.dtype), AXHIP_ERR_INVALID_ARG, "axhip_sample: bad dtype %d", p.dtype);
    AXHIP_REQUIRE(p.rows >= 0 && p.rows < (int64_t(1) << 22), AXHIP_ERR_INVALID_ARG, "axhip_sample: bad number of rows");
    AXHIP_REQUIRE(p.vocab > 0, AXHIP_ERR_INVALID_ARG, "axhip_sample: an empty vocabulary");
    AXHIP_REQUIRE(p.vocab <= MOST_VOCAB, AXHIP_ERR_UNSUPPORTED, "axhip_sample: a vocabulary of %lld (up to %lld)", static_cast<long long>(p.vocab), static_cast<long long>(MOST_VOCAB));
    AXHIP_REQUIRE(p.ld >= p.vocab && p.ld < (int64_t(1) << 40), AXHIP_ERR_INVALID_ARG, "axhip_sample: bad leading dimension");
    AXHIP_REQUIRE(p.uniform == 0 || p.uniform == 1, AXHIP_ERR_INVALID_ARG, "axhip_sample: uniform is %d, neither 0 nor 1", p.uniform);
    AXHIP_REQUIRE(!p.uniform || !(p.temperature || p.top_k || p.top_p || p.min_p), AXHIP_ERR_INVALID_ARG, "axhip_sample: an array of settings beside uniform ones");
    if (p.rows == 0) return AXHIP_OK;
    AXHIP_REQUIRE(logits && tokens && p.u, AXHIP_ERR_INVALID_ARG, "axhip_sample: NULL buffer");
    AXHIP_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (dtype_size(p.dtype) - 1)) == 0 && (reinterpret_cast<uintptr_t>(tokens) & 7u) == 0 &&
                      ((reinterpret_cast<uintptr_t>(probs) | reinterpret_cast<uintptr_t>(p.temperature) | reinterpret_cast<uintptr_t>(p.top_k) | reinterpret_cast<uintptr_t>(p.top_p) |
                        reinterpret_cast<uintptr_t>(p.min_p) | reinterpret_cast<uintptr_t>(p.u)) & 3u) == 0,
                  AXHIP_ERR_INVALID_ARG, "axhip_sample: a buffer is not aligned to its elements");
    int rc = ensure_init();
    if (rc) return rc;
    hipStream_t s = resolve_stream(stream);
    SampleArgs a{logits, tokens, probs, p.temperature, p.top_k, p.top_p, p.min_p, p.u, p.ld, static_cast<int>(p.vocab), 0, 1.0f, 1.0f, 0.0f};
    if (p.uniform) {
        a.all_top_k = p.all_top_k;
        a.all_temperature = p.all_temperature;
        a.all_top_p = p.all_top_p;
        a.all_min_p = p.all_min_p;
    }
    rc = p.dtype == AXHIP_DTYPE_F32 ? launch_sample_f32(a, p.rows, s) : p.dtype == AXHIP_DTYPE_F16 ? launch_sample_f16(a, p.rows, s) : launch_sample_bf16(a, p.rows, s);
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
