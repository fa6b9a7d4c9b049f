// ops::sample with one setting for every row: queued like any other operation, not waited for.
#include <chrono>
#include <cmath>

#include "axhip.h"
#include "oracle_util.hpp"
#include "test_framework.hpp"

using namespace axiom;

GPU_TEST(Sample, OneSettingForEveryRowDoesNotWait) {
    const Tensor logits = axtest::randn({4, 5003}, 7).gpu(), u = Tensor::full<float>({4}, 0.37f, Device::GPU);
    const Tensor room = Tensor::empty({size_t(1) << 28}, DType::Float32, Device::GPU);
    const auto want = ops::sample(logits, u, 0.8f, 40, 0.9f, 0.05f); // (and its outputs' memory is there for the next call)
    const Tensor tokens = want.tokens.cpu();
    for (int i = 0; i < 100; ++i) // some 20 ms of writing
        if (axhip_fill(room.storage()->raw(), AXHIP_DTYPE_F32, 0.0, int64_t(1) << 28, nullptr) != 0) throw RuntimeError("axhip_fill");
    using Clock = std::chrono::steady_clock;
    const auto start = Clock::now();
    const auto got = ops::sample(logits, u, 0.8f, 40, 0.9f, 0.05f);
    const auto called = Clock::now();
    const Tensor again = got.tokens.cpu();
    const auto done = Clock::now();
    EXPECT_TRUE(called - start < done - called); // (the wait for what was queued before it is the program's own, behind the call)
    for (size_t i = 0; i < 4; ++i) EXPECT_EQ(again.typed_data<int64_t>()[i], tokens.typed_data<int64_t>()[i]);
}

GPU_TEST(Sample, OneSettingForEveryRowIsThatOfATensor) {
    const Tensor u = Tensor::full<float>({2, 3}, 0.61f, Device::GPU);
    const float nan = std::nanf("");
    struct Setting { float temperature; int k; float p, m; };
    for (DType dt : {DType::Float32, DType::Float16, DType::BFloat16}) {
        const Tensor logits = axtest::randn({2, 3, 3001}, 9).astype(dt).gpu();
        for (const Setting &s : {Setting{1.0f, 0, 1.0f, 0.0f}, Setting{0.7f, 40, 1.0f, 0.0f}, Setting{1.3f, 0, 0.9f, 0.0f}, Setting{1.0f, 700, 0.8f, 0.02f}, Setting{0.0f, 5, 0.5f, 0.0f},
                                 Setting{nan, 0, 1.0f, 0.0f}, Setting{1.0f, -3, nan, nan}, Setting{0.9f, 1 << 30, 2.0f, 5.0f}}) {
            const auto one = ops::sample(logits, u, s.temperature, s.k, s.p, s.m);
            const auto each = ops::sample(logits, u, ops::SampleSettings{Tensor::full<float>({2, 3}, s.temperature, Device::GPU), Tensor::full<int32_t>({2, 3}, s.k, Device::GPU),
                                                                       Tensor::full<float>({2, 3}, s.p, Device::GPU), Tensor::full<float>({2, 3}, s.m, Device::GPU)});
            const Tensor a = one.tokens.cpu(), b = each.tokens.cpu(), p = one.probabilities.cpu(), q = each.probabilities.cpu();
            for (size_t i = 0; i < 6; ++i) {
                EXPECT_EQ(a.typed_data<int64_t>()[i], b.typed_data<int64_t>()[i]);
                EXPECT_EQ(p.typed_data<float>()[i], q.typed_data<float>()[i]);
            }
        }
    }
}
