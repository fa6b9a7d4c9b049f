// Rows in 8 bits, products of them, the module over them and sampling: argument checks on any machine, results on the GPU against the definitions in doubles.
#include <algorithm>
#include <numeric>

#include "oracle_util.hpp"
#include "test_framework.hpp"

using namespace axiom;

static std::vector<double> doubles(const Tensor &t) {
    const Tensor c = t.cpu().astype(DType::Float32).ascontiguousarray();
    const float *p = c.typed_data<float>();
    return std::vector<double>(p, p + c.size());
}
static std::vector<int8_t> bytes(const Tensor &t) {
    const Tensor c = t.cpu().ascontiguousarray();
    const int8_t *p = c.typed_data<int8_t>();
    return std::vector<int8_t>(p, p + c.size());
}
// rows of values -> integers and largest magnitudes
static void nearest(const std::vector<double> &y, size_t cols, std::vector<int8_t> &q, std::vector<double> &largest) {
    q.resize(y.size());
    largest.assign(y.size() / cols, 0.0);
    for (size_t i = 0; i < y.size(); ++i) largest[i / cols] = std::max(largest[i / cols], std::fabs(y[i]));
    for (size_t i = 0; i < y.size(); ++i) q[i] = largest[i / cols] > 0 ? static_cast<int8_t>(std::nearbyint(127.0 * y[i] / largest[i / cols])) : 0;
}

TEST(Quantized, CpuTensorsAndMismatchesThrow) {
    const Tensor x = Tensor::zeros({2, 8});
    const ops::Quantized q{Tensor::zeros({2, 8}, DType::Int8), Tensor::zeros({2})};
    EXPECT_THROW(ops::quantize_int8(x), RuntimeError);
    EXPECT_THROW(ops::quantize_int8(Tensor()), ValueError);
    EXPECT_THROW(ops::rms_norm_int8(x, Tensor(), Tensor()), RuntimeError);
    EXPECT_THROW(ops::linear_int8(q, q, DType::Float32), RuntimeError);
    EXPECT_THROW(ops::sample(x, Tensor::zeros({2})), RuntimeError);
    nn::QuantizedLinear l;
    EXPECT_THROW(l.forward(x), RuntimeError);
    EXPECT_THROW(l.forward(q, DType::Float32, Tensor()), RuntimeError); // no weight
    EXPECT_THROW(nn::QuantizedLinear(nn::Linear()), RuntimeError);
    EXPECT_EQ(l.named_parameters().size(), size_t(3));
    EXPECT_EQ(nn::QuantizedLinear(false).named_parameters().size(), size_t(2));
}

GPU_TEST(Quantized, RowsAndNorm) {
    for (DType dt : {DType::Float32, DType::Float16, DType::BFloat16}) {
        const size_t cols = 333;
        const Tensor x = axtest::randn({3, 5, cols}, 3).astype(dt), r = axtest::randn({3, 5, cols}, 4).astype(dt), w = axtest::randn({cols}, 5).astype(dt);
        const auto q = ops::quantize_int8(x.gpu());
        EXPECT_EQ(q.values.shape(), (Shape{3, 5, cols}));
        EXPECT_EQ(q.scales.shape(), (Shape{3, 5}));
        std::vector<int8_t> want;
        std::vector<double> largest;
        nearest(doubles(x), cols, want, largest);
        EXPECT_TRUE(bytes(q.values) == want);
        const auto scales = doubles(q.scales);
        for (size_t i = 0; i < scales.size(); ++i) EXPECT_NEAR(scales[i], largest[i] / 127, 3e-7 * largest[i] / 127);

        const auto n = ops::rms_norm_int8(x.gpu(), r.gpu(), w.gpu());
        const auto h = doubles(n.sum), wd = doubles(w);
        const auto hx = doubles(x), hr = doubles(r);
        const double half_step = dt == DType::Float32 ? std::ldexp(1.0, -24) : dt == DType::Float16 ? std::ldexp(1.0, -11) : std::ldexp(1.0, -8);
        for (size_t i = 0; i < h.size(); ++i) EXPECT_NEAR(h[i], hx[i] + hr[i], 1.01 * half_step * std::fabs(hx[i] + hr[i]) + 1e-7);
        std::vector<double> y(h.size()), mean(h.size() / cols, 0.0);
        for (size_t i = 0; i < h.size(); ++i) {
            y[i] = h[i] * wd[i % cols];
            mean[i / cols] += h[i] * h[i] / cols;
        }
        nearest(y, cols, want, largest);
        EXPECT_TRUE(bytes(n.normalized.values) == want);
        const auto s = doubles(n.normalized.scales);
        for (size_t i = 0; i < s.size(); ++i) {
            const double expected = largest[i] / 127 / std::sqrt(mean[i] + 1e-5);
            EXPECT_NEAR(s[i], expected, 2e-6 * expected); // (sums of 333 squares: 22 roundings at most, and five more)
        }
        const auto plain = ops::rms_norm_int8(x.gpu(), Tensor(), Tensor());
        EXPECT_TRUE(plain.sum.empty());
    }
    const Tensor g = axtest::randn({4, 8}, 1).gpu();
    EXPECT_THROW(ops::rms_norm_int8(g, axtest::randn({4, 9}, 1).gpu(), Tensor()), ShapeError);
    EXPECT_THROW(ops::rms_norm_int8(g, Tensor(), axtest::randn({9}, 1).gpu()), ShapeError);
    EXPECT_THROW(ops::rms_norm_int8(g, g.half(), Tensor()), TypeError);
    EXPECT_THROW(ops::rms_norm_int8(g, Tensor(), Tensor(), -1.0f), ValueError);
    EXPECT_THROW(ops::quantize_int8(Tensor::zeros({4, 8}, DType::Int32).gpu()), TypeError);
    // a lazy input and a transposed view are settled first
    const auto lazy = ops::quantize_int8(ops::relu(g)), view = ops::quantize_int8(g.transpose({1, 0}));
    EXPECT_EQ(lazy.values.shape(), (Shape{4, 8}));
    std::vector<int8_t> want;
    std::vector<double> largest;
    nearest(doubles(g.transpose({1, 0}).ascontiguousarray()), 4, want, largest);
    EXPECT_TRUE(bytes(view.values) == want);
}

GPU_TEST(Quantized, LinearAgainstItsIntegers) {
    for (DType dt : {DType::Float32, DType::BFloat16}) {
        const size_t m = 6, n = 70, k = 200;
        nn::Linear l;
        l.load_state_dict({{"weight", axtest::randn({n, k}, 1).astype(dt).gpu()}, {"bias", axtest::randn({n}, 2).astype(dt).gpu()}});
        const nn::QuantizedLinear q(l);
        const Tensor x = axtest::randn({2, 3, k}, 3).astype(dt).gpu(), res = axtest::randn({2, 3, n}, 4).astype(dt).gpu();
        const auto qx = ops::quantize_int8(x);
        const auto a = bytes(qx.values), b = bytes(q.weight());
        const auto sa = doubles(qx.scales), sb = doubles(q.weight_scale()), bias = doubles(l.bias()), r = doubles(res);
        const Tensor y = q(x), z = q.forward(qx, dt, res, "relu");
        EXPECT_EQ(y.shape(), (Shape{2, 3, n}));
        EXPECT_EQ(y.dtype(), dt);
        const auto yd = doubles(y), zd = doubles(z);
        const double half_step = dt == DType::Float32 ? 0.0 : std::ldexp(1.0, -8);
        for (size_t i = 0; i < m; ++i)
            for (size_t j = 0; j < n; ++j) {
                int64_t sum = 0;
                for (size_t e = 0; e < k; ++e) sum += int64_t(a[i * k + e]) * b[j * k + e];
                const double v = sum * sa[i] * sb[j] + bias[j], w = std::max(0.0, v + r[i * n + j]);
                EXPECT_NEAR(yd[i * n + j], v, half_step * 1.01 * std::fabs(v) + 1e-5);
                EXPECT_NEAR(zd[i * n + j], w, half_step * 1.01 * w + 1e-5);
            }
        // the product of the original weight is as near as 8 bits are: each factor is off by half an integer of 127 at most
        const auto full = doubles(l(x));
        double off = 0, size = 0;
        for (size_t i = 0; i < full.size(); ++i) {
            off += (full[i] - yd[i]) * (full[i] - yd[i]);
            size += full[i] * full[i];
        }
        EXPECT_TRUE(off < 0.02 * 0.02 * size);
    }
    const ops::Quantized q{Tensor::zeros({2, 8}, DType::Int8).gpu(), Tensor::zeros({2}).gpu()};
    EXPECT_THROW(ops::linear_int8(q, {Tensor::zeros({3, 9}, DType::Int8).gpu(), Tensor::zeros({3}).gpu()}, DType::Float32), ShapeError);
    EXPECT_THROW(ops::linear_int8(q, {Tensor::zeros({3, 8}, DType::Int8).gpu(), Tensor::zeros({2}).gpu()}, DType::Float32), ShapeError);
    EXPECT_THROW(ops::linear_int8(q, q, DType::Int32), TypeError);
    EXPECT_THROW(ops::linear_int8(q, q, Tensor(), Tensor(), "softplus", DType::Float32), ValueError);
    EXPECT_THROW(ops::linear_int8(q, q, Tensor::zeros({3}).gpu(), Tensor(), "none", DType::Float32), ShapeError);
    EXPECT_THROW(ops::linear_int8(q, q, Tensor::zeros({2}).gpu(), Tensor(), "none", DType::BFloat16), TypeError);
    EXPECT_THROW(ops::linear_int8(q, q, Tensor(), Tensor::zeros({2, 3}).gpu(), "none", DType::Float32), ShapeError);
}

// one row: the token by the definition
static int64_t token_of(const std::vector<double> &l, double u, double temperature, size_t k, double p, double m) {
    std::vector<size_t> order(l.size());
    std::iota(order.begin(), order.end(), size_t(0));
    std::stable_sort(order.begin(), order.end(), [&](size_t a, size_t b) { return l[a] > l[b]; });
    size_t n = k ? std::min(k, l.size()) : l.size();
    std::vector<double> w(l.size());
    double total = 0;
    for (size_t i = 0; i < l.size(); ++i) w[i] = std::exp((l[i] - l[order[0]]) / temperature);
    for (size_t i = 0; i < n; ++i) total += w[order[i]];
    size_t kept = 0;
    for (double before = 0; kept < n && (kept == 0 || (before < p * total && w[order[kept]] >= m)); ++kept) before += w[order[kept]];
    std::vector<double> mass(l.size(), 0.0);
    total = 0;
    for (size_t i = 0; i < kept; ++i) total += mass[order[i]] = w[order[i]];
    double upto = 0;
    for (size_t i = 0; i < l.size(); ++i)
        if ((upto += mass[i]) > u * total) return static_cast<int64_t>(i);
    return -2;
}

GPU_TEST(Sample, TokensOfEveryRow) {
    const size_t vocab = 5003;
    for (DType dt : {DType::Float32, DType::BFloat16}) {
        const Tensor logits = axtest::randn({2, 4, vocab}, 7).astype(dt), u = Tensor::full<float>({2, 4}, 0.37f);
        const auto l = doubles(logits);
        for (int c = 0; c < 4; ++c) {
            const float t = c == 0 ? 1.0f : 0.8f, p = c == 2 ? 0.9f : 1.0f, m = c == 3 ? 0.125f : 0.0f;
            const int k = c == 1 ? 50 : c == 2 ? 1000 : 0;
            const auto got = ops::sample(logits.gpu(), u.gpu(), t, k, p, m);
            EXPECT_EQ(got.tokens.shape(), (Shape{2, 4}));
            const Tensor tokens = got.tokens.cpu();
            const auto probs = doubles(got.probabilities);
            for (size_t i = 0; i < 8; ++i) {
                EXPECT_EQ(tokens.typed_data<int64_t>()[i], token_of({l.begin() + i * vocab, l.begin() + (i + 1) * vocab}, 0.37f, t, k, p, m));
                EXPECT_TRUE(probs[i] > 0 && probs[i] <= 1);
            }
        }
        const Tensor greedy = ops::sample(logits.gpu(), u.gpu(), 0.0f).tokens.cpu(), want = ops::argmax(logits.gpu(), -1).cpu();
        for (size_t i = 0; i < 8; ++i) EXPECT_EQ(greedy.typed_data<int64_t>()[i], want.typed_data<int64_t>()[i]);
    }
    const Tensor g = axtest::randn({3, 10}, 1).gpu();
    EXPECT_THROW(ops::sample(g, Tensor::zeros({2}).gpu()), ShapeError);
    EXPECT_THROW(ops::sample(g, Tensor::zeros({3}).gpu(), ops::SampleSettings{Tensor::zeros({1}).gpu(), {}, {}, {}}), ShapeError);
    EXPECT_THROW(ops::sample(g, Tensor::zeros({3}).gpu(), ops::SampleSettings{{}, Tensor::zeros({3}).gpu(), {}, {}}), TypeError);
    EXPECT_THROW(ops::sample(Tensor::zeros({3, 10}, DType::Int8).gpu(), Tensor::zeros({3}).gpu()), TypeError);
    EXPECT_THROW(ops::sample(g, Tensor()), ValueError);
}

// the end of a decoding step as a program runs it: sum and norm in 8 bits, feed-forward block in 8 bits, logits, a token
GPU_TEST(Quantized, TheEndOfADecodingStep) {
    const size_t tokens = 5, width = 256, inner = 1024, vocab = 3001;
    const DType dt = DType::BFloat16;
    auto linear = [&](size_t out, size_t in, unsigned seed) {
        auto l = std::make_unique<nn::Linear>(false);
        l->load_state_dict({{"weight", (axtest::randn({out, in}, seed).gpu() * (1.0f / std::sqrt(float(in)))).astype(dt)}});
        return l;
    };
    const auto up = linear(inner, width, 1), down = linear(width, inner, 2), head = linear(vocab, width, 3);
    const nn::QuantizedLinear qup(*up), qdown(*down), qhead(*head);
    const Tensor x = axtest::randn({tokens, width}, 4).astype(dt).gpu(), res = axtest::randn({tokens, width}, 5).astype(dt).gpu();
    const Tensor w = Tensor::full<float>({width}, 1.0f, Device::GPU).astype(dt);

    const auto n1 = ops::rms_norm_int8(x, res, w);
    const Tensor hidden = qup.forward(n1.normalized, dt, Tensor(), "silu");
    const Tensor out = qdown.forward(ops::quantize_int8(hidden), dt, n1.sum);
    const auto n2 = ops::rms_norm_int8(out, Tensor(), w);
    const Tensor logits = qhead.forward(n2.normalized, DType::Float32, Tensor());
    const auto got = ops::sample(logits, Tensor::full<float>({tokens}, 0.6f, Device::GPU), 0.9f, 40, 0.95f);

    // the same in the weights' own type: as near as the 8 bits leave it
    const Tensor sum = ops::add(x, res), h2 = ops::silu((*up)(ops::rms_norm(sum, w)));
    const auto full = doubles((*head)(ops::rms_norm(ops::add((*down)(h2), sum), w))), l = doubles(logits);
    double off = 0, size = 0;
    for (size_t i = 0; i < l.size(); ++i) {
        off += (full[i] - l[i]) * (full[i] - l[i]);
        size += full[i] * full[i];
    }
    EXPECT_TRUE(off < 0.05 * 0.05 * size);
    const Tensor t = got.tokens.cpu();
    for (size_t i = 0; i < tokens; ++i)
        EXPECT_EQ(t.typed_data<int64_t>()[i], token_of({l.begin() + i * vocab, l.begin() + (i + 1) * vocab}, 0.6f, 0.9f, 40, 0.95f, 0.0));
}
