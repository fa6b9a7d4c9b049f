// Rotary positions, packed attention and the paged cache: bookkeeping and argument checks on any machine, results on the GPU against the definitions in doubles.
#include <algorithm>
#include <map>
#include <set>

#include "axhip.h"
#include "oracle_util.hpp"
#include "test_framework.hpp"

using namespace axiom;
using nn::PageBook;

namespace {
std::vector<double> doubles(const Tensor &t) {
    const Tensor c = t.cpu().astype(DType::Float32).ascontiguousarray();
    const float *p = c.typed_data<float>();
    return std::vector<double>(p, p + c.size());
}
Tensor ints(const std::vector<int32_t> &v) { return Tensor::from_data(v.data(), Shape{v.size()}, Device::GPU); }
double half_step(DType dt) { return dt == DType::Float32 ? std::ldexp(1.0, -24) : dt == DType::Float16 ? std::ldexp(1.0, -11) : std::ldexp(1.0, -8); }

// one sequence in doubles: q [rows][heads][dim] against keys and values [n][kv][dim]; row i sees keys up to n - rows + i
std::vector<double> attention(const std::vector<double> &q, const std::vector<double> &k, const std::vector<double> &v, size_t heads, size_t kv, size_t dim, bool causal) {
    const size_t rows = q.size() / (heads * dim), n = k.size() / (kv * dim);
    std::vector<double> o(q.size(), 0.0);
    for (size_t i = 0; i < rows; ++i)
        for (size_t h = 0; h < heads; ++h) {
            const size_t g = h / (heads / kv), seen = causal ? (n + i + 1 > rows ? n + i + 1 - rows : 0) : n;
            std::vector<double> s(seen);
            double top = -1e300, sum = 0;
            for (size_t j = 0; j < seen; ++j) {
                for (size_t d = 0; d < dim; ++d) s[j] += q[(i * heads + h) * dim + d] * k[(j * kv + g) * dim + d];
                s[j] /= std::sqrt(double(dim));
                top = std::max(top, s[j]);
            }
            for (size_t j = 0; j < seen; ++j) sum += s[j] = std::exp(s[j] - top);
            for (size_t j = 0; j < seen; ++j)
                for (size_t d = 0; d < dim; ++d) o[(i * heads + h) * dim + d] += s[j] / sum * v[(j * kv + g) * dim + d];
        }
    return o;
}
// Weights round once in numerator and denominator and values are below 5: an output is off by 2 * 5 half steps and, of values below 1, its own (16 bits); in 32 bits by the sums' roundings:
// 64 products of a score, up to 200 keys
double tolerance(DType dt) { return dt == DType::Float32 ? 2e-5 : 11 * half_step(dt); }

std::vector<double> rotated(std::vector<double> x, const std::vector<int64_t> &positions, size_t heads, size_t dim, size_t rot, double theta, bool interleaved) {
    for (size_t t = 0; t < positions.size(); ++t)
        for (size_t h = 0; h < heads; ++h)
            for (size_t i = 0; i < rot / 2; ++i) {
                const double angle = positions[t] * std::pow(theta, -2.0 * i / rot);
                double *head = &x[(t * heads + h) * dim], &a = head[interleaved ? 2 * i : i], &b = head[interleaved ? 2 * i + 1 : i + rot / 2], pa = a, pb = b;
                a = pa * std::cos(angle) - pb * std::sin(angle);
                b = pb * std::cos(angle) + pa * std::sin(angle);
            }
    return x;
}
} // namespace

TEST(PageBook, AddsForksAndGivesBack) {
    PageBook book(8, 4);
    std::vector<PageBook::Copy> copies;
    const int a = book.add();
    book.extend({a}, {6}, copies);
    EXPECT_EQ(book.length(a), size_t(6));
    EXPECT_TRUE(book.pages(a) == (std::vector<int32_t>{0, 1}));
    EXPECT_EQ(book.slot(a, 5), int64_t(5));
    EXPECT_EQ(book.free_pages(), size_t(6));
    const int b = book.fork(a);
    EXPECT_EQ(book.free_pages(), size_t(6));
    book.extend({a, b}, {1, 3}, copies); // both write to page 1: the first one copies it, the other one keeps it
    EXPECT_EQ(copies.size(), size_t(1));
    EXPECT_EQ(copies[0].src, int32_t(1));
    EXPECT_EQ(copies[0].dst, int32_t(2));
    EXPECT_EQ(copies[0].rows, int32_t(2));
    EXPECT_TRUE(book.pages(a) == (std::vector<int32_t>{0, 2}));
    EXPECT_TRUE(book.pages(b) == (std::vector<int32_t>{0, 1, 3}));
    book.release(a);
    EXPECT_EQ(book.free_pages(), size_t(5)); // page 0 is b's too
    EXPECT_THROW(book.length(a), IndexError);
    EXPECT_EQ(book.add(), a);
    book.truncate(b, 4);
    EXPECT_TRUE(book.pages(b) == (std::vector<int32_t>{0}));
    EXPECT_THROW(book.truncate(b, 5), ValueError);
    EXPECT_THROW(book.slot(b, 4), IndexError);
}

TEST(PageBook, RunsOutWithoutAChange) {
    PageBook book(4, 4);
    std::vector<PageBook::Copy> copies;
    const int a = book.add(), b = book.add();
    book.extend({a}, {10}, copies);
    EXPECT_THROW(book.extend({a, b}, {3, 2}, copies), RuntimeError); // two pages, one is free
    EXPECT_EQ(book.length(a), size_t(10));
    EXPECT_EQ(book.length(b), size_t(0));
    EXPECT_EQ(book.free_pages(), size_t(1));
    EXPECT_TRUE(copies.empty());
    book.extend({a, b}, {2, 4}, copies);
    EXPECT_EQ(book.free_pages(), size_t(0));
    const int c = book.fork(a);
    book.truncate(c, 11);
    EXPECT_THROW(book.extend({c}, {1}, copies), RuntimeError); // its last page is a's too
    EXPECT_THROW(book.extend({a, a}, {1, 1}, copies), ValueError);
    EXPECT_THROW(book.extend({a}, {1, 1}, copies), ValueError);
    EXPECT_THROW(book.extend({7}, {1}, copies), IndexError);
    EXPECT_THROW(PageBook(4, 3), ValueError);
    EXPECT_THROW(PageBook(4, 0), ValueError);
}

// Every page has as many users as sequences list it; what a sequence holds survives copies, forks and compaction
TEST(PageBook, RandomOperationsKeepWhatSequencesHold) {
    PageBook book(40, 4);
    std::vector<int> live;
    std::map<int, std::vector<int>> tokens;            // what a sequence holds
    std::vector<std::vector<int>> pool(40, std::vector<int>(4, -1)); // what the pages hold
    uint32_t r = 12345;
    int next = 0;
    auto any = [&](uint32_t n) {
        r = r * 1664525u + 1013904223u;
        return (r >> 12) % n;
    };
    auto apply = [&](const std::vector<PageBook::Copy> &copies) {
        for (const auto &c : copies)
            for (int32_t i = 0; i < c.rows; ++i) pool[c.dst][i] = pool[c.src][i];
    };
    for (int turn = 0; turn < 3000; ++turn) {
        const uint32_t what = any(10);
        if (what == 0 || live.empty()) {
            live.push_back(book.add());
            tokens[live.back()] = {};
        } else if (what == 1) {
            const int from = live[any(live.size())];
            live.push_back(book.fork(from));
            tokens[live.back()] = tokens[from];
        } else if (what == 2) {
            const size_t i = any(live.size());
            book.release(live[i]);
            tokens.erase(live[i]);
            live.erase(live.begin() + i);
        } else if (what == 3) {
            const int s = live[any(live.size())];
            const size_t n = any(tokens[s].size() + 1);
            book.truncate(s, n);
            tokens[s].resize(n);
        } else if (what == 4) {
            apply(book.compact());
            for (int s : live)
                for (int32_t p : book.pages(s)) EXPECT_TRUE(size_t(p) < book.page_count() - book.free_pages());
        } else {
            std::vector<int> batch;
            std::vector<size_t> more;
            for (int s : live)
                if (any(3) == 0) {
                    batch.push_back(s);
                    more.push_back(any(6));
                }
            std::vector<PageBook::Copy> copies;
            try {
                book.extend(batch, more, copies);
            } catch (const RuntimeError &) {
                EXPECT_TRUE(copies.empty());
                continue;
            }
            apply(copies);
            for (size_t i = 0; i < batch.size(); ++i)
                for (size_t t = 0; t < more[i]; ++t) {
                    const int64_t slot = book.slot(batch[i], tokens[batch[i]].size());
                    pool[slot / 4][slot % 4] = next;
                    tokens[batch[i]].push_back(next++);
                }
        }
        std::set<int32_t> used;
        for (int s : live) {
            ASSERT_TRUE(book.length(s) == tokens[s].size());
            for (size_t t = 0; t < tokens[s].size(); ++t) {
                const int64_t slot = book.slot(s, t);
                ASSERT_TRUE(pool[slot / 4][slot % 4] == tokens[s][t]);
            }
            used.insert(book.pages(s).begin(), book.pages(s).end());
        }
        ASSERT_TRUE(used.size() + book.free_pages() == 40);
    }
}

// Groups of neighbours behind the pages that they share: no other division leaves fewer pages to read, by trying all of them
TEST(PageBook, GroupsReadTheFewestPages) {
    uint32_t r = 4242;
    auto any = [&](uint32_t n) {
        r = r * 1664525u + 1013904223u;
        return (r >> 12) % n;
    };
    for (int turn = 0; turn < 400; ++turn) {
        PageBook book(400, 2);
        std::vector<PageBook::Copy> copies;
        std::vector<int> batch;
        const size_t n = 1 + any(8);
        for (size_t i = 0; i < n; ++i) {
            if (i == 0 || any(4) == 0) {
                batch.push_back(book.add());
            } else { // another one's first tokens
                batch.push_back(book.fork(batch[any(3) ? any(i) : i - 1]));
                book.truncate(batch.back(), any(book.length(batch.back()) + 1));
            }
            book.extend({batch.back()}, {any(20)}, copies);
        }
        std::vector<size_t> more;
        for (size_t i = 0; i < n; ++i) more.push_back(1 + any(3));
        book.extend(batch, more, copies);
        auto whole = [&](size_t i) { return (book.length(batch[i]) - more[i]) / 2; }; // pages in front of the new tokens
        auto shared = [&](size_t from, size_t end) { // by all of [from, end); one by itself shares none
            if (end == from + 1) return size_t(0);
            size_t most = whole(from);
            for (size_t i = from + 1; i < end; ++i) {
                size_t same = 0;
                while (same < std::min(most, whole(i)) && book.pages(batch[i])[same] == book.pages(batch[from])[same]) ++same;
                most = same;
            }
            return most;
        };
        size_t most = 0; // pages that need not be read again
        for (uint32_t cuts = 0; cuts < 1u << (n - 1); ++cuts) {
            size_t saved = 0, from = 0;
            for (size_t end = 1; end <= n; ++end)
                if (end == n || (cuts >> (end - 1) & 1)) {
                    saved += (end - from - 1) * shared(from, end);
                    from = end;
                }
            most = std::max(most, saved);
        }
        size_t saved = 0, from = 0;
        for (const PageBook::Group &g : book.groups(batch, more)) {
            ASSERT_TRUE(g.end > from && g.end <= n);
            ASSERT_TRUE(g.pages == shared(from, g.end));
            ASSERT_TRUE(g.end == from + 1 || g.pages > 0);
            saved += (g.end - from - 1) * g.pages;
            from = g.end;
        }
        ASSERT_TRUE(from == n);
        ASSERT_TRUE(saved == most);
    }
    PageBook book(4, 2);
    EXPECT_TRUE(book.groups({}, {}).empty());
    EXPECT_THROW(book.groups({0}, {1}), IndexError);
}

// Extensions that are taken back leave no trace: pages, their users and the order in which free ones are taken are as before
TEST(PageBook, ExtensionsAreTakenBack) {
    PageBook book(40, 4), twin(40, 4);
    std::vector<int> live;
    uint32_t r = 777;
    auto any = [&](uint32_t n) {
        r = r * 1664525u + 1013904223u;
        return (r >> 12) % n;
    };
    for (int turn = 0; turn < 2000; ++turn) {
        const uint32_t what = any(8);
        if (what == 0 || live.empty()) {
            live.push_back(book.add());
            twin.add();
        } else if (what == 1) {
            const int from = live[any(live.size())];
            live.push_back(book.fork(from));
            twin.fork(from);
        } else if (what == 2) {
            const size_t i = any(live.size()), n = any(book.length(live[i]) + 1);
            book.truncate(live[i], n);
            twin.truncate(live[i], n);
        } else if (what == 3) {
            const size_t i = any(live.size());
            book.release(live[i]);
            twin.release(live[i]);
            live.erase(live.begin() + i);
        } else {
            std::vector<int> batch;
            std::vector<size_t> more;
            for (int s : live)
                if (any(3) == 0) {
                    batch.push_back(s);
                    more.push_back(any(6));
                }
            const bool keep = any(2) == 0;
            std::vector<PageBook::Copy> copies;
            try {
                book.extend(batch, more, copies);
            } catch (const RuntimeError &) {
                continue;
            }
            std::vector<PageBook::Copy> same;
            if (keep) twin.extend(batch, more, same);
            else book.take_back(batch, more, copies);
        }
        ASSERT_TRUE(book.free_pages() == twin.free_pages());
        for (int s : live) {
            ASSERT_TRUE(book.length(s) == twin.length(s));
            ASSERT_TRUE(book.pages(s) == twin.pages(s));
        }
    }
}

TEST(Cache, CpuTensorsAndMismatchesThrow) {
    const Tensor x = Tensor::zeros({2, 4, 8}), i = Tensor::zeros({2}, DType::Int32);
    EXPECT_THROW(ops::rotary(x, i, i), RuntimeError);
    EXPECT_THROW(ops::rotary(Tensor(), i, i), ValueError);
    EXPECT_THROW(ops::rotary_turns(3), ValueError);
    EXPECT_THROW(ops::packed_attention(x, x, x, i, i), RuntimeError);
    EXPECT_THROW(nn::PagedCache(1, 4, 3, 2, 8, DType::Float32), ValueError);
    EXPECT_THROW(nn::PagedCache(1, 4, 4, 2, 8, DType::Int32), TypeError);
    EXPECT_THROW(nn::PagedCache(0, 4, 4, 2, 8, DType::Float32), ValueError);
}

GPU_TEST(Cache, Rotary) {
    const std::vector<int64_t> positions{0, 1, 77, 5000, 123456, 9};
    const Tensor pos = Tensor::from_data(positions.data(), Shape{2, 3}, Device::GPU);
    for (DType dt : {DType::Float32, DType::Float16, DType::BFloat16})
        for (bool interleaved : {false, true}) {
            const Tensor x = axtest::randn({2, 3, 5, 24}, 3).astype(dt), turns = ops::rotary_turns(16, 1000.0);
            const Tensor y = ops::rotary(x.gpu(), pos, turns, interleaved);
            EXPECT_EQ(y.shape(), x.shape());
            EXPECT_EQ(y.dtype(), dt);
            const auto want = rotated(doubles(x), positions, 5, 24, 16, 1000.0, interleaved), got = doubles(y);
            // sines within 2^-22 and three roundings of 32 bits of two values below 5 each; the result's own rounding
            for (size_t k = 0; k < want.size(); ++k) EXPECT_NEAR(got[k], want[k], half_step(dt) * std::fabs(want[k]) + 10 * std::ldexp(1.0, -21) + 1e-7);
            const auto back = doubles(ops::rotary(y, pos, turns, interleaved, true)), was = doubles(x);
            for (size_t k = 0; k < was.size(); ++k) EXPECT_NEAR(back[k], was[k], 3 * half_step(dt) * 5 + 1e-5);
        }
    const Tensor g = axtest::randn({6, 5, 24}, 1).gpu(), turns = ops::rotary_turns(16);
    EXPECT_THROW(ops::rotary(g, ints({1, 2, 3}), turns), ShapeError);
    EXPECT_THROW(ops::rotary(g, axtest::randn({6}, 1).gpu(), turns), TypeError);
    EXPECT_THROW(ops::rotary(g, ints({0, 1, 2, 3, 4, 5}), ops::rotary_turns(26)), ShapeError);
    EXPECT_THROW(ops::rotary(g, ints({0, 1, 2, 3, 4, 5}), g), TypeError);
    ops::RotaryScaling bad;
    bad.kind = ops::RotaryScaling::Linear;
    bad.factor = 0;
    EXPECT_THROW(ops::rotary_turns(16, 10000.0, bad), ValueError);
    // a lazy input and a transposed view are settled first
    EXPECT_EQ(ops::rotary(ops::relu(g), ints({0, 1, 2, 3, 4, 5}), turns).shape(), (Shape{6, 5, 24}));
    EXPECT_EQ(ops::rotary(g.transpose({1, 0, 2}), ints({0, 1, 2, 3, 4}), turns).shape(), (Shape{5, 6, 24}));
}

GPU_TEST(Cache, PackedAttention) {
    const std::vector<int32_t> starts{0, 70, 71, 71, 200};
    for (DType dt : {DType::Float32, DType::Float16, DType::BFloat16})
        for (bool causal : {true, false}) {
            const size_t heads = 6, kv = 2, dim = 64;
            const Tensor q = axtest::randn({203, heads, dim}, 1).astype(dt), qkv = axtest::randn({203, 2 * kv, dim}, 2).astype(dt);
            const Tensor dev = qkv.gpu(), k = dev.slice({Slice(), Slice(0, kv), Slice()}), v = dev.slice({Slice(), Slice(kv, 2 * kv), Slice()});
            const Tensor o = ops::packed_attention(q.gpu(), k, v, ints(starts), ints(starts), causal);
            const auto got = doubles(o), qd = doubles(q), kd = doubles(k.ascontiguousarray()), vd = doubles(v.ascontiguousarray());
            for (size_t s = 0; s + 1 < starts.size(); ++s) {
                auto part = [&](const std::vector<double> &x, size_t h) { return std::vector<double>(x.begin() + starts[s] * h * dim, x.begin() + starts[s + 1] * h * dim); };
                const auto want = attention(part(qd, heads), part(kd, kv), part(vd, kv), heads, kv, dim, causal), mine = part(got, heads);
                for (size_t i = 0; i < want.size(); ++i) EXPECT_NEAR(mine[i], want[i], tolerance(dt));
            }
            for (size_t i = 200 * heads * dim; i < got.size(); ++i) EXPECT_EQ(got[i], 0.0); // rows that no sequence owns
        }
    const Tensor g = axtest::randn({10, 4, 8}, 1).gpu();
    EXPECT_THROW(ops::packed_attention(g, g, axtest::randn({10, 4, 16}, 1).gpu(), ints({0, 10}), ints({0, 10})), ShapeError);
    EXPECT_THROW(ops::packed_attention(g, axtest::randn({10, 3, 8}, 1).gpu(), axtest::randn({10, 3, 8}, 1).gpu(), ints({0, 10}), ints({0, 10})), ShapeError);
    EXPECT_THROW(ops::packed_attention(g, g, g, ints({0, 10}), ints({0, 5, 10})), ShapeError);
    EXPECT_THROW(ops::packed_attention(g, g.half(), g, ints({0, 10}), ints({0, 10})), TypeError);
    EXPECT_THROW(ops::packed_attention(g, g, g, g, ints({0, 10})), TypeError);
    EXPECT_THROW(ops::packed_attention(g, g, g, ints({0, 10}).reshape({1, 2}), ints({0, 10})), ShapeError);
}

// A decoder's day: prompts in chunks, forks that share their first pages, single tokens, sequences that leave, a pool that is compacted
GPU_TEST(Cache, PromptsForksAndSteps) {
    const size_t layers = 2, heads = 8, kv = 2, dim = 64, page = 16;
    for (DType dt : {DType::Float32, DType::BFloat16}) {
        nn::PagedCache cache(layers, 64, page, kv, dim, dt);
        const Tensor turns = ops::rotary_turns(dim);
        std::map<int, std::vector<std::vector<double>>> keys, values; // of each sequence and layer, rotated, as the cache has them
        uint64_t seed = 1;
        auto pass = [&](const std::vector<int> &seqs, const std::vector<size_t> &more) {
            const nn::CacheStep step = cache.extend(seqs, more);
            const std::vector<int64_t> positions = [&] {
                const Tensor p = step.positions.cpu();
                return std::vector<int64_t>(p.typed_data<int64_t>(), p.typed_data<int64_t>() + p.size());
            }();
            for (size_t layer = 0; layer < layers; ++layer) {
                const Tensor qkv = axtest::randn({step.tokens, heads + 2 * kv, dim}, seed++).astype(dt), dev = qkv.gpu();
                auto part = [&](size_t from, size_t to) { return dev.slice({Slice(), Slice(from, to), Slice()}); };
                const Tensor q = cache.append(layer, step, part(0, heads), part(heads, heads + kv), part(heads + kv, heads + 2 * kv), turns);
                const Tensor o = cache.attend(layer, step, q);
                const auto qd = doubles(q), od = doubles(o), vd = doubles(part(heads + kv, heads + 2 * kv).ascontiguousarray());
                const auto want_q = rotated(doubles(part(0, heads).ascontiguousarray()), positions, heads, dim, dim, 10000.0, false);
                Tensor kr(Shape{step.tokens, kv, dim}, DType::Float32);
                const auto want_k = rotated(doubles(part(heads, heads + kv).ascontiguousarray()), positions, kv, dim, dim, 10000.0, false);
                for (size_t i = 0; i < want_k.size(); ++i) kr.typed_data<float>()[i] = static_cast<float>(want_k[i]);
                const auto kd = doubles(kr.astype(dt)); // (as the cache holds them, a rounding's border aside)
                for (size_t i = 0; i < qd.size(); ++i) EXPECT_NEAR(qd[i], want_q[i], half_step(dt) * std::fabs(want_q[i]) + 1e-5);
                size_t at = 0;
                for (size_t s = 0; s < seqs.size(); ++s) {
                    auto &ks = keys[seqs[s]], &vs = values[seqs[s]];
                    ks.resize(layers);
                    vs.resize(layers);
                    ks[layer].insert(ks[layer].end(), kd.begin() + at * kv * dim, kd.begin() + (at + more[s]) * kv * dim);
                    vs[layer].insert(vs[layer].end(), vd.begin() + at * kv * dim, vd.begin() + (at + more[s]) * kv * dim);
                    const std::vector<double> mine(qd.begin() + at * heads * dim, qd.begin() + (at + more[s]) * heads * dim);
                    const auto want = attention(mine, ks[layer], vs[layer], heads, kv, dim, true);
                    // (a key next to a rounding's border may differ by a step in one of its dims: a score by 5 * 2 half steps of 5 / 8, a weight by as much)
                    for (size_t i = 0; i < want.size(); ++i) EXPECT_NEAR(od[at * heads * dim + i], want[i], 3 * tolerance(dt));
                    at += more[s];
                }
            }
            return step;
        };
        const int a = cache.add(), b = cache.add();
        pass({a, b}, {37, 5});
        pass({a, b}, {20, 1});
        const int c = cache.fork(a), d = cache.fork(a);
        for (int s : {c, d}) {
            keys[s] = keys[a];
            values[s] = values[a];
        }
        auto step = pass({a, c, d, b}, {1, 1, 1, 1}); // three of them begin with the same 48 tokens
        EXPECT_EQ(step.longest_prefix, size_t(48));
        EXPECT_EQ(step.prefix_lengths.size(), size_t(2));
        for (int turn = 0; turn < 8; ++turn) pass({a, c, d, b}, {1, 1, 1, 1});
        pass({d, a}, {2, 2});
        cache.release(a);
        EXPECT_TRUE(cache.compact() > 0);
        pass({c, d}, {1, 1});
        pass({b, d, c}, {7, 1, 3});
        cache.truncate(c, 40);
        for (size_t layer = 0; layer < layers; ++layer) {
            keys[c][layer].resize(40 * kv * dim);
            values[c][layer].resize(40 * kv * dim);
        }
        pass({c, d}, {1, 1});
        EXPECT_EQ(cache.length(c), size_t(41));
        EXPECT_THROW(cache.length(a), IndexError);
        EXPECT_THROW(cache.extend({c}, {0}), ValueError);
        EXPECT_THROW(cache.extend({}, {}), ValueError);
        EXPECT_THROW(cache.extend({c}, {2000}), RuntimeError);
        const auto last = cache.extend({c}, {1});
        const Tensor q = axtest::randn({1, heads, dim}, 1).astype(dt).gpu(), k = axtest::randn({1, kv, dim}, 1).astype(dt).gpu();
        EXPECT_THROW(cache.append(layers, last, q, k, k), IndexError);
        EXPECT_THROW(cache.append(0, last, q, q, k), ShapeError);
        EXPECT_THROW(cache.append(0, last, q, k, axtest::randn({2, kv, dim}, 1).astype(dt).gpu()), ShapeError);
        EXPECT_THROW(cache.append(0, last, q, k, k, q), TypeError);
        EXPECT_THROW(cache.attend(0, last, axtest::randn({1, 3, dim}, 1).astype(dt).gpu()), ShapeError);
        EXPECT_THROW(cache.attend(layers, last, q), IndexError);
        EXPECT_THROW(cache.attend(0, step, q), ValueError); // the sequences have changed since
        EXPECT_THROW(cache.append(0, nn::CacheStep(), q, k, k), ValueError);
        EXPECT_THROW(nn::PagedCache(layers, 64, page, kv, dim, dt).attend(0, last, q), ValueError);
        EXPECT_THROW(cache.attend(0, last, q.astype(DType::Float16)), TypeError);
    }
}

// Device work that fails (copies of 2^20 layers are refused on the host, before any launch) leaves the book and the steps as they were
GPU_TEST(Cache, FailedCopiesChangeNothing) {
    nn::PagedCache cache(size_t(1) << 20, 4, 2, 1, 1, DType::Float32);
    const Tensor x = axtest::randn({1, 1, 1}, 1).gpu();
    const int a = cache.add();
    const nn::CacheStep step = cache.extend({a}, {1});
    const int b = cache.fork(a);
    EXPECT_THROW(cache.extend({a, b}, {2, 3}), DeviceError); // one of them is to copy the page that both have
    for (int s : {a, b}) {
        EXPECT_EQ(cache.length(s), size_t(1));
        EXPECT_TRUE(cache.book().pages(s) == (std::vector<int32_t>{0}));
    }
    EXPECT_EQ(cache.book().free_pages(), size_t(3));
    EXPECT_EQ(cache.append(5, step, x, x, x).shape(), x.shape()); // the step is as good as before
    const int c = cache.add();
    cache.extend({c}, {1});
    cache.release(a);
    cache.release(b);
    const nn::CacheStep more = cache.extend({c}, {1});
    EXPECT_THROW(cache.compact(), DeviceError); // page 1 is to move to the place of page 0
    EXPECT_EQ(cache.length(c), size_t(2));
    EXPECT_TRUE(cache.book().pages(c) == (std::vector<int32_t>{1}));
    EXPECT_EQ(cache.book().free_pages(), size_t(3));
    EXPECT_EQ(cache.append(5, more, x, x, x).shape(), x.shape());
    const int d = cache.add();
    cache.extend({d}, {6});
    EXPECT_TRUE(cache.book().pages(d) == (std::vector<int32_t>{0, 2, 3}));
}

// A neighbour that shares little does not take their long prefix from the others, wherever it stands
GPU_TEST(Cache, PrefixesOfUnequalNeighbours) {
    const size_t page = 16, kv = 2, dim = 64;
    nn::PagedCache cache(1, 64, page, kv, dim, DType::BFloat16);
    const int deep = cache.add();
    cache.extend({deep}, {20 * page});
    const int other = cache.fork(deep);
    cache.truncate(other, page); // the first page only
    cache.extend({other}, {5 * page});
    const int second = cache.fork(deep), third = cache.fork(deep);
    auto lengths = [&](const nn::CacheStep &step) {
        const Tensor p = step.prefix_lengths.cpu();
        return std::vector<int32_t>(p.typed_data<int32_t>(), p.typed_data<int32_t>() + p.size());
    };
    const int32_t long_one = 20 * page;
    EXPECT_TRUE(lengths(cache.extend({deep, second, third, other}, {1, 1, 1, 1})) == (std::vector<int32_t>{long_one, 0}));
    EXPECT_TRUE(lengths(cache.extend({other, third, second, deep}, {1, 1, 1, 1})) == (std::vector<int32_t>{0, long_one}));
    EXPECT_TRUE(lengths(cache.extend({second, other, third, deep}, {1, 1, 1, 1})) == (std::vector<int32_t>{16, long_one}));
    const int sixth = cache.fork(other);
    EXPECT_TRUE(lengths(cache.extend({other, sixth, third, deep}, {1, 1, 1, 1})) == (std::vector<int32_t>{6 * 16, long_one}));
}

// Without longest_keys the division of the work goes by the number of sequences too, not as though each had all keys
GPU_TEST(Cache, PackedAttentionWithoutAHint) {
    auto kernel_of = [](size_t sequences, size_t each, size_t heads, size_t kv, size_t dim, size_t hint) {
        std::vector<int32_t> starts;
        for (size_t i = 0; i <= sequences; ++i) starts.push_back(static_cast<int32_t>(i * each));
        const Tensor q = axtest::randn({sequences * each, heads, dim}, 1).bfloat16().gpu(), k = axtest::randn({sequences * each, kv, dim}, 2).bfloat16().gpu();
        ops::packed_attention(q, k, k, ints(starts), ints(starts), true, -1.0f, hint);
        return std::string(axhip_sdpa_cache_last_kernel());
    };
    EXPECT_EQ(kernel_of(20, 60, 8, 8, 64, 60), std::string("tile"));
    EXPECT_EQ(kernel_of(20, 60, 8, 8, 64, 0), std::string("tile"));
    EXPECT_EQ(kernel_of(64, 256, 32, 8, 128, 256), std::string("tile"));
    EXPECT_EQ(kernel_of(64, 256, 32, 8, 128, 0), std::string("tile"));
    EXPECT_EQ(kernel_of(1, 4096, 32, 8, 128, 0), std::string("tile, eight waves")); // (one sequence has them all)
}
