"""Sampling against its definition in 64 bits.  Tokens are compared for equality wherever the random number is not within 1e-9 of the sum from a border of two
tokens (weights are held to 2^-44 of the largest: 2^20 of them are off by less than 2^-24 only if all errors had one sign; 1e-9 is 50 times what random signs
give); the probability is fp32 of a quotient of such sums."""
import ctypes as C

import numpy as np
import pytest
import torch

from axiom_amd import capi
from tests import q8_harness as q8

pytestmark = pytest.mark.gpu


def logits_of(seed, rows, vocab, dt, scale=2.5):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen) * scale).to(q8.DTYPES[dt][1]).cuda(), torch.rand(rows, generator=gen).clamp(max=1 - 2.0**-24)


def check(logits, dt, u, **settings):
    rows = logits.shape[0]
    tokens, probs = q8.sample(logits, dt, u, **settings)
    l = q8.f64(logits)
    told = 0
    for i in range(rows):
        mine = {k: (float(torch.as_tensor(v, dtype=torch.float32).expand(rows)[i]) if k != "top_k" else int(torch.as_tensor(v).expand(rows)[i])) for k, v in settings.items()}
        token, prob, margin = q8.sampled(l[i], float(torch.as_tensor(u, dtype=torch.float32).expand(rows)[i]), **mine)
        if margin > 1e-9:
            assert tokens[i] == token, (i, mine)
            assert abs(probs[i] - prob) <= 1e-6 * prob + 1e-12, (i, probs[i], prob)
            told += 1
    assert told >= rows - 1
    return tokens


VOCABS = [1, 2, 7, 64, 511, 512, 513, 1000, 8191, 8192, 10007, 32000, 51865, 100001, 131072, 131080, 200003]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", VOCABS)
def test_every_filter(dt, vocab):
    logits, u = logits_of(vocab, 3, vocab, dt)
    check(logits, dt, u)
    check(logits, dt, u, temperature=0.7)
    check(logits, dt, u, top_k=[1, 50, 1000])
    check(logits, dt, u, top_p=[0.5, 0.9, 0.99], temperature=1.3)
    check(logits, dt, u, min_p=[0.01, 0.1, 1.0])
    check(logits, dt, u, temperature=[0.5, 1.0, 2.0], top_k=[40, 0, 7], top_p=[0.9, 0.8, 1.0], min_p=[0.0, 0.05, 0.02])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 17, 300])
def test_rows_with_settings_of_their_own(dt, rows):
    logits, u = logits_of(rows, rows, 3001, dt)
    gen = torch.Generator()
    gen.manual_seed(rows)
    check(logits, dt, u, temperature=torch.rand(rows, generator=gen) * 1.5, top_k=torch.randint(-1, 60, (rows,), generator=gen, dtype=torch.int32),
          top_p=torch.rand(rows, generator=gen) * 1.1, min_p=torch.rand(rows, generator=gen) * 0.2 - 0.05)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [600, 5000, 140000])
def test_equal_logits_are_kept_by_index(dt, vocab):
    """Few distinct values: every border lies inside a run of equal logits."""
    gen = torch.Generator()
    gen.manual_seed(vocab)
    logits = torch.randint(0, 4, (6, vocab), generator=gen).to(q8.DTYPES[dt][1]).cuda()
    u = torch.rand(6, generator=gen)
    check(logits, dt, u, top_k=[1, 3, vocab // 4, vocab // 3, vocab // 2, vocab - 1])
    check(logits, dt, u, top_k=[1, 3, vocab // 4, vocab // 3, vocab // 2, vocab - 1], top_p=0.61803)
    check(logits, dt, u, top_p=[0.001, 0.1, 0.3, 0.7, 0.9, 0.99991])


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [100, 20000])
def test_masked_logits_are_never_drawn(dt, vocab):
    logits, u = logits_of(3, 8, vocab, dt)
    logits[:, ::2] = -float("inf")
    logits[1, 1::4] = float("nan")
    logits[2] = -float("inf")
    logits[3] = float("nan")
    logits[4, 5], logits[4, 7] = float("inf"), float("inf")
    lowest = torch.finfo(logits.dtype).min
    logits[5] = lowest
    logits[6, 1:] = lowest
    for settings in ({}, dict(top_k=5), dict(top_p=0.9), dict(min_p=0.5), dict(top_k=vocab - 1, top_p=0.5, temperature=0.9)):
        tokens = check(logits, dt, u, **settings)
        assert tokens[2] == -1 and tokens[3] == -1 and tokens[4] in (5, 7) and tokens[0] % 2 == 1
    tokens, probs = q8.sample(logits, dt, u)
    assert probs[2] == 0 and probs[3] == 0 and probs[4] == 0.5


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_no_temperature_is_the_first_largest(dt):
    logits, u = logits_of(4, 5, 9000, dt)
    logits[0, [40, 8000]] = 30.0
    logits[1, 8999] = 40.0
    logits[2] = float("nan")
    tokens, probs = q8.sample(logits, dt, u, temperature=[0.0, -1.0, 0.0, float("nan"), 0.0], top_k=1, top_p=0.3)
    assert tokens.tolist() == [40, 8999, -1, int(torch.argmax(logits[3].float())), int(torch.argmax(logits[4].float()))]
    assert probs.tolist() == [1, 1, 0, 1, 1]


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [300, 51865])
def test_the_ends_of_the_random_numbers(dt, vocab):
    logits, _ = logits_of(5, 4, vocab, dt)
    l = q8.f64(logits)
    tokens, _ = q8.sample(logits, dt, [0.0, -1.0, float("nan"), 0.0], top_k=20)
    first = [min(np.argsort(-l[i], kind="stable")[:20]) for i in range(4)]
    assert tokens.tolist() == first
    tokens, _ = q8.sample(logits, dt, [1.0, 1 - 2.0**-24, 5.0, float("inf")], top_k=20)
    assert tokens.tolist() == [max(np.argsort(-l[i], kind="stable")[:20]) for i in range(4)]


def test_extreme_temperatures():
    logits, u = logits_of(6, 4, 4000, "f32")
    tokens = check(logits, "f32", u, temperature=[1e-30, 1e30, 1e-3, 50.0])
    assert tokens[0] == int(torch.argmax(logits[0]))


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,ld,offset", [(1000, 1000, 1), (8193, 8193, 0), (51865, 51872, 3), (131073, 131075, 1)])
def test_rows_apart_and_off_the_grid(dt, vocab, ld, offset):
    big, u = logits_of(vocab, 1, 3 * ld + offset, dt)
    logits = big[0, offset:].view(3, ld)[:, :vocab]
    check(logits, dt, u, top_k=100, top_p=0.95)
    check(logits, dt, u)


def test_frequencies_follow_the_probabilities():
    """4096 random numbers spread evenly: every token as often as its probability says, to within one."""
    logits = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]]).expand(4096, 5).contiguous().cuda()
    tokens, _ = q8.sample(logits, "f32", (torch.arange(4096) + 0.5) / 4096, top_k=4)
    w = np.exp(np.array([0.0, 1.0, -np.inf, 2.0, 0.5]))
    assert np.all(np.abs(np.bincount(tokens, minlength=5) - 4096 * w / w.sum()) <= 1)


def test_the_same_call_gives_the_same_tokens_and_no_probabilities_are_asked_for():
    logits, u = logits_of(8, 40, 51865, "bf16")
    settings = dict(temperature=0.9, top_k=300, top_p=0.97, min_p=0.001)
    tokens, probs = q8.sample(logits, "bf16", u, **settings)
    for _ in range(3):
        again, p = q8.sample(logits, "bf16", u, **settings)
        assert np.array_equal(tokens, again) and np.array_equal(probs, p)
    again, p = q8.sample(logits, "bf16", u, want_probs=False, **settings)
    assert np.array_equal(tokens, again) and p is None


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("values", [1, 2, 3])
def test_more_than_65535_equal_logits(dt, values):
    gen = torch.Generator()
    gen.manual_seed(values)
    vocab = 140003 if values < 3 else 230001
    logits = torch.randint(0, values, (4, vocab), generator=gen).to(q8.DTYPES[dt][1]).cuda()
    u = torch.rand(4, generator=gen)
    check(logits, dt, u, top_p=[0.2, 0.618, 0.9, 0.98])
    check(logits, dt, u, top_k=[700, 70000, 100001, vocab - 1])
    check(logits, dt, u, top_k=[700, 70000, 100001, vocab - 1], top_p=0.71)
    check(logits, dt, u, temperature=0.5, min_p=0.3)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [4000, 51865])
def test_top_k_of_every_size(dt, vocab):
    ks = [2, 64, 127, 128, 129, 300, 511, 512, 513, 1024, 3000, vocab // 2, vocab - 1, vocab, vocab + 7, 2**31 - 1]
    logits, u = logits_of(vocab + 1, len(ks), vocab, dt)
    check(logits, dt, u, top_k=ks)
    check(logits, dt, u, top_k=ks, top_p=0.93, temperature=1.5)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-4, 0.02, 0.3, 40.0, 3000.0])
@pytest.mark.parametrize("shift", [0.0, -500.0, 3000.0])
def test_flat_and_steep_logits(dt, scale, shift):
    """From rows whose every token is as likely as any other to rows with one that is; far from zero, where the type leaves few values."""
    logits, u = logits_of(5, 6, 30000, dt, scale)
    logits = (logits.float() + shift).clamp(-6e4, 6e4).to(logits.dtype)
    check(logits, dt, u)
    check(logits, dt, u, top_p=[0.1, 0.5, 0.9, 0.95, 0.99, 0.9999])
    check(logits, dt, u, top_p=[0.1, 0.5, 0.9, 0.95, 0.99, 0.9999], temperature=[0.05, 0.3, 3.0, 20.0, 500.0, 1.0], min_p=0.001)
    check(logits, dt, u, top_k=[1, 10, 100, 500, 5000, 29999], temperature=[0.05, 0.3, 3.0, 20.0, 500.0, 1.0])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_the_largest_vocabulary(dt):
    logits, u = logits_of(7, 2, 1 << 20, dt)
    check(logits, dt, u)
    check(logits, dt, u, top_k=[40, 2000], top_p=0.9)
    check(logits, dt, u, top_p=[0.6, 0.97])


def test_many_short_rows():
    logits, u = logits_of(8, 3000, 37, "bf16")
    check(logits, "bf16", u, top_k=9, top_p=0.8)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_masked_halves_and_infinities_under_every_filter(dt):
    """Rows of 60000 of which most are masked by -inf, NaN or the lowest number, and rows with infinite logits."""
    logits, u = logits_of(9, 6, 60000, dt)
    lowest = torch.finfo(logits.dtype).min
    logits[0, 100:] = -float("inf")
    logits[1, :59900] = float("nan")
    logits[2, 50:] = lowest
    logits[3, ::2] = float("nan")
    logits[4, [7, 50000, 59999]] = float("inf")
    logits[5] = lowest
    for settings in ({}, dict(top_k=3), dict(top_k=700), dict(top_p=0.9), dict(min_p=0.2), dict(top_k=1000, top_p=0.7, min_p=0.01)):
        tokens = check(logits, dt, u, temperature=0.8, **settings)
        assert tokens[0] < 100 and tokens[1] >= 59900 and tokens[2] < 50 and tokens[3] % 2 == 1 and tokens[4] in (7, 50000, 59999)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("equal", [1, 63, 64, 65, 127, 128, 129, 255, 257, 511, 512, 513, 1023, 1024, 1025, 5000, 19997])
def test_any_number_of_largest_logits(dt, equal):
    """`equal` of them, anywhere in the row: all of them reach the bound of a small top_k."""
    vocab = 20000
    gen = torch.Generator()
    gen.manual_seed(equal)
    logits, u = logits_of(equal, 5, vocab, dt, 1.0)
    logits = logits.clamp(max=2.0)
    for row in range(5):
        logits[row, torch.randperm(vocab, generator=gen)[:equal].cuda()] = 4.0
    ks = [1, 2, 100, 300, 512]
    check(logits, dt, u, top_k=ks)
    check(logits, dt, u, top_k=ks, top_p=[0.5, 0.9, 0.3, 0.75, 0.98], min_p=0.1)
    check(logits, dt, u, top_p=[0.5, 0.9, 0.3, 0.75, 0.98], temperature=0.5)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [3, 64, 65, 200, 1000, 1023, 1024, 1025, 2000])
def test_short_rows_under_every_filter(dt, vocab):
    logits, u = logits_of(vocab, 4, vocab, dt)
    logits[1] = logits[1].round()
    logits[2, vocab // 2:] = -float("inf")
    check(logits, dt, u, top_k=[vocab, vocab // 2, 1 + vocab // 3, 2], top_p=[0.99, 0.9, 0.5, 0.7])
    check(logits, dt, u, top_p=[0.0, 1e-7, 0.4, 1.0 - 2.0**-24], min_p=[0.0, 0.5, 0.0, 1e-3])


def test_settings_that_are_not_numbers():
    """temperature NaN is 0; of the others NaN is off."""
    nan = float("nan")
    logits, u = logits_of(3, 4, 5000, "bf16")
    largest = logits.float().argmax(1).cpu()
    tokens, probs = q8.sample(logits, "bf16", u, temperature=[nan, 0.0, -1.0, nan])
    assert list(tokens) == largest.tolist() and all(p == 1.0 for p in probs)
    want, _ = q8.sample(logits, "bf16", u)
    got, _ = q8.sample(logits, "bf16", u, top_p=nan, min_p=nan)
    assert list(got) == list(want)


def test_calls_on_two_streams_at_once():
    lib = capi.lib()
    cases, calls = [(1, "f32", dict(top_k=60)), (70, "bf16", dict(top_p=0.9)), (260, "f16", dict(top_k=700, top_p=0.8)), (33, "f32", dict(top_p=0.95))], []
    for rows, dt, settings in cases:
        logits, u = logits_of(rows, rows, 40001, dt)
        want, _ = q8.sample(logits, dt, u, **settings)
        on = {k: torch.full((rows,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in settings.items()}
        u, tokens = u.cuda(), torch.empty(rows, dtype=torch.int64, device="cuda")
        calls.append((logits, q8.sample_params(logits, dt, u, **on), tokens, want, on, u))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    q8.sync()
    for _ in range(5):
        for i, (logits, p, tokens, _, _, _) in enumerate(calls):
            capi.check(lib.axhip_sample(q8.at(logits), q8.at(tokens), None, C.byref(p), streams[i % 2].cuda_stream))
    torch.cuda.synchronize()
    for _, _, tokens, want, _, _ in calls:
        assert tokens.tolist() == list(want)
