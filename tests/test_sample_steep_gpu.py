"""Rows of which fewer logits weigh anything than top_k asks for: small temperatures, masks, infinities.  Tokens as in the definition in 64 bits."""
import numpy as np
import pytest
import torch

from tests import q8_harness as q8

pytestmark = pytest.mark.gpu


def check(logits, dt, u, temperature, top_k, top_p=1.0, min_p=0.0):
    tokens, probs = q8.sample(logits, dt, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    l, told = q8.f64(logits), 0
    for i in range(len(l)):
        token, prob, margin = q8.sampled(l[i], float(u[i]), float(np.float32(temperature)), top_k, top_p, min_p)
        if margin > 1e-9:
            assert tokens[i] == token, (i, temperature, top_k)
            assert abs(probs[i] - prob) <= 1e-6 * prob + 1e-12
            told += 1
    assert told >= len(l) - 1


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1100, 5003, 8192, 51865, 140001])
def test_small_temperatures(dt, vocab):
    gen = torch.Generator()
    gen.manual_seed(vocab)
    logits = (torch.randn(6, vocab, generator=gen) * 2.5).to(q8.DTYPES[dt][1]).cuda()
    u = torch.rand(6, generator=gen)
    for temperature in (1e-3, 0.02, 0.05, 0.1, 0.2):
        for top_k in (1, 50, 512):
            check(logits, dt, u, temperature, top_k)
        check(logits, dt, u, temperature, 200, 0.9, 0.01)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("left", [1, 2, 49, 50, 51, 63, 64, 65, 1023, 1024, 1025, 3000])
def test_few_that_are_left(dt, left):
    """All but `left` logits masked by -infinity, NaN, the lowest number or 40 temperatures below the rest."""
    gen = torch.Generator()
    gen.manual_seed(left)
    vocab = 20000
    logits = torch.full((6, vocab), -float("inf"))
    logits[1], logits[2], logits[3] = float("nan"), torch.finfo(q8.DTYPES[dt][1]).min, -40.0
    for row in range(6):
        at = torch.randperm(vocab, generator=gen)[:left]
        logits[row, at] = torch.randn(left, generator=gen) if row != 4 else torch.full((left,), float("inf"))
    logits = logits.to(q8.DTYPES[dt][1]).cuda()
    u = torch.rand(6, generator=gen)
    for top_k in (50, 512):
        check(logits, dt, u, 1.0, top_k)
        check(logits, dt, u, 1.0, top_k, 0.7)
    check(logits, dt, u, 1.0, 64, 1.0, 0.3)
