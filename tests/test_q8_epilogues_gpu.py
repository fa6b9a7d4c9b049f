"""What the products in 8 bits do behind the sum: rows that are not finite under every activation, and the activations themselves over the whole range of a 16-bit result."""
import numpy as np
import pytest
import torch

from tests import q8_harness as q8

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "gelu", "silu", "sigmoid", "tanh"]
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def int8s(seed, *shape):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return torch.randint(-127, 128, shape, generator=gen, dtype=torch.int8).cuda()


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 130, 256), (2, 130, 255), (20, 131, 256), (400, 130, 256), (300, 1030, 640), (300, 1030, 643), (1300, 1630, 256), (7, 30, 9)])
def test_a_row_that_is_not_a_number_stays_one(m, n, k, act, dt):
    a, b = int8s(m, m, k), int8s(n, n, k)
    sa, sb = torch.full((m,), 0.01, device="cuda"), torch.full((n,), 0.01, device="cuda")
    want, _ = q8.gemm(a, b, sa, sb, dt, act=act)
    assert not bool(torch.isnan(want).any())
    row, col = m // 2, n - 2
    sa[row] = float("nan")  # (what axhip_quantize_q8 and axhip_rms_norm_q8 give to a row with an infinity)
    sb[col] = float("nan")
    c, kernel = q8.gemm(a, b, sa, sb, dt, act=act)
    nan = torch.isnan(c)
    assert bool(nan[row].all()) and bool(nan[:, col].all()), kernel
    nan[row], nan[:, col] = True, True
    assert torch.equal(torch.where(nan, want, c), want)


def test_a_token_that_overflowed_is_seen_behind_the_activation():
    """f16 activations of which one token holds an infinity, through the first product of a feed-forward block."""
    gen = torch.Generator()
    gen.manual_seed(1)
    x = torch.randn(5, 512, generator=gen).half().cuda()
    x[3, 100] = float("inf")
    q, scales = q8.quantize(x, "f16")
    w, ws = q8.quantize(torch.randn(300, 512, generator=gen).half().cuda(), "f16")
    c, _ = q8.gemm(q, w, scales, ws, "f16", act="relu")
    assert torch.isnan(c).any(1).tolist() == [False, False, False, True, False] and bool(torch.isnan(c[3]).all())


# ---- one product is one number: row i of A holds a one, column j of B holds an integer, their scales the rest
def through(act, dt, m):
    k = 64
    a, b = torch.zeros(m, k, dtype=torch.int8), torch.zeros(255, k, dtype=torch.int8)
    a[:, 5] = 1
    b[:, 5] = torch.arange(-127, 128)
    sa = torch.ldexp(torch.ones(m), torch.linspace(-24, -3, m).round().int()) * torch.linspace(1.0, 1.9, m)
    one = torch.ones(255)
    c, _ = q8.gemm(a.cuda(), b.cuda(), sa.cuda(), one.cuda(), dt, act=act)
    x = torch.outer(sa, torch.arange(-127, 128).float())  # (what fp32 makes of the sum and its scales)
    return q8.f64(c), x.double()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid", "tanh"])
@pytest.mark.parametrize("m", [1, 2, 40, 600])
def test_sixteen_bit_activations_are_rounded_once(act, dt, m):
    """|x| from 6e-8 to 30.  Before the rounding an activation is near its value.  GELU: its fit is off by 2^-18.2 (f16) or 2^-13.0 (bf16) of itself, nine roundings of an exponent of up to 32 (f16)
    or 128 (bf16) are 9 * 2^-24 * 32 ln 2 = 2^-16.4 or 2^-14.4 at most, all together below 2^-15 and 2^-12; bf16 results below 2^-122 may be zero (a factor that is flushed below
    2^-126 times |x| < 2^4).  The others: the exponent's roundings (30 times 2^-23) and half a dozen of 2^-24, below 2^-15."""
    got, x = through(act, dt, m)
    y = {"gelu": lambda: x * 0.5 * torch.special.erfc(-x / 2**0.5), "silu": lambda: x * torch.sigmoid(x), "sigmoid": lambda: torch.sigmoid(x), "tanh": lambda: torch.tanh(x)}[act]().numpy()
    least = {"f16": 2.0**-14, "bf16": 2.0**-126}[dt]  # (of the subnormal ones a step is that of the smallest normal)
    off = np.abs(got - y)
    allowed = HALF_STEP[dt] * np.maximum(np.abs(y), least) * 1.001 + 2.0**-15 * np.abs(y)
    if act == "gelu" and dt == "bf16":
        allowed += 2.0**-12 * np.abs(y) + 2.0**-122
    assert np.all(off <= allowed), (float((off / allowed).max()), float(x.flatten()[(off / allowed).argmax()]))
