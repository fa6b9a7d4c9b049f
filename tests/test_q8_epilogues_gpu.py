"""What the products in 8 bits do behind the sum: rows that are not finite under every activation."""
import pytest
import torch

from tests import q8_harness as q8

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "gelu", "silu", "sigmoid", "tanh"]


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
