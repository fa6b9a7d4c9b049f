"""The RMS norm's scale where the squares leave fp32's range: sums of squares above 2^128 and below 2^-149.

The largest magnitude and the sum of squares are held exactly enough in 64 bits; the root and its reciprocal, the product with the largest, the division by 127 and the last conversion
are roundings of 2^-24 each, the root's argument adds half of one: six at most.  (A scale below fp32's normal numbers is off by half of 2^-149 besides.)"""
import numpy as np
import pytest
import torch

from tests import q8_harness as q8

pytestmark = pytest.mark.gpu


def rows(seed, n, cols, exponent, dt):
    gen = torch.Generator()
    gen.manual_seed(seed)
    x = torch.ldexp(torch.randn(n, cols, generator=gen, dtype=torch.float64), torch.tensor(exponent))
    return x.to(q8.DTYPES[dt][1]).cuda()


def check(q, scales, h, w, eps):
    y = h if w is None else h * w
    largest, want = q8.nearest(y)
    expected = largest / 127 / np.sqrt((h * h).mean(-1) + np.float64(np.float32(eps)))
    assert np.all(np.isfinite(expected)) and np.all(expected > 0)
    assert np.array_equal(q.cpu().numpy(), want)
    assert np.all(np.abs(scales.cpu().double().numpy() - expected) <= 6 * 2.0**-24 * expected + 2.0**-150)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 200, 1280, 20000, 70000])
@pytest.mark.parametrize("exponent", [50, 63, 64, 70, 100, 120])
def test_large_rows(dt, cols, exponent):
    x = rows(cols, 3, cols, exponent, dt)
    q, scales, _ = q8.rms_norm(x, None, None, dt)
    check(q, scales, q8.f64(x), None, 1e-5)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1, 200, 1280, 20000, 70000])
@pytest.mark.parametrize("exponent", [-120, -100, -80, -70, -60, -40])
def test_small_rows_without_eps(dt, cols, exponent):
    x = rows(cols, 3, cols, exponent, dt)
    q, scales, _ = q8.rms_norm(x, None, None, dt, eps=0.0)
    check(q, scales, q8.f64(x), None, 0.0)


@pytest.mark.parametrize("cols", [300, 70000])
@pytest.mark.parametrize("h,w", [(-100, -60), (-60, -100), (60, -120), (90, 30), (-90, 100)])
def test_products_beyond_and_within_fp32(cols, h, w):
    """fp32 rows and a weight whose products lie below fp32's numbers, the normalised ones within them."""
    x, weight = rows(cols, 3, cols, h, "f32"), rows(cols + 1, 1, cols, w, "f32")[0]
    q, scales, _ = q8.rms_norm(x, None, weight, "f32", eps=0.0)
    check(q, scales, q8.f64(x), q8.f64(weight), 0.0)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [300, 70000])
def test_a_large_row_stays_by_itself(dt, cols):
    """Its neighbours, and the sum with a residual, are those of ordinary rows; a row of zeros keeps scale 0, whatever eps."""
    x, r = rows(1, 4, cols, 0, dt), rows(2, 4, cols, 0, dt)
    plain, s0, _ = q8.rms_norm(x, r, None, dt)
    x[1], r[1] = x[1] * 2.0**80, r[1] * 2.0**80
    x[2], r[2] = 0, 0
    q, scales, total = q8.rms_norm(x, r, None, dt)
    h = (x.float() + r.float()).to(x.dtype)
    assert torch.equal(total, h)
    for row in (0, 3):
        assert torch.equal(q[row], plain[row]) and scales[row] == s0[row]
    assert scales[2] == 0 and not bool(q[2].any())
    check(q[1:2], scales[1:2], q8.f64(h[1:2]), None, 1e-5)
