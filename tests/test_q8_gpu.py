"""Rows in 8 bits, the RMS norm that ends in them, and products of them, against their definitions in 64 bits.

Integers are compared for equality: which one is nearest is decided on exact products.  Scales are fp32: the largest magnitude is exact, the
sum of n squares of a row is added up by at least 64 threads (sequences of n / 64 + 16 additions at most), and four more roundings follow."""
import ctypes as C

import numpy as np
import pytest
import torch

from axiom_amd import capi
from tests import q8_harness as q8

pytestmark = pytest.mark.gpu
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def normal(seed, *shape, scale=1.0, shift=0.0, dt="bf16"):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale + shift).to(q8.DTYPES[dt][1]).cuda()


def int8s(seed, *shape):
    gen = torch.Generator()
    gen.manual_seed(seed)
    return torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8).cuda()


def check_rows(q, scales, y, factor, cols, norm):
    largest, want = q8.nearest(y)
    assert np.array_equal(q.cpu().numpy(), want)
    want_scales = np.where(np.isfinite(largest), largest * factor / 127, np.nan)
    tolerance = (4 + (cols / 64 + 16) / 2 if norm else 2) * 2.0**-24  # (half of the sum's: its root is taken)
    got = scales.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want_scales))
    fine = ~np.isnan(got)
    assert np.all(np.abs(got[fine] - want_scales[fine]) <= tolerance * want_scales[fine])


COLS = [1, 7, 8, 63, 512, 513, 1000, 1024, 1280, 2047, 2048, 4096, 4099, 8192, 11008, 16384]


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", COLS + [16392, 65536, 65537, 131071])
def test_quantize(dt, cols):
    x = normal(cols, 5, cols, dt=dt)
    x[1] = 0
    x[2, : cols // 2] *= 100
    q, scales = q8.quantize(x, dt)
    check_rows(q, scales, q8.f64(x), 1.0, cols, False)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", COLS + [32768, 65543, 70000])
@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm(dt, cols, residual):
    x, w = normal(cols, 7, cols, dt=dt), normal(cols + 1, cols, scale=0.3, shift=1.0, dt=dt)
    r = normal(cols + 2, 7, cols, scale=3.0, dt=dt) if residual else None
    x[1] = 0
    if residual:
        r[1] = 0
    q, scales, total = q8.rms_norm(x, r, w, dt)
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    if residual:
        assert torch.equal(total, h)
    h = q8.f64(h)
    check_rows(q, scales, h * q8.f64(w), 1 / np.sqrt((h * h).mean(-1) + np.float64(np.float32(1e-5))), cols, True)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 255, 4097])
def test_any_number_of_rows(dt, rows):
    x, w = normal(rows, rows, 200, dt=dt), normal(rows + 1, 200, dt=dt)
    q, scales, _ = q8.rms_norm(x, None, w, dt, eps=0.0)
    h = q8.f64(x)
    check_rows(q, scales, h * q8.f64(w), 1 / np.sqrt((h * h).mean(-1)), 200, True)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("cols,offset,ld", [(129, 1, 131), (512, 3, 519), (1280, 8, 1288), (1280, 4, 1300), (4096, 1, 4097), (70000, 1, 70003)])
def test_rows_apart_and_off_the_grid(dt, cols, offset, ld):
    x = normal(ld, 4 * ld + offset, dt=dt)[offset:].view(4, ld)[:, :cols]
    r = normal(ld + 1, 4 * (ld + 2), dt=dt).view(4, ld + 2)[:, 1 : cols + 1]
    w = normal(ld + 2, cols + 1, dt=dt)[1:]
    q, scales = q8.quantize(x, dt, ld_q=cols + 3)
    check_rows(q, scales, q8.f64(x), 1.0, cols, False)
    q, scales, total = q8.rms_norm(x, r, w, dt)
    h = (x.float() + r.float()).to(x.dtype)
    assert torch.equal(total, h)
    h = q8.f64(h)
    check_rows(q, scales, h * q8.f64(w), 1 / np.sqrt((h * h).mean(-1) + np.float64(np.float32(1e-5))), cols, True)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [77, 4096, 70000])
@pytest.mark.parametrize("place", ["x", "residual", "none"])
def test_the_sum_in_place_and_left_out(dt, cols, place):
    x, r, w = normal(1, 3, cols, dt=dt), normal(2, 3, cols, dt=dt), normal(3, cols, dt=dt)
    h = (x.float() + r.float()).to(x.dtype)
    q0, s0, _ = q8.rms_norm(x, r, w, dt)
    q1, s1, total = q8.rms_norm(x, r, w, dt, want_sum=place != "none", in_place={"x": x, "residual": r, "none": None}[place])
    assert torch.equal(q0, q1) and torch.equal(s0, s1)
    if place != "none":
        assert torch.equal(total, h)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_no_weight_is_ones(dt):
    x = normal(4, 3, 640, dt=dt)
    q0, s0, _ = q8.rms_norm(x, None, None, dt)
    q1, s1, _ = q8.rms_norm(x, None, torch.ones(640, dtype=x.dtype, device="cuda"), dt)
    assert torch.equal(q0, q1) and torch.equal(s0, s1)


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [40, 1000, 70000])
def test_rows_that_are_not_finite(dt, cols):
    x = normal(5, 6, cols, dt=dt)
    x[0, cols - 1], x[2, 0], x[3, cols // 2] = float("nan"), float("inf"), -float("inf")
    q, scales = q8.quantize(x, dt)
    assert torch.isnan(scales).tolist() == [True, False, True, True, False, False]
    assert not bool(q[[0, 2, 3]].any())
    q, scales, _ = q8.rms_norm(x, None, normal(6, cols, dt=dt), dt)
    assert torch.isnan(scales).tolist() == [True, False, True, True, False, False]
    assert not bool(q[[0, 2, 3]].any()) and bool(q[[1, 4, 5]].any())


@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_halves_go_to_the_even_integer(dt):
    """Rows whose largest is 127 (or 254, or a tiny power of two of it): values k + 1/2 are exact halves."""
    values = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 62.5, 63.5, -126.5, 126.5, 3.0])
    for scale in (1.0, 2.0, 0.5, 2.0**-10):
        x = (values * scale).to(q8.DTYPES[dt][1]).cuda()[None]
        q, scales = q8.quantize(x, dt)
        assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -2, 62, 64, -126, 126, 3]
        assert scales.item() == scale


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("exponent", [-140, -126, -120, -104, -101, -99, 100, 120])
def test_tiny_and_huge_rows(dt, exponent):
    """127 / a overflows below 2^-121, and a / 127 loses bits below 2^-119: the integers stay the nearest."""
    if dt == "bf16" and exponent < -126:
        exponent = -126
    x = torch.ldexp(normal(7, 2, 96, dt="f32"), torch.tensor(exponent, device="cuda")).to(q8.DTYPES[dt][1])
    q, scales = q8.quantize(x, dt)
    largest, want = q8.nearest(q8.f64(x))
    assert np.array_equal(q.cpu().numpy(), want)
    assert np.all(np.abs(scales.cpu().double().numpy() - largest / 127) <= np.maximum(2.0**-23 * largest / 127, 2.0**-150))


def test_no_columns_and_no_rows():
    x = torch.empty(3, 0, device="cuda")
    q, scales = q8.quantize(x, "f32", ld_q=4)
    assert scales.tolist() == [0, 0, 0]
    q8.quantize(torch.empty(0, 8, device="cuda"), "f32")


# ------------------------------------------------------------------- products
def operands(m, n, k, dt, seed=0):
    gen = torch.Generator()
    gen.manual_seed(1000 + seed + m + n + k)
    a, b = int8s(seed + m * 7 + k, m, k), int8s(seed + n * 5 + k, n, k)
    sa, sb = ((torch.rand(x, generator=gen) + 0.5).cuda() / (60 * k**0.25) for x in (m, n))
    return a, b, sa, sb


def close(c, a, b, sa, sb, dt, bias=None, residual=None, act=None):
    """fp32: the sum to a float, the scales' product, their product, two additions: five roundings of what they add up; the activations within 2e-6 (1 + |y|), the 16-bit GELU
    within 5e-5 (their comments); then half a step of the type (f16: of its smallest normal at least)."""
    s = (a.cpu().double() @ b.cpu().double().T).numpy() * np.outer(q8.f64(sa), q8.f64(sb))
    y, size = s.copy(), np.abs(s)
    for more in (bias, residual):
        if more is not None:
            y, size = y + q8.f64(more), size + np.abs(q8.f64(more))
    t = torch.from_numpy(y)
    y = {None: lambda: t, "relu": lambda: t.relu(), "gelu": lambda: t * torch.special.ndtr(t), "silu": lambda: t * t.sigmoid(), "sigmoid": lambda: t.sigmoid(), "tanh": lambda: t.tanh()}[act]().numpy()
    tolerance = 1.2 * 5 * 2.0**-24 * size + HALF_STEP[dt] * 1.01 * np.maximum(np.abs(y), 2.0**-14 if dt == "f16" else 0)
    if act not in (None, "relu"):
        tolerance += 2e-6 * (1 + np.abs(y)) + (5e-5 if act == "gelu" and dt != "f32" else 0)
    off = np.abs(q8.f64(c) - y)
    assert np.all(off <= tolerance), (float((off - tolerance).max()), np.unravel_index((off - tolerance).argmax(), off.shape))


SHAPES = [(1, 1, 1), (1, 64, 16), (1, 1280, 1280), (3, 5, 17), (2, 51865, 384), (7, 4096, 1024), (8, 256, 4096), (9, 257, 130), (16, 64, 64), (17, 100, 333), (33, 1000, 1000), (64, 512, 2048),
          (100, 77, 63), (128, 128, 128), (130, 250, 1280), (255, 257, 259), (256, 256, 256), (300, 700, 96), (500, 1280, 5120), (513, 384, 1000), (1000, 1001, 1003), (1500, 1280, 640), (2048, 2304, 192)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_products(m, n, k, dt):
    a, b, sa, sb = operands(m, n, k, dt)
    bias, residual = normal(m, n, dt=dt), normal(n, m, n, dt=dt)
    c, _ = q8.gemm(a, b, sa, sb, dt)
    close(c, a, b, sa, sb, dt)
    c, _ = q8.gemm(a, b, sa, sb, dt, bias, residual, "gelu" if m % 2 else "silu")
    close(c, a, b, sa, sb, dt, bias, residual, "gelu" if m % 2 else "silu")


@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "sigmoid", "tanh"])
@pytest.mark.parametrize("m,n,k", [(4, 200, 256), (40, 96, 160), (300, 520, 512)])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_activations(act, m, n, k, dt):
    a, b, sa, sb = operands(m, n, k, dt, 3)
    bias = normal(m, n, dt=dt)
    c, _ = q8.gemm(a, b, sa, sb, dt, bias, None, act)
    close(c, a, b, sa, sb, dt, bias, None, act)


@pytest.mark.parametrize("m,n,k", [(5, 64, 256), (50, 90, 320), (260, 270, 384), (700, 520, 1024)])
@pytest.mark.parametrize("offset,pad", [(0, 16), (4, 4), (1, 3), (16, 1)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_products_of_rows_apart_and_off_the_grid(m, n, k, offset, pad, dt):
    a = int8s(m, m * (k + pad) + offset)[offset:].view(m, k + pad)[:, :k]
    b = int8s(n, n * (k + pad) + offset)[offset:].view(n, k + pad)[:, :k]
    _, _, sa, sb = operands(m, n, k, dt)
    c, _ = q8.gemm(a, b, sa, sb, dt, ldc=n + 5)
    close(c, a, b, sa, sb, dt)


@pytest.mark.parametrize("m,n", [(3, 70), (40, 70), (300, 300)])
def test_sums_at_the_ends_of_32_bits(m, n):
    """131071 products of -128 by -128 are 16384 below 2^31; of -128 by 127 no farther down."""
    k = 131071
    a, b = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    one = torch.ones(max(m, n), device="cuda")
    c, _ = q8.gemm(a, b, one, one, "f32")
    want = torch.tensor([16384.0 * k, -128.0 * 127 * k], dtype=torch.float64).float().cuda()  # (rounded to fp32 once)
    assert bool((c[:, 0::2] == want[0]).all()) and bool((c[:, 1::2] == want[1]).all())


@pytest.mark.parametrize("m,n,k", [(4, 96, 128), (64, 96, 128), (300, 300, 320), (33, 65, 100)])
def test_the_residual_in_the_results_place(m, n, k):
    a, b, sa, sb = operands(m, n, k, "bf16")
    r = normal(1, m, n)
    want, _ = q8.gemm(a, b, sa, sb, "bf16", None, r)
    got, _ = q8.gemm(a, b, sa, sb, "bf16", None, r, out=r)
    assert torch.equal(got, want)


def test_no_k_is_bias_and_residual():
    a, b = torch.empty(3, 0, dtype=torch.int8, device="cuda"), torch.empty(5, 0, dtype=torch.int8, device="cuda")
    one, bias, r = torch.ones(5, device="cuda"), normal(1, 5, dt="f32"), normal(2, 3, 5, dt="f32")
    c, _ = q8.gemm(a, b, one, one, "f32", bias, r)
    assert torch.equal(c, bias + r)


@pytest.mark.parametrize("m", [1, 20, 400])
def test_a_scale_that_is_not_finite_stays_in_its_row(m):
    a, b, sa, sb = operands(m, 130, 256, "bf16")
    sa[m // 2] = float("nan")
    c, _ = q8.gemm(a, b, sa, sb, "bf16")
    rows = torch.isnan(c).all(1).tolist()
    assert rows == [i == m // 2 for i in range(m)] and int(torch.isnan(c).any(1).sum()) == 1


def test_the_same_call_twice_and_on_another_stream():
    a, b, sa, sb = operands(700, 520, 1024, "bf16")
    first, _ = q8.gemm(a, b, sa, sb, "bf16")
    other = torch.cuda.Stream()
    second, _ = q8.gemm(a, b, sa, sb, "bf16", stream=other.cuda_stream)
    assert torch.equal(first, second)
    x = normal(1, 64, 1280)
    q0, s0 = q8.quantize(x, "bf16")
    q1, s1 = q8.quantize(x, "bf16", stream=other.cuda_stream)
    assert torch.equal(q0, q1) and torch.equal(s0, s1)


@pytest.mark.parametrize("k", [8, 100, 1280, 2049])
@pytest.mark.parametrize("act", [None, "gelu", "silu", "tanh"])
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
def test_a_row_has_the_same_bits_whatever_the_others(dt, act, k):
    m, n = 1500, 1000
    a, b, sa, sb = operands(m, n, k, dt)
    bias, residual = normal(m, n, dt=dt), normal(n, m, n, dt=dt)
    want, whole = q8.gemm(a, b, sa, sb, dt, bias, residual, act)
    kernels = {whole}
    for first, last in [(0, 1), (700, 702), (5, 8), (3, 20), (64, 128), (100, 400), (800, 1499)]:
        rows = slice(first, last)
        c, kernel = q8.gemm(a[rows], b, sa[rows].contiguous(), sb, dt, bias, residual[rows].contiguous(), act)
        assert torch.equal(c, want[rows]), kernel
        kernels.add(kernel)
    far = a[:1].as_strided((1, k), (1 << 22, 1))  # (one row, whatever its leading dimension)
    c, kernel = q8.gemm(far, b, sa[:1].contiguous(), sb, dt, bias, residual[:1].contiguous(), act)
    assert kernel == "generic" and torch.equal(c, want[:1])
    assert k < 16 or len(kernels) > 2


@pytest.mark.parametrize("m", [1, 20, 300, 2048])
@pytest.mark.parametrize("large,small", [(1e33, 1e-20), (1e-20, 1e33), (1e-36, 1e30), (1e36, 1e-36)])
def test_scales_of_which_one_is_huge(m, large, small):
    """Their product is an ordinary number; the sum times either of them is not."""
    a, b, sa, sb = operands(m, 520, 1024, "f32")
    sa, sb = sa * large, sb * small
    c, _ = q8.gemm(a, b, sa, sb, "f32")
    close(c, a, b, sa, sb, "f32")


@pytest.mark.parametrize("m", [1, 2])
def test_more_columns_than_one_launch_has_threads_for(m):
    n, k = (1 << 27) + 3, 16
    a = int8s(m, m, k)
    b = torch.empty(n, k, dtype=torch.int8, device="cuda")
    b.view(-1)[:] = torch.arange(16 * 4099, dtype=torch.int32, device="cuda").remainder(251).sub(125).to(torch.int8).repeat(n // 4099 + 1)[: n * k]
    one = torch.ones(n, device="cuda")
    c, kernel = q8.gemm(a, b, one[:m], one, "f32")
    assert kernel != "skinny"
    for first in (0, 1 << 20, 1 << 26, n - 5000):
        part = slice(first, first + 5000)
        assert torch.equal(c[:, part].cpu(), (a.cpu().int()[:, None] * b[part].cpu().int()[None]).sum(-1).float())


def test_rows_farther_apart_than_32_bits():
    """Three rows 2^30 elements apart: the last one's bytes, and its elements' number, lie past 2^31."""
    far, cols = (1 << 30) + 3, 700
    x = normal(5, 3, cols)
    apart = torch.empty(3, far, dtype=torch.bfloat16, device="cuda")[:, :cols]
    apart.copy_(x)
    want, scales = q8.quantize(x, "bf16")
    got, more = q8.quantize(apart, "bf16", ld_q=far)
    assert torch.equal(got, want) and torch.equal(more, scales)
    weight = normal(6, cols)
    want = q8.rms_norm(x, x, weight, "bf16")
    total = torch.empty(3, far, dtype=torch.bfloat16, device="cuda")[:, :cols]
    got = q8.rms_norm(apart, apart, weight, "bf16", in_place=total)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    u = torch.tensor([0.1, 0.5, 0.9])
    assert list(q8.sample(apart, "bf16", u, top_p=0.9)[0]) == list(q8.sample(x, "bf16", u, top_p=0.9)[0])


@pytest.mark.parametrize("m,k", [(3, 640), (3, 8), (3, 100)])
def test_products_with_rows_farther_apart_than_32_bits(m, k):
    far = (1 << 30) + 16
    a, b, sa, sb = operands(m, 300, k, "f32")
    residual = normal(1, m, 300, dt="f32")
    want, _ = q8.gemm(a, b, sa, sb, "f32", None, residual)
    place = torch.empty(m, far, device="cuda")
    place[:, :300] = residual
    got, _ = q8.gemm(a, b, sa, sb, "f32", None, place, ldc=far, out=place)
    assert torch.equal(got[:, :300], want)
    apart = torch.empty(m, far, dtype=torch.int8, device="cuda")[:, :k]
    apart.copy_(a)
    got, kernel = q8.gemm(apart, b, sa, sb, "f32", None, residual)
    assert kernel == "generic" and torch.equal(got, want)
