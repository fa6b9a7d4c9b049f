"""Every kernel that axhip_gemm_q8 has, by name, on matrices whose last rows, columns and chunks are parts, against the integers' products in 64 bits."""
import re
from pathlib import Path

import pytest
import torch

from axiom_amd import capi
from tests import q8_harness as q8

HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}

# (m, n, k) that the choice gives to a kernel; k = 0 modulo 16: rows on the 16-byte grid
KERNELS = {
    "generic": [(37, 131, 9)],
    "skinny": [(1, 8191, 1001), (1, 1283, 4112), (2, 4097, 1000), (2, 1283, 4115)],
    "small_16x16_4": [(16, 8985, 544), (12, 8985, 129)],
    "small_16x16_8": [(12, 41, 8976), (13, 43, 1983)],
    "small_32x16_4": [(3248, 67, 864), (3170, 71, 505)],
    "small_32x16_8": [(60, 1027, 1968), (30, 2049, 1943)],
    "small_32x32_4": [(2457, 159, 144), (3559, 267, 2039)],
    "small_32x32_8": [(89, 1361, 1936), (55, 2053, 1959)],
    "small_32x64_4": [(93, 8261, 1488), (280, 3565, 1933)],
    "small_32x64_8": [(602, 435, 1952), (23, 8247, 1179)],
    "small_64x64_4": [(5240, 177, 1936), (229, 4049, 8155)],
    "small_64x64_8": [(630, 811, 8848), (39, 8209, 5859)],
    "tile_64x128": [(4072, 497, 192), (163, 5609, 8096)],
    "tile_128x128_pair": [(2106, 7259, 144), (853, 8297, 560)],
    "tile_128x128": [(767, 2907, 176), (1278, 1625, 1952)],
    "tile_192x128": [(930, 6415, 144), (532, 7475, 1984)],
    "tile_256x128": [(1922, 4079, 160), (2467, 3111, 1040)],
    "tile_256x256": [(4345, 7591, 192), (5879, 2499, 528)],
    "tile_128x128_ragged": [(2149, 1903, 133), (481, 7923, 2089)],
}


def inputs(m, n, k, dt):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m + 3 * n + 7 * k)
    ints = lambda *s: torch.randint(-128, 128, s, generator=gen, device="cuda", dtype=torch.int8)  # noqa: E731
    normal = lambda *s: torch.randn(s, generator=gen, device="cuda").to(q8.DTYPES[dt][1])  # noqa: E731
    scale = lambda rows: (torch.rand(rows, generator=gen, device="cuda") + 0.5) / (60 * k**0.25)  # noqa: E731
    return ints(m, k), ints(n, k), scale(m), scale(n), normal(n), normal(m, n)


def compare(c, y, size, dt, act_error=0.0):
    """fp32: the sum to a float, the scales' product, their product, two additions: five roundings of what they add up; then half a step of the type (f16: of its smallest
    normal at least)."""
    floor = 2.0**-14 if dt == "f16" else 0.0
    allowed = 5 * 1.001 * 2.0**-24 * size + HALF_STEP[dt] * 1.001 * y.abs().clamp(min=floor) + act_error * (1 + y.abs())
    off = (c.double() - y).abs()
    worst = int((off - allowed).argmax())
    assert bool((off <= allowed).all()), (float(off.flatten()[worst]), float(allowed.flatten()[worst]), divmod(worst, y.shape[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("name,m,n,k", [(name, *shape) for name, shapes in KERNELS.items() for shape in shapes])
def test_the_kernel_that_ran_and_what_it_gave(name, m, n, k, dt):
    a, b, sa, sb, bias, residual = inputs(m, n, k, dt)
    total = torch.mm(a.double(), b.double().t()) * torch.outer(sa.double(), sb.double())
    size = total.abs()
    c, ran = q8.gemm(a, b, sa, sb, dt)
    assert ran == name
    compare(c, total, size, dt)
    c, ran = q8.gemm(a, b, sa, sb, dt, bias, residual, "silu")
    assert ran == name
    y, more = total + bias.double() + residual.double(), size + bias.double().abs() + residual.double().abs()
    compare(c, y * torch.sigmoid(y), 1.2 * more, dt, 2e-6)  # (SiLU's slope is 1.1 at most)
    c, ran = q8.gemm(a, b, sa, sb, dt, bias, residual, out=residual)  # the residual in C's place
    assert ran == name and c.data_ptr() == residual.data_ptr()
    compare(c, y, more, dt)


def test_no_kernel_is_left_out():
    """(no device) The names in the source are those that are compared above."""
    source = (Path(capi.__file__).parent / "csrc" / "gemm_q8.hip").read_text()
    table = source[source.index("Q8_KERNELS[] = {") : source.index("Q8_CANDIDATES")]
    names = set(re.findall(r'"(\w+)"\}', table)) | set(re.findall(r'q8_last_kernel = "(\w+)"', source)) - {"none", "empty"}
    assert len(names) == 19 and names == set(KERNELS)
