"""The integers of the fp32 norm next to a half: products of two fp32 numbers have 48 bits, and so does the row's largest, so that 127 y / a is compared with Python's whole numbers."""
from fractions import Fraction

import pytest
import torch

from tests import q8_harness as q8

pytestmark = pytest.mark.gpu


def integers(h, w):
    """Rows of whole numbers, a weight -> the nearest integers to 127 y / max |y|, halves to the even one."""
    out = []
    for row in h:
        y = [int(a) * int(b) for a, b in zip(row, w)]
        largest = max(abs(v) for v in y)
        out.append([round(Fraction(127 * v, largest)) for v in y])
    return out


def norm(h, w, residual=None):
    on = lambda v: torch.tensor(v, dtype=torch.float64).float().cuda()  # noqa: E731
    q, _, _ = q8.rms_norm(on(h), None if residual is None else on(residual), on(w), "f32")
    return q.tolist()


# (h, w, the row's largest as a product, the nearest integer): whole numbers below 2^24 with |127 h w / (h0 w0) - half| of 5 / (2 h0 w0) at most
NEAR = [(8662177, 10900178, 6057755, 15772805, 125), (7184036, 10919771, 8642775, 15268121, 75), (3590189, 11512987, 15895151, 11587761, 28), (8872901, 16459352, 11686837, 14901689, 106),
        (5769873, 5822756, 11686837, 14901689, 24), (5843990, 10826525, 11810805, 8666687, 79), (5037169, 8212972, 16479181, 9517221, 34), (8901997, 11291843, 16717943, 14273135, 53),
        (8522132, 9114218, 11059413, 14990715, 59), (12508721, 12611631, 10745811, 16283329, 115), (9555017, 13510453, 10434269, 16626899, 94), (7832687, 15258142, 11705947, 15716493, 83),
        (8832535, 15562977, 15462395, 10502593, 108), (7161577, 11565050, 14450609, 10324871, 71), (5277176, 6090955, 9016677, 16463095, 27)]


@pytest.mark.parametrize("cols", [2, 77, 70000])
@pytest.mark.parametrize("case", range(len(NEAR)))
def test_quotients_next_to_a_half(case, cols):
    h, w, h0, w0, want = NEAR[case]
    rows, weight = [[h0, h] + [0] * (cols - 2), [h0, -h] + [0] * (cols - 2)], [w0, w] + [1] * (cols - 2)
    got = norm(rows, weight)
    assert integers([r[:2] for r in rows], weight) == [[127, want], [127, -want]]
    assert [r[:2] for r in got] == [[127, want], [127, -want]] and not any(any(r[2:]) for r in got)


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("cols", [254, 70000])
def test_halves_of_products_go_to_the_even_integer(cols, seed):
    """The largest is 127 q w, the others (2 n + 1) q / 2 times w: 127 y / a is n + 1/2 for every n, whatever q and w are."""
    gen = torch.Generator()
    gen.manual_seed(seed)
    rows = []
    for q in torch.randint(1 << 15, 1 << 16, (6,), generator=gen).tolist():
        row = [2 * 127 * q] + [(2 * n + 1) * q * (1 if n % 3 else -1) for n in range(126)]
        rows.append(row + [0] * (cols - len(row)))
    w = int(torch.randint(1 << 23, 1 << 24, (1,), generator=gen)) | 1
    want = integers([r[:127] for r in rows], [w] * 127)
    assert want[0][1:4] == [0, 2, 2]
    got = norm(rows, [w] * cols)
    assert [r[:127] for r in got] == want


def test_halves_of_a_sum_with_a_residual():
    q, w = 50051, 12345677
    x = [[254 * q - 3] + [(2 * n + 1) * q + 5 for n in range(126)]]
    r = [[3] + [-5] * 126]
    h = [[a + b for a, b in zip(x[0], r[0])]]
    assert norm(x, [w] * 127, r) == integers(h, [w] * 127)
