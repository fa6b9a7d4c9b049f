"""The table of angles (host code, no device): against the definitions in exact fractions of a turn."""
import math

import pytest

from axiom_amd import capi
from tests import cache_harness as ch


def radians(rot, theta=10000.0, kind=capi.ROPE_PLAIN, factor=1.0, low=1.0, high=4.0, length=8192.0):
    """Frequencies in 53 bits, by the definition."""
    if kind == capi.ROPE_BASE and rot > 2:
        theta *= factor ** (rot / (rot - 2))
    for i in range(rot // 2):
        f = theta ** (-2 * i / rot)
        if kind == capi.ROPE_LINEAR:
            f /= factor
        if kind == capi.ROPE_BANDS:
            keep = min(1.0, max(0.0, (length * f / (2 * math.pi) - low) / (high - low)))
            f = f * keep + f / factor * (1 - keep)
        yield f


@pytest.mark.parametrize("rot", [2, 20, 64, 128, 256])
@pytest.mark.parametrize("how", [dict(), dict(theta=1e6), dict(theta=1.0), dict(kind=capi.ROPE_LINEAR, factor=4.0), dict(kind=capi.ROPE_LINEAR, factor=0.01), dict(kind=capi.ROPE_BASE, factor=8.0),
                                 dict(theta=500000.0, kind=capi.ROPE_BANDS, factor=8.0), dict(kind=capi.ROPE_BANDS, factor=32.0, low=0.0, high=1.0, length=100.0)])
def test_the_table(rot, how):
    for got, f in zip(ch.turns(rot, **how), radians(rot, **how)):
        off = abs(got / 2**64 - f / (2 * math.pi) % 1.0)
        # powers and quotients in 53 bits: 2^-53 of the exponent's logarithm and some; a turn may wrap
        assert min(off, 1 - off) <= 64 * 2.0**-53 * max(1.0, f), (got, f)


def test_the_fastest_angle_is_a_radian():
    assert abs(ch.turns(128)[0] - 2**64 / (2 * math.pi)) <= 2**11  # (2^64 / 2 pi in 53 bits)


@pytest.mark.parametrize("change", [dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=-2), dict(rot_dim=1026), dict(kind=4), dict(kind=-1), dict(theta=0.5), dict(theta=float("inf")), dict(theta=float("nan")),
                                    dict(kind=1, factor=0.0), dict(kind=1, factor=float("nan")), dict(kind=2, factor=-1.0), dict(kind=3, low=-1.0), dict(kind=3, low=4.0), dict(kind=3, length=0.0),
                                    dict(kind=3, high=float("inf"))])
def test_refusals(change):
    s = ch.scaling(64, factor=2.0)
    for name, value in change.items():
        setattr(s, name, value)
    table = (ch.C.c_uint64 * 1024)()
    assert capi.lib().axhip_rope_turns(ch.C.byref(s), table) == capi.ERR_INVALID_ARG
    assert capi.lib().axhip_rope_turns(None, table) == capi.ERR_INVALID_ARG and capi.lib().axhip_rope_turns(ch.C.byref(s), None) == capi.ERR_INVALID_ARG
