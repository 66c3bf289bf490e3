"""The casts' arithmetic on small gradients' scales, s = max(RN(amax / 448), 2^-92) for amax < 1e-4: the
same three steps as for activations' scales stay correctly rounded down to that floor. Exact rational
arithmetic, no GPU.

2^-92 is the least scale for which no step leaves fp32's range: a remainder x - s q of the division is a
multiple of ulp(s) ulp(q), and with q at or above 2^-11 (below 2^-10 a code is zero either way) that is
at least 2^(-92 - 23) 2^(-11 - 23) = 2^-149, the least subnormal.
"""

from __future__ import annotations

import math
from fractions import Fraction as F

from test_scale_reciprocal import _bits, _from_bits, markstein_reciprocal, rn32

FLOOR = F(2) ** -92


def rn(q: F) -> F:
    """rn32 with gradual underflow."""
    if abs(q) >= F(2) ** -126:
        return rn32(q)
    unit = F(2) ** -149
    m = q / unit
    fl = m.numerator // m.denominator
    rem = m - fl
    if rem > F(1, 2) or (rem == F(1, 2) and fl % 2 == 1):
        fl += 1
    return fl * unit


def divide(x: F, s: F, rc: F) -> tuple[F, bool]:
    """The kernels' division (their div2_rn), and whether its remainder was untouched by underflow:
    the same as the remainder of the problem scaled up by 2^80."""
    q0 = rn(x * rc)
    exact = x - q0 * s
    rem = rn(exact)
    return rn(q0 + rem * rc), rem * 2**80 == rn(exact * 2**80)


def maxima():
    """Every bf16 magnitude whose scale is at or above the floor and below the activations' 1e-4 (the
    gradients' cast takes those below 1e-4 itself)."""
    for b in range(1, 0x7F80):
        a = F(_from_bits(b << 16))
        if a / 448 >= F(1, 10000):
            return
        if a / 448 >= FLOOR:
            yield a


def test_scales_and_their_reciprocals_are_correctly_rounded():
    rc448 = rn32(F(1, 448))
    seen = 0
    for a in [*maxima(), FLOOR * 448]:
        s, exact = divide(a, F(448), rc448)
        assert exact and s == rn32(a / 448)
        want = rn32(1 / s)
        wb = _bits(float(want))
        for k in (-2, -1, 0, 1, 2):
            assert markstein_reciprocal(s, F(_from_bits(wb + k))) == want, (s, k)
        seen += 1
    assert seen > 78 * 128


def test_division_is_correctly_rounded_at_the_least_scales():
    """Elements from half the least code's value to the group's maximum."""
    for a in list(maxima())[: 2 * 128 : 3]:
        s = rn32(a / 448)
        rc = rn32(1 / s)
        for e in (-19, -18, -17, -9, -1):
            for m in range(128, 256, 5):
                x = F(m, 128) * F(2) ** (math.floor(math.log2(float(a))) + e)
                if x > a or x / s < F(2) ** -11:
                    continue
                q, exact = divide(x, s, rc)
                assert exact and q == rn(x / s), (x, s)


def test_one_binade_below_the_floor_the_remainder_underflows():
    """The check above is not vacuous."""
    inexact = 0
    for m in range(129, 256, 2):
        s = rn32(F(m, 448) * F(2) ** -97)
        rc = rn32(1 / s)
        for n in range(128, 256, 3):
            x = F(n, 128) * s * F(2) ** -11
            x = F(_from_bits(_bits(float(x)) & 0xFFFF0000))
            if x > 0:
                inexact += not divide(x, s, rc)[1]
    assert inexact > 0
