"""The residual norm's quotients (`divide` in csrc/add_rmsnorm_quant.cu) give the e4m3 bytes of the IEEE quotients, for every pair of 24-bit significands.

With y = RN(1 / d): q = RN(x y), r = RN(x - d q), q' = RN(q + r y).  y is off by at most 2^-24 of itself and q by 2^-23 of x / d (and 2^-48), so q + r y, in
which the error of q remains times those of y and r, is off by less than 2^-46 (1 + 2^-20) of x / d.  A byte depends on whether a quotient lies below, on or
above a border t of five significant bits.  RN(x / d) is t where x / d lies between m1 = t - half a step and m2 = t + half a step, numbers of 25 bits;
q' can only differ in that where x / d is within 2^-46 (1 + 2^-20) of m1 or m2.  With x = X 2^i, d = D 2^j, m = M 2^l and integers X, D < 2^24, M < 2^25 that is
|X 2^k - D M| < 2^-46 D M (1 + 2^-20) < 9.  All D and M with a multiple of 2^k that near are found here (with twice the margin), and the scheme is
followed in exact arithmetic for each."""
from __future__ import annotations

from fractions import Fraction

import numpy as np

MARGIN = 18


def to_float(v: Fraction) -> Fraction:
    """Rounded to 24 significant bits, ties to even; no limit of exponents (the norm's quotients are far from them)."""
    if v == 0:
        return v
    sign, v = (-1 if v < 0 else 1), abs(v)
    e = v.numerator.bit_length() - v.denominator.bit_length() - 24
    while v / Fraction(2) ** e >= 1 << 24:
        e += 1
    while v / Fraction(2) ** e < 1 << 23:
        e -= 1
    return sign * round(v / Fraction(2) ** e) * Fraction(2) ** e  # (round() of a Fraction: ties to even)


def divide(x, d):
    y = to_float(1 / d)
    q = to_float(x * y)
    return to_float(q + to_float(x - d * q) * y)


def test_rounding_to_float():
    rng = np.random.default_rng(1)
    for v in rng.standard_normal(500):
        assert to_float(Fraction(float(v))) == Fraction(float(np.float32(v)))
    for v in ((1 << 24) + 1, (1 << 24) + 3, (1 << 25) - 1):
        assert to_float(Fraction(v)) == Fraction(float(np.float32(v)))


def test_quotients_beside_the_borders_of_bytes():
    d = np.arange(1 << 23, 1 << 24, dtype=np.int64)
    pairs = []
    for t in range(16, 33):  # the border, in units of 2^20; half a step beside it is one unit (a step below a power of two is half as wide)
        for side in (-1, 1):
            if (t, side) in ((16, -1), (32, 1)):
                continue
            m = (t << 20) + side
            product = d * m
            k = np.where(product < 1 << 48, 24, 25)
            rest = product & ((np.int64(1) << k) - 1)
            near = np.minimum(rest, (np.int64(1) << k) - rest) <= MARGIN
            for dd, kk, pp in zip(d[near].tolist(), k[near].tolist(), product[near].tolist()):
                x = (pp + (1 << (kk - 1))) >> kk
                assert (1 << 23) <= x <= 1 << 24
                pairs.append((Fraction(x << kk), Fraction(dd), t << 20))
    assert len(pairs) > 100
    for x, d, t in pairs:
        ours, exact = divide(x, d), to_float(x / d)
        assert (ours > t) == (exact > t) and (ours < t) == (exact < t), (x, d, t)


def test_scales():
    """The scale, a quotient by 448 = 7 2^6, is the IEEE one itself: x / 7 is at least 1 / 14 of a step from the middle of two floats."""
    rng = np.random.default_rng(2)
    for x in [*range(1 << 23, (1 << 23) + 2000), *range((1 << 24) - 2000, 1 << 24), *rng.integers(1 << 23, 1 << 24, 3000).tolist()]:
        assert divide(Fraction(x), Fraction(448)) == to_float(Fraction(x, 448))
