"""What quantising to E4M3 relies on for codes that are those of x / scale rounded to fp32, without a division: scale = largest / 448 from a product with the
rounded 1 / 448 and its remainder, x / scale from a sum of two numbers that is the scale's inverse but for 2^-43.

Let q = x / scale.  With n the hardware's inverse of the scale less two of its last steps, 1 - n scale is at most 2^-21, n (1 - n scale) short of what n lacks by
2^-42 of that at most, its rounding and that of its product with x are 2^-24 of 2^-21: x n + x rest is q (1 + e), |e| below 2^-41, rounded once.
The code differs from that of q rounded to fp32 only if one of the two is a tie of E4M3 and the other the number next to it.  Ties are T 2^i with T odd below
32.  With 448 x other than T 2^i times the largest magnitude, integers of at most 11 bits, the quotient is at least 2^-17 of itself away from the tie.  Where
they are equal, q = T 2^i / (1 + d) with the scale's own rounding d: all of these are looked at here."""
from fractions import Fraction

import numpy as np


def _rounded(v):
    """A positive fraction rounded to 24 bits, ties to even"""
    e = 0
    while v >= 1 << 24:
        v, e = v / 2, e + 1
    while v < 1 << 23:
        v, e = v * 2, e - 1
    n, rest = v.numerator // v.denominator, v - v.numerator // v.denominator
    if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and n % 2):
        n += 1
    return Fraction(n) * Fraction(2) ** e


def test_scales_without_a_division():
    """fma(fma(-q0, 448, a), c, q0) with c = 1/448 rounded and q0 = a c rounded, for every significand of 11 bits."""
    c = _rounded(Fraction(1, 448))
    for a in range(1024, 2048):
        q0 = _rounded(a * c)
        remainder = a - q0 * 448
        assert remainder == 0 or _rounded(abs(remainder)) == abs(remainder)
        assert _rounded(q0 + remainder * c) == _rounded(Fraction(a, 448)), a


def test_ties_are_not_next_to_a_midpoint_of_fp32():
    margin = Fraction(1, 1 << 41)
    nearest, seen = 1, 0
    for a in range(1024, 2048):
        scale = _rounded(Fraction(a, 448))
        for odd in range(1, 32, 2):
            # x = odd a / 7 but for powers of two, if that is an integer of 11 bits
            x = odd * a // 7
            if odd * a % 7 or x // (x & -x) >= 2048:
                continue
            seen += 1
            q = odd * Fraction(a, 448) / scale
            step = Fraction(2) ** (odd.bit_length() - 1 - 23)
            # (below a power of two, T = 1, the steps are half as long)
            for midpoint in (odd + step / 2, odd - (step / 2 if odd > 1 else step / 4)):
                away = abs(q - midpoint) / midpoint
                nearest = min(nearest, away)
                assert away > margin, (a, odd)
    assert seen > 2000 and Fraction(1, 1 << 36) < nearest < Fraction(1, 1 << 30)


def test_other_quotients_are_far_from_ties():
    x, largest = np.arange(1, 2048)[:, None].astype(np.int64), np.arange(1024, 2048)[None, :].astype(np.int64)
    for odd in range(1, 32, 2):
        # 448 x against odd 2^i largest, the power of two that brings them nearest
        ratio = 448 * x / (odd * largest)
        for i in (np.floor(np.log2(ratio)).astype(np.int64), np.ceil(np.log2(ratio)).astype(np.int64)):
            left, right = 448 * x * 2 ** np.maximum(-i, 0), odd * largest * 2 ** np.maximum(i, 0)
            off = np.abs(left - right)
            assert bool(((off == 0) | (off * 2 ** 17 > right)).all())
