"""The quantizer's quotients by a rounded reciprocal and one residual take the
code of the correctly rounded quotient, always.

With x = a 2^i, s = b 2^j, a and b in [1, 2) on the grid of 2^-23, no step under-
or overflows where the code is not 0 either way (s >= 1e-12, |x / s| <= 448 and a
unit), so a and b decide.  r = RN(1 / b) is off by at most 2^-25.  The first
quotient q0 = RN(a r) is off by at most (a + 1) 2^-25 for a < b (a quotient in
(1/2, 1)) and (a + 2) 2^-25 for a >= b, so the residual e = a - q0 b, rounded
once, is at most 8 * 2^-25, and the sum q0 + RN(e) r before its rounding is off
from a / b by at most |e| (2^-24 + 2^-25) <= 12 * 2^-49.

Its rounding can differ from RN(a / b) only where the middle between two
neighbouring f32 lies that near to a / b, and the code only if one of the two is
a middle h between codes: five bits, h = k / 16 or k / 32.  There a / b is within
12 * 2^-49 of m = h +- half a unit, so |a - h b -+ (half a unit) b| <= 24 * 2^-49,
and a - h b is on the grid of 2^-27 (2^-28 for h < 1): b has to lie within 12
units of 2^-23 of a multiple of 1/8.  That leaves few pairs; all are tried here
in exact arithmetic, with two units to spare."""
from fractions import Fraction

import pytest

P = 24


def rn(v: Fraction) -> Fraction:
    """To the nearest f32 (no limits of its exponent), ties to even."""
    if v == 0:
        return v
    sign, v = (-1, -v) if v < 0 else (1, v)
    e = v.numerator.bit_length() - v.denominator.bit_length()
    while v >= Fraction(2) ** (e + 1):
        e += 1
    while v < Fraction(2) ** e:
        e -= 1
    unit = Fraction(2) ** (e - P + 1)
    n, rest = divmod(v, unit)
    n = int(n)
    if rest * 2 > unit or (rest * 2 == unit and n % 2):
        n += 1
    return sign * n * unit


def quotient(a: Fraction, b: Fraction) -> Fraction:
    r = rn(1 / b)
    q0 = rn(a * r)
    return rn(q0 + rn(a - q0 * b) * r)


def critical_divisors():
    unit = Fraction(1, 1 << 23)
    for j in range(8, 17):
        for d in range(-14, 15):
            b = Fraction(j, 8) + d * unit
            if 1 <= b < 2:
                yield b


def critical_pairs():
    unit = Fraction(1, 1 << 23)
    for b in critical_divisors():
        for k in range(16, 33):
            for h, half in ((Fraction(k, 16), Fraction(1, 1 << 24)), (Fraction(k, 32), Fraction(1, 1 << 25))):
                for m in (h, h + half, h - half, h - half / 2):  # h a power of two: the unit below is half as wide
                    n = int(m * b / unit)
                    for a in ((n - 1) * unit, n * unit, (n + 1) * unit, (n + 2) * unit):
                        if 1 <= a < 2:
                            yield a, b, h


def test_rounding_by_hand():
    assert rn(Fraction(1, 3)) == Fraction(11184811, 1 << 25)
    assert rn(Fraction((1 << 24) + 1)) == 1 << 24 and rn(Fraction((1 << 24) + 3)) == (1 << 24) + 4
    assert rn(Fraction(-5, 4)) == Fraction(-5, 4)


@pytest.mark.parametrize("part", range(4))
def test_every_critical_pair_takes_the_same_code(part):
    """Below h, on it or above it: the same side as the correctly rounded one."""
    seen = 0
    for i, (a, b, h) in enumerate(critical_pairs()):
        if i % 4 != part:
            continue
        want, got = rn(a / b), quotient(a, b)
        assert (want > h) - (want < h) == (got > h) - (got < h), (a, b, h)
        seen += 1
    assert seen > 10000
