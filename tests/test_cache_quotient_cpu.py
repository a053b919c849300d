"""The quantising write's quotients in exact arithmetic: with y the rounded reciprocal of the scale, q = x y, r = q scale - x and
q - r y, each rounded once to fp32, give the correctly rounded x / scale -- for every pair of mantissas of a bf16 row's largest
element and another one, and a sample of fp16's."""
from fractions import Fraction

import pytest


def _f32(v):
    """Nearest fp32 value, ties to even (normal range)."""
    if v == 0:
        return v
    a = abs(v)
    e = a.numerator.bit_length() - a.denominator.bit_length()
    e -= Fraction(2) ** e > a
    n, r = divmod(a / Fraction(2) ** (e - 23), 1)
    n += r > Fraction(1, 2) or (r == Fraction(1, 2) and n % 2 == 1)
    return (n if v > 0 else -n) * Fraction(2) ** (e - 23)


@pytest.mark.parametrize("bits,step", [(7, 1), (10, 13)])
def test_quotients_are_correctly_rounded(bits, step):
    one = 2 ** bits
    for i in range(0, one, step):
        top = Fraction(one + i, one)
        scale = _f32(top / 448)
        y = _f32(1 / scale)
        for j in range(0, one, step):
            x = Fraction(one + j, one)
            x /= 1 + (x > top)  # (powers of two change nothing in the normal range)
            q = _f32(x * y)
            assert _f32(q - _f32(q * scale - x) * y) == _f32(x / scale)
