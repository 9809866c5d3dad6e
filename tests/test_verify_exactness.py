"""The 64-bit exponential of ovf_verify.cu, emulated step by step with exact
arithmetic (each operation rounded to nearest once, as the device does), against e^x to 60
digits: its stated bounds of 2^-43.8 for |x| < 700 and 2^-44.4 for |x| < 40."""
import random
from decimal import Decimal, localcontext
from fractions import Fraction

import pytest

LN2 = 0.693147180559945309417
SCALE, STEP = 64.0 / LN2, -LN2 / 64.0
SHIFT = 1.5 * 2.0 ** 52


def fma(a, b, c):
    x = Fraction(a) * Fraction(b) + Fraction(c)
    return x.numerator / x.denominator  # (a quotient of integers is rounded to nearest once)


def table():
    with localcontext() as c:
        c.prec = 60
        return [float(Decimal(2) ** (Decimal(i) / 64)) for i in range(64)]


TAB = table()


def error(x):
    """Of vf_exp(x), relative."""
    kd = fma(x, SCALE, SHIFT)
    n = kd - SHIFT
    r = fma(n, STEP, x)
    y = fma(r, 1 / 24, 1 / 6)
    for c in (0.5, 1.0, 1.0):
        y = fma(y, r, c)
    k = int(n)
    with localcontext() as c:
        c.prec = 60
        true = Decimal(x).exp() / Decimal(2) ** (k >> 6)
        return float(abs(Decimal(y * TAB[k & 63]) - true) / true)


@pytest.mark.parametrize("most,bound", [(40.0, -44.4), (700.0, -43.8)])
def test_exponential(most, bound):
    rng = random.Random(1)
    # the worst reduced argument (half a step from both neighbours) at every 16th multiple, and anywhere
    ends = [s * (n + 0.5) * LN2 / 64 * (1 + d) for n in range(0, int(most * SCALE) - 1, 16) for s in (1, -1) for d in (-1e-9, 1e-9)]
    points = [x for x in ends if abs(x) < most] + [rng.uniform(-most, most) for _ in range(4000)]
    assert max(map(error, points)) < 2.0 ** bound
