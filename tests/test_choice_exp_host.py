"""The choice's exponential, its steps carried out exactly on the CPU with the constants of csrc/router.hip, against 50 digits."""
import math
import os
import random
import re
from decimal import Decimal, getcontext
from fractions import Fraction

from conftest import PKG_NAME, ROOT


def constants():
    with open(os.path.join(ROOT, PKG_NAME, "csrc", "router.hip")) as f:
        body = re.search(r"double choice_exp\(double x\) \{\n(.*?)\n\}", f.read(), re.S).group(1)
    floor = re.search(r"x = x < (-[\d.]+) \? \1 : x;", body).group(1)
    inv, ln2 = re.search(r"fma\(x, ([\d.]+), 0x1.8p52\);\n.*fma\(t - 0x1.8p52, -([\d.]+), x\);", body).groups()
    poly = re.findall(r"(?:p = |p, r, )(0x1\.[0-9a-f]+p[+-]\d+|1\.0)[;)]", body)
    assert len(poly) == 11 and poly[-1] == "1.0"
    return float(floor), float(inv), float(ln2), [float.fromhex(c) for c in poly]


def fma(a, b, c):
    return float(Fraction(a) * Fraction(b) + Fraction(c))              # rounded once


def choice_exp(x, floor, inv, ln2, poly):
    x = max(x, floor)
    t = fma(x, inv, 1.5 * 2.0 ** 52)
    n = t - 1.5 * 2.0 ** 52
    r = fma(n, -ln2, x)
    p = poly[0]
    for c in poly[1:]:
        p = fma(p, r, c)
    return math.ldexp(p, int(n))


def points(low, high, n):
    rng = random.Random(1)
    yield from (low, high)
    for _ in range(n):
        yield rng.uniform(low, high)
    for k in range(math.ceil(low / math.log(2)), math.floor(high / math.log(2))):       # where n changes
        yield (k + 0.5) * math.log(2)


def test_how_far_it_is_off():
    getcontext().prec = 50
    c = constants()
    for low, high, bound in ((-200.0, 200.0, 2.0 ** -46), (-708.0, 708.0, 2.0 ** -45)):
        worst = max(abs(Decimal(choice_exp(x, *c)) / Decimal(x).exp() - 1) for x in points(low, high, 4000))
        assert worst <= Decimal(bound)
    assert choice_exp(0.0, *c) == 1.0


def test_past_the_normal_range():
    """Whole numbers of 2^-1074, half of one off at most beside what holds above; no step back on the way down, 0 in the end."""
    getcontext().prec = 50
    c = constants()
    before = math.inf
    for i in range(0, 4000):
        x = -707.0 - i / 100
        v = choice_exp(x, *c)
        want = Decimal(x).exp()
        assert abs(Decimal(v) - want) <= want * Decimal(2.0 ** -45) + Decimal(2) ** -1075
        assert v <= before
        before = v
    assert choice_exp(-746.0, *c) == 0.0 and choice_exp(-1e300, *c) == 0.0 and choice_exp(-744.0, *c) > 0.0
