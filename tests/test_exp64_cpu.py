"""The beam selection's exponential in 64 bits (csrc/beam.hip): its polynomial against exp in 50 digits over the
reduced range, without a GPU."""

import os
import re
from decimal import Decimal, localcontext

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mini-llama-cpp-release_amd", "csrc", "beam.hip")


def test_polynomial():
    """Interpolation of exp at the nine Chebyshev points of [-h, h], h = ln 2 / 2, is off by e^h h^9 / (9! 2^8) at the
    most, 1.10e-12 of a value not below e^-h: 1.56e-12 of it.  The coefficients' and the steps' roundings, 2^-53 of a term each,
    nine terms whose sum of magnitudes is below e^h, add 2e-15."""
    with open(SOURCE) as f:
        body = re.search(r"double exp64\(double d\) \{(.*?)\n\}", f.read(), re.S).group(1)
    first = re.search(r"double y = (\S+);", body).group(1)
    coefficients = [Decimal(float(c)) for c in (first, *re.findall(r"y = fma\(y, r, (\S+)\);", body))]
    assert len(coefficients) == 9
    with localcontext() as c:
        c.prec = 50
        h = Decimal(2).ln() / 2
        worst = Decimal(0)
        for i in range(-1000, 1001):
            r, y = h * i / 1000, Decimal(0)
            for a in coefficients:
                y = y * r + a
            worst = max(worst, abs(y / r.exp() - 1))
    assert worst < Decimal("1.56e-12") + Decimal("2e-15") < Decimal(2) ** -39
