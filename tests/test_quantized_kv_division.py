"""The cache's scale is max/15 - min/15 in IEEE single precision.  The kernel divides by 15 as q = x * (1/15) and one correction,
q + (x - 15 q) * (1/15), each step rounded once: restated here in rational numbers, over every value of both 16-bit types."""
from fractions import Fraction

import numpy as np
import pytest
import torch


def single(x: Fraction) -> Fraction:
    """x rounded to single precision, ties to even, subnormals included."""
    if x == 0:
        return x
    n, d = abs(x.numerator), x.denominator
    e = n.bit_length() - d.bit_length()
    if Fraction(n, d) < Fraction(2) ** e:
        e -= 1
    step = Fraction(2) ** max(e - 23, -149)
    return round(x / step) * step


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_division_by_15_is_exact_to_the_last_bit(dtype):
    inv = single(Fraction(1, 15))
    x = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)      # negative values: the same by symmetry
    x = x[x.isfinite()].double().tolist()
    # a full division never lands between two floats where rounding twice would matter: fp32's own quotient agrees with it
    quotients = (np.asarray(x, np.float32) / np.float32(15)).astype(np.float64)
    for value, quotient in zip(x, quotients):
        value = Fraction(value)
        q = single(value * inv)
        got = single(single(value - 15 * q) * inv + q)
        assert got == single(value / 15) == Fraction(float(quotient)), value
