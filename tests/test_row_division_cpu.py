"""The row kernels divide a maximum by 127 or 448 with one residual step, q + (m - q * d) * r, r = 1 / d rounded: the IEEE quotient for every
mantissa (a power of two in front changes nothing in the normal range)."""
import numpy as np
import pytest


@pytest.mark.parametrize("divisor", [127, 448])
def test_one_residual_step_is_the_ieee_quotient(divisor):
    f, wide = np.float32, np.longdouble
    d, r = f(divisor), f(1) / f(divisor)
    for part in np.split(np.arange(0x3F800000, 0x40000000, dtype=np.uint32), 8):
        m = part.view(f)
        q = m * r
        rest = m.astype(wide) - q.astype(wide) * divisor
        assert (rest.astype(f) == rest).all()  # the first fma rounds nothing
        got = (q.astype(wide) + rest * wide(r)).astype(f)
        assert np.array_equal(got, m / d)
