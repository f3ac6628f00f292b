"""CPU: the frequencies of a scaled base where that base itself is past the range of a double."""

import math

import numpy as np
import pytest

from zenjpegai_amd import nn


@pytest.mark.parametrize("dim,base,factor", [(4, 1e200, 1e60), (4, 1e300, 2.0 ** 100), (64, 1e300, 1e9), (8, 10000.0, 1e280), (128, 10000.0, 8.0)])
def test_frequencies_follow_the_formula(dim, base, factor):
    f, m = nn.rotary_frequencies(dim, base, scaling="ntk", factor=factor)
    assert m == 1.0 and f[0] == 1.0
    for i, got in enumerate(f):
        # (base s^(dim / (dim - 2)))^(-2i / dim) by its logarithm, which is off by three roundings and their products with it.
        log = -2.0 * i / dim * (math.log(base) + dim / (dim - 2.0) * math.log(factor))
        assert got == pytest.approx(math.exp(log), rel=2.0 ** -53 * (8 * abs(log) + 8)), i
    assert np.isclose(f[-1], nn.rotary_frequencies(dim, base)[0][-1] / factor, rtol=1e-12, atol=0)
