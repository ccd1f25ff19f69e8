"""swamp_rope_freqs' ramp at its ends, without a GPU: a pair that turns less than
beta_slow times in the trained context is divided by the factor, one that turns more
than beta_fast times is not, whatever the context and the betas."""
import math

import numpy as np
import pytest


@pytest.mark.parametrize("n,base,ctx,fast,slow", [
    (128, 10000.0, 4, 32.0, 1.0),       # even the fastest pair turns less than once
    (64, 500000.0, 6, 32.0, 1.0),
    (128, 10000.0, 4096, 2000.0, 1000.0),
    (8, 10.0, 100000, 32.0, 1.0),       # even the slowest turns more than 32 times
    (2, 10000.0, 4096, 32.0, 1.0),
    (2, 10000.0, 3, 32.0, 1.0),
    (128, 10000.0, 4096, 32.0, 1.0),
    (128, 10000.0, 4096, 1.0001, 1.0),  # nearly no room between the two
    (96, 500000.0, 8192, 32.0, 1.0),
])
@pytest.mark.parametrize("factor", [8.0, 0.5])
def test_pairs_beyond_the_ramp(pkg, n, base, ctx, fast, slow, factor):
    f = pkg.rope_freqs(n, base, factor, ctx, fast, slow)
    plain = base ** (-2.0 * np.arange(n // 2) / n)
    turns = plain * ctx / (2 * math.pi)
    np.testing.assert_allclose(f[turns < slow], plain[turns < slow] / factor, rtol=1e-12)
    np.testing.assert_allclose(f[turns > fast], plain[turns > fast], rtol=1e-12)
    between = (turns <= fast) & (turns >= slow)
    lo, hi = sorted((1.0, 1.0 / factor))
    assert np.all(f[between] >= plain[between] * lo * (1 - 1e-12))
    assert np.all(f[between] <= plain[between] * hi * (1 + 1e-12))
