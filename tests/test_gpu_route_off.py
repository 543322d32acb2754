"""Routing with experts that a bias switches off, by a large finite value as well as by -infinity."""
import numpy as np
import pytest

from tests import test_gpu_route as R

pytestmark = pytest.mark.gpu

LOWEST = np.finfo(np.float32).min
# T, E, K, groups, top, best
SHAPES = [(5000, 256, 24, 8, 4, 2), (5000, 128, 20, 1, 1, 1), (4200, 512, 24, 16, 5, 2), (600, 64, 18, 4, 3, 1), (4500, 250, 24, 10, 5, 2), (4200, 400, 40, 1, 1, 1)]


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,K,groups,top,best", SHAPES)
def test_the_value_that_switches_off_does_not_matter(T, E, K, groups, top, best, sigmoid):
    """The same choice and the same bits of the weights.  (More chosen experts than a token has lanes: a token that is chosen for again in double has its
    weights' sum added up in another order, and so other bits, which few of these tokens need.)"""
    rng = np.random.default_rng(T + E)
    z = (rng.standard_normal((T, E)) * 1.5).astype(np.float32)
    bias = (rng.standard_normal(E) * (0.2 if sigmoid else 1.0 / E)).astype(np.float32)
    off = rng.choice(E, E // 8, replace=False)
    got = []
    for value in (-np.inf, -1e9, LOWEST):
        b = bias.copy()
        b[off] = value
        if groups > 1:
            b[:E // groups] = value                   # a whole group as well
        got.append(R.check(z, b, K, sigmoid=sigmoid, groups=groups, top=top, best=best))
    for ids, w, counts in got[1:]:
        assert np.array_equal(ids, got[0][0]) and np.array_equal(counts, got[0][2])
        assert np.array_equal(w, got[0][1])
