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


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T", [7, 200, 4200])
@pytest.mark.parametrize("E", [8, 24, 128, 384])
def test_groups_worth_less_than_the_lowest_number(E, T, sigmoid):
    """The sum of two worths may lie below what fp32 holds: such a group is behind the others and in front of one that has nothing open."""
    rng = np.random.default_rng(E + T)
    groups, n = 4, E // 4
    z = rng.standard_normal((T, E)).astype(np.float32)
    b = (0.1 * rng.standard_normal(E)).astype(np.float32)
    z[:, 3:n] = -np.inf                               # the first group: three open at most
    z[:, n:2 * n] = -np.inf                           # the second: nothing
    for low in (LOWEST, LOWEST / 2):                  # the third: switched off; the fourth: a little less so
        b[2 * n:3 * n] = LOWEST
        b[3 * n:] = low
        for top in (2, 3):
            R.check(z, b, 2 * n if n < 5 else 7, sigmoid=sigmoid, groups=groups, top=top, best=2)
        b[3 * n:] = 0.05
        R.check(z, b, 2, sigmoid=sigmoid, groups=groups, top=3, best=2)
