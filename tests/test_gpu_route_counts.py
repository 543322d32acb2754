"""Counts of routing are those of the ids that are written, whichever way a token was chosen for."""
import numpy as np
import pytest

from tests import test_gpu_route as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,K,groups,top", [(200, 64, 8, 4, 2), (64, 128, 8, 8, 3), (3000, 96, 8, 4, 2), (5000, 256, 8, 8, 4), (4200, 512, 20, 16, 4), (17, 12, 6, 1, 1), (4500, 40, 3, 1, 1)])
def test_counts_are_those_of_the_ids(T, E, K, groups, top, sigmoid):
    """Few different logits and biases, so that many tokens are told apart in double, some in place and some by a wave at the end of their workgroup."""
    rng = np.random.default_rng(E + T)
    z = rng.choice(rng.standard_normal(3).astype(np.float32), (T, E))
    near = rng.random((T, E)) < 0.5
    z[near] = (z[near].view(np.int32) + rng.integers(-2, 3, near.sum(), dtype=np.int32)).view(np.float32)
    z[rng.random((T, E)) < 0.1] = -np.inf
    z[rng.random(T) < 0.1] = -np.inf
    z[:3] = 0.25
    for b in (None, np.zeros(E, np.float32), rng.choice(np.float32([0.0, 0.125]), E), (1e-7 * rng.standard_normal(E)).astype(np.float32)):
        for best in (1, 2):
            ids, w, counts = R.forward(z, b, K, sigmoid=sigmoid, groups=groups, top=top, best=best)
            assert ((ids >= -1) & (ids < E)).all() and not w[ids < 0].any()
            assert np.array_equal(counts, np.bincount(ids[ids >= 0], minlength=E))
            order = np.sort(np.where(ids < 0, -1 - np.arange(K), ids), 1)
            assert (order[:, 1:] != order[:, :-1]).all()              # a token's ids differ
