"""Routing of batches that are cut otherwise than small ones: many tokens, more experts than 256, the widths of groups that lie across a lane's
experts, and the batches around what one workgroup takes at once."""
import numpy as np
import pytest

from tests import test_gpu_route as R
from tests import test_gpu_route_layer as RL

pytestmark = pytest.mark.gpu

INF = np.inf
# T, E, K, groups, top, best
SHAPES = [(4600, 512, 8, 16, 4, 2), (4300, 300, 33, 1, 1, 1), (4200, 384, 6, 32, 5, 2), (4200, 290, 4, 29, 3, 2), (4100, 512, 16, 64, 9, 2), (4300, 257, 31, 1, 1, 1),
          (4500, 256, 8, 8, 4, 2), (5000, 130, 3, 13, 2, 2), (4100, 129, 64, 3, 2, 1), (9000, 64, 6, 2, 1, 2), (300, 320, 5, 5, 3, 2),
          (16, 256, 8, 8, 4, 2), (17, 256, 8, 8, 4, 2), (32, 256, 8, 8, 4, 2), (33, 256, 8, 8, 4, 2), (64, 128, 8, 4, 2, 2), (65, 128, 8, 4, 2, 2), (40, 200, 64, 2, 2, 2)]


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,K,groups,top,best", SHAPES)
def test_against_the_definition(T, E, K, groups, top, best, sigmoid, biased):
    rng = np.random.default_rng(T + E + K)
    z = (rng.standard_normal((T, E)) * 1.5 + rng.standard_normal(E)).astype(np.float32)
    z[rng.random((T, E)) < 0.05] = -INF
    z[rng.random(T) < 0.1] = -INF                    # a padded batch
    b = (0.2 * rng.standard_normal(E)).astype(np.float32) if biased else None
    dw = rng.standard_normal((T, K)).astype(np.float32)
    R.check(z, b, K, dw, sigmoid=sigmoid, renorm=biased, scale=2.5, groups=groups, top=top, best=best)


@pytest.mark.parametrize("E,K,groups", [(512, 8, 1), (400, 31, 8), (384, 4, 32)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_worths_that_fp32_cannot_tell_apart(E, K, groups, sigmoid):
    rng = np.random.default_rng(E)
    T = 4200
    pool = rng.standard_normal(3).astype(np.float32)
    z = rng.choice(pool, (T, E))
    near = rng.random((T, E)) < 0.5
    z[near] = (z[near].view(np.int32) + rng.integers(-2, 3, near.sum(), dtype=np.int32)).view(np.float32)
    z[:3] = 0.25
    for b in (None, rng.choice(np.float32([0.0, 0.125]), E)):
        R.check(z, b, K, sigmoid=sigmoid, groups=groups, top=max(1, groups // 2), best=2)


@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("case", [dict(E=256, K=6, groups=16, top=3, sigmoid=True, biased=True, dtype="bf16"), dict(E=252, K=17, d=256, groups=12, top=5, best=1, biased=True)],
                         ids=lambda c: f"E{c['E']}-K{c['K']}")
def test_a_layer_of_many_experts(case, T):
    RL.test_forward_and_backward(case, T)
