"""Routing: an expert is closed to a token by whatever bits its logit is no number, the signalling ones among them."""
import numpy as np
import pytest

from tests import test_gpu_route as R

pytestmark = pytest.mark.gpu

# quiet and signalling, of both signs, the first and the last pattern of each
NO_NUMBERS = np.array([0x7F800001, 0x7FA00000, 0x7FBFFFFF, 0x7FC00000, 0x7FFFFFFF, 0xFF800001, 0xFFBFFFFF, 0xFFC00000, 0xFFFFFFFF], np.uint32).view(np.float32)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,groups", [(20, 8, 1), (20, 60, 5), (70, 128, 1), (20, 256, 8), (20, 512, 1), (4200, 128, 8), (4200, 300, 1)])
def test_no_numbers_of_every_kind(T, E, groups, sigmoid):
    rng = np.random.default_rng(E + T)
    K = 4
    z = (rng.standard_normal((T, E)) * 1.5).astype(np.float32)
    n = len(NO_NUMBERS)
    for t in range(T):
        at = rng.choice(E, min(E // 2, 1 + t % 7), replace=False)
        z[t, at] = NO_NUMBERS[(t + np.arange(len(at))) % n]
    z[:n, 0], z[:n, E - 1] = NO_NUMBERS, NO_NUMBERS[::-1]
    z[n] = NO_NUMBERS[0]                              # nothing open
    z[n + 1, :-1] = NO_NUMBERS[1]                     # the last alone
    assert np.isnan(z[:n, 0]).all() and z[0, 0].view(np.uint32) == 0x7F800001
    b = (rng.standard_normal(E) * 0.1).astype(np.float32)
    odd = b.copy()
    odd[[1, 3, 6]] = NO_NUMBERS[[0, 5, 3]]
    dw = rng.standard_normal((T, K)).astype(np.float32)
    for bias in (None, b, odd):
        for renorm in (True, False):
            R.check(z, bias, K, dw, sigmoid=sigmoid, renorm=renorm, groups=groups, top=max(1, groups // 2), best=2)
