"""Layer norm where a workgroup takes three rows or more, for every number of lanes that share a row: the next row is asked for while one
is worked on, and the words of LDS that carry a row's sums are used in turn."""
import numpy as np
import pytest

from tests.lm_util import U32, normal, rounded, unit, within
from tests.test_gpu_layernorm import reference, run

pytestmark = pytest.mark.gpu

# lanes a row: 64, 256, 512, 1024; a forward launch has 2048 lanes a compute unit, at 64 lanes four rows a workgroup
SHAPES = [(20000, 40), (17000, 100), (6200, 520), (2150, 2056), (2100, 4096), (1100, 4104), (1030, 8192)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", SHAPES)
def test_rows_in_turn(T, d, dtype):
    rng = np.random.default_rng(T + d)
    # rows of very different size, so that a sum of the wrong row shows
    x = rounded(normal(rng, T, d) * np.exp(rng.standard_normal((T, 1))).astype(np.float32) + np.float32(0.3), dtype)
    gamma, beta, dy = normal(rng, d) + np.float32(1), normal(rng, d), normal(rng, T, d, dtype=dtype)
    got, again = run(x, gamma, beta, dy, dtype, 1), run(x, gamma, beta, dy, dtype, 1)
    for k, (want, tol) in reference(x, gamma, beta, dy).items():
        u = unit(dtype) * np.abs(want) * (1 + 1e-3) if k in ("out", "dx") else U32 * np.abs(want)
        within(got[k], want, tol + u, k)
        assert np.array_equal(got[k], again[k]), (k, "the same inputs give other bits")
