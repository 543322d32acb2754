"""Clipping of gradients that are zero for the most part, as those of an embedding's table and of experts without tokens are: zeros beside
numbers whose squares fp32 does not hold, and beside ordinary ones."""
import numpy as np
import pytest

from tests.lm_util import P, U32, Buf, ctx, rounded, unit, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 9, 8192, 100_003, 3_000_001])
def test_zeros_and_what_is_among_them(n, dtype):
    rng = np.random.default_rng(n)
    zero = np.zeros(n, np.float32)
    zero[rng.random(n) < 0.5] = -0.0
    # value, the share of elements that have it: squares below fp32's smallest, denormals (of both types), ordinary, squares beyond fp32's largest
    for value, share in ((0.0, 0.0), (1e-30, 1e-3), (1e-39, 1.0), (1e-22, 0.5), (3.0, 1e-3), (1e25, 1e-3), (1e-30, 0.0)):
        a = np.where(rng.random(n) < share, np.float32(value), zero)
        a[n // 2] = value if share == 0 else a[n // 2]                # (one element alone)
        a = rounded(a, dtype)
        norm = np.sqrt((a.astype(np.float64) ** 2).sum())
        t = Buf((n,), dtype, a, shift=n % 3)
        clip = P.GradClip(ctx(), [t.buf])
        limit = 0.5 * norm if norm > 1e-4 else 1.0
        got = clip.clip(limit).to_numpy()
        coef = min(1.0, float(np.float32(limit)) / (norm + 1e-6))
        # (the norm as a float: half a step of the denormals besides)
        assert abs(got[0] - norm) <= 2 * U32 * norm + 2.0 ** -150 and abs(got[1] - coef) <= 2 * U32 * coef, (value, share)
        if coef == 1.0:
            assert np.array_equal(t.get(), a)
        else:
            within(t.get(), a.astype(np.float64) * coef, (3 * U32 + unit(dtype)) * np.abs(a) * coef, (value, share))
        clip.close()
        t.free()
