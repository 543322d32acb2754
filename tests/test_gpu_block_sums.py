"""A norm that keeps its input in 8 bits goes back the same way when x has been freed and the sum, in a buffer of the caller, written over."""
import numpy as np
import pytest

from tests.lm_util import P, ctx, normal, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", [(3, 100), (70, 1000), (40, 4096), (5, 9001)])
def test_x_and_the_sum_may_go(T, d, dtype):
    c, rng = ctx(), np.random.default_rng(T + d)
    up = lambda a, dt=dtype: P.DeviceBuffer.from_numpy(c, a, dt)  # noqa: E731
    x, r, dy, ds = (normal(rng, T, d, dtype=dtype) for _ in range(4))
    g, dyb, dsb = up(normal(rng, d) + np.float32(1), "f32"), up(dy), up(ds)
    xb, rb = up(x), up(r)
    own = P.RMSLayer(d, ctx=c, dtype=dtype, gamma=g, keep8=True)
    want = [own.forward(xb, rb).to_numpy(), own.sum.to_numpy(), own.back(dyb, dsb).to_numpy(), own.diffGamma.to_numpy()]
    assert np.array_equal(want[1], rounded(x + r, dtype))
    own.close()
    layer = P.RMSLayer(d, ctx=c, dtype=dtype, gamma=g, keep8=True)
    for into in ("x", "residual", "other"):
        xb2, rb2, other = up(x), up(r), up(x)
        s = dict(x=xb2, residual=rb2, other=other)[into]
        got = [layer.forward(xb2, rb2, sum=s).to_numpy(), s.to_numpy()]
        assert layer.sum is s
        s.upload(np.full((T, d), np.nan, np.float32))
        for b in (xb2, rb2, other):
            if b is not s:
                b.free()
        got += [layer.back(dyb, dsb).to_numpy(), layer.diffGamma.to_numpy()]
        assert all(np.array_equal(a, b) for a, b in zip(got, want)), into
        s.free()
    # whole rows go back from the caller's sum
    whole = P.RMSLayer(d, ctx=c, dtype=dtype, gamma=g)
    a = whole.forward(xb, rb).to_numpy(), whole.back(dyb).to_numpy()
    b = whole.forward(xb, rb, sum=rb).to_numpy(), whole.back(dyb).to_numpy()
    assert whole.input is rb and all(np.array_equal(p, q) for p, q in zip(a, b))
    for o in (layer, whole):
        o.close()
    for o in (g, dyb, dsb, xb, rb):
        o.free()
