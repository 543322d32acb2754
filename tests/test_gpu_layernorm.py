"""Layer norm, forward and backward, against the formulas in 64 bits and against differences of the forward formula."""
import numpy as np
import pytest

from tests.lm_util import DT, U32, Buf, ctx, normal, unit, within

pytestmark = pytest.mark.gpu

EPS = np.float64(np.float32(1e-5))
SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (4, 512), (7, 513), (64, 1000), (9, 2050), (3, 4096), (2, 8192), (2, 8200), (3, 9001), (600, 96), (2500, 40),
          (2100, 768), (1100, 130)]
ADDS = 100    # no sum over a row has more than this many fp32 additions behind one another: 36 elements a lane, six steps in a wave, four waves


def reference(x, gamma, beta, dy):
    x, gamma, beta, dy = (np.asarray(a, np.float64) for a in (x, gamma, beta, dy))
    mu = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + EPS)
    xh = (x - mu) * r
    g = dy * gamma
    dx = r * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    # an element of xh: the mean's additions, weighed by r, and the variance's, relative; of y and dx: what follows from it
    e = ADDS * U32 * (np.abs(xh) + r * np.abs(x).mean(1, keepdims=True))
    ey = np.abs(gamma) * e + 4 * U32 * (np.abs(xh * gamma) + np.abs(beta))
    edx = r * (ADDS * U32 * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + np.abs(xh) * np.abs(g * xh).mean(1, keepdims=True))
               + e * np.abs((g * xh).mean(1, keepdims=True)) + np.abs(xh) * (np.abs(g) * e).mean(1, keepdims=True))
    n = len(x)
    edg = (np.abs(dy) * e).sum(0) + (n + 8) * U32 * np.abs(dy * xh).sum(0)
    return dict(out=(xh * gamma + beta, ey), mean=(mu[:, 0], ADDS * U32 * np.abs(x).mean(1)), rstd=(r[:, 0], ADDS * U32 * r[:, 0] * (1 + r[:, 0] * np.abs(x).mean(1))),
                dx=(dx, edx), dgamma=((dy * xh).sum(0), edg), dbeta=(dy.sum(0), (n + 8) * U32 * np.abs(dy).sum(0)))


def run(x, gamma, beta, dy, dtype, shift, stats=True):
    T, d = x.shape
    c, lib = ctx(), ctx().lib
    b = dict(x=Buf((T, d), dtype, x, shift), gamma=Buf((d,), "f32", gamma, shift), beta=Buf((d,), "f32", beta, shift), dy=Buf((T, d), dtype, dy, shift),
             out=Buf((T, d), dtype, shift=shift), mean=Buf((T,), "f32"), rstd=Buf((T,), "f32"), dx=Buf((T, d), dtype, shift=shift),
             dgamma=Buf((d,), "f32", shift=shift), dbeta=Buf((d,), "f32", shift=shift))
    p = {k: v.ptr for k, v in b.items()}
    c.check(lib.omega_hip_layernorm_forward(c.handle, p["x"], DT[dtype], T, d, p["gamma"], p["beta"], EPS, p["out"], p["mean"] if stats else None,
                                            p["rstd"] if stats else None))
    if stats:
        c.check(lib.omega_hip_layernorm_backward(c.handle, p["x"], p["dy"], DT[dtype], T, d, p["gamma"], p["mean"], p["rstd"], p["dx"], p["dgamma"], p["dbeta"]))
    got = {k: b[k].get() for k in (("out", "mean", "rstd", "dx", "dgamma", "dbeta") if stats else ("out",))}
    for v in b.values():
        v.free()
    return got


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", SHAPES)
def test_against_the_formulas(T, d, dtype):
    rng = np.random.default_rng(T + d)
    for shift, offset in ((0, 0.3), (1, 0.0), (2, 50.0), (4, -1.0)):
        x = normal(rng, T, d, dtype=dtype) if offset == 0 else normal(rng, T, d)
        x = np.asarray(x + np.float32(offset), np.float32)
        if dtype == "bf16":
            from tests.lm_util import rounded
            x = rounded(x, dtype)
        gamma, beta, dy = normal(rng, d) + np.float32(1), normal(rng, d), normal(rng, T, d, dtype=dtype)
        ref = reference(x, gamma, beta, dy)
        got = run(x, gamma, beta, dy, dtype, shift)
        again = run(x, gamma, beta, dy, dtype, shift)
        for k, (want, tol) in ref.items():
            u = unit(dtype) * np.abs(want) * (1 + 1e-3) if k in ("out", "dx") else U32 * np.abs(want)
            within(got[k], want, tol + u, (k, shift))
            assert np.array_equal(got[k], again[k]), (k, "the same inputs give other bits")
        assert np.array_equal(run(x, gamma, beta, dy, dtype, shift, stats=False)["out"], got["out"])   # serving: no statistics kept


def test_gradients_against_differences():
    """Central differences of sum(y * dy) in 64 bits, for a few elements of x and of the parameters."""
    rng = np.random.default_rng(3)
    T, d, h = 3, 10, 1e-6
    x, gamma, beta, dy = normal(rng, T, d), normal(rng, d) + np.float32(1), normal(rng, d), normal(rng, T, d)
    got = run(x, gamma, beta, dy, "f32", 0)

    def f(x, gamma, beta):
        mu = x.mean(1, keepdims=True)
        return float((((x - mu) / np.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + EPS) * gamma + beta) * dy.astype(np.float64)).sum())

    args = [a.astype(np.float64) for a in (x, gamma, beta)]
    for k, name in enumerate(("dx", "dgamma", "dbeta")):
        for at in list(np.ndindex(args[k].shape))[::3]:
            side = []
            for s in (h, -h):
                moved = [a.copy() for a in args]
                moved[k][at] += s
                side.append(f(*moved))
            # differences: h^2 times a third derivative (of order 10) and cancellation 1e-16 / h; the gradient itself: 1e-5 of its terms
            assert abs((side[0] - side[1]) / (2 * h) - got[name][at]) < 3e-5, (name, at)


def test_rows_of_one_value_and_no_rows():
    T, d = 4, 100
    x = np.full((T, d), 2.5, np.float32)
    got = run(x, np.ones(d, np.float32), np.full(d, 0.25, np.float32), np.ones((T, d), np.float32), "f32", 0)
    assert np.array_equal(got["out"], np.full((T, d), 0.25)) and not got["dgamma"].any() and np.array_equal(got["dbeta"], np.full(d, 4.0))
    assert np.abs(got["dx"]).max() <= got["rstd"].max() * 100 * U32      # dy - mean(dy) = 0 up to the mean's roundings
    c, dg, db = ctx(), Buf((d,), "f32"), Buf((d,), "f32")
    c.check(c.lib.omega_hip_layernorm_forward(c.handle, None, DT["f32"], 0, d, None, None, 1e-5, None, None, None))
    c.check(c.lib.omega_hip_layernorm_backward(c.handle, None, None, DT["f32"], 0, d, None, None, None, None, dg.ptr, db.ptr))
    assert not dg.get().any() and not db.get().any()
    dg.free()
    db.free()


@pytest.mark.parametrize("d", [96, 1500, 9001])
def test_no_numbers_stay_in_their_rows(d):
    rng = np.random.default_rng(d)
    x, dy = normal(rng, 6, d), normal(rng, 6, d)
    x[2, 5] = np.inf
    x[4, 0] = np.nan
    got = run(x, np.ones(d, np.float32), np.zeros(d, np.float32), dy, "f32", 0)
    rows = [0, 1, 3, 5]
    clean = run(x[rows], np.ones(d, np.float32), np.zeros(d, np.float32), dy[rows], "f32", 0)
    for k in ("out", "dx"):
        assert np.array_equal(got[k][rows], clean[k]) and np.isnan(got[k][[2, 4]]).any(1).all()
