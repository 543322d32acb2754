"""The head with its softmax cross entropy, loss and gradients, against the formulas in 64 bits."""
import numpy as np
import pytest

from tests.lm_util import DT, U16, U32, Buf, ctx, normal, rounded, unit, within

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (1, 1000, 64), (2, 33, 7), (3, 257, 40), (16, 1000, 256), (16, 40000, 64), (17, 300, 256), (64, 512, 320), (65, 513, 333), (130, 700, 64),
          (193, 769, 260), (257, 1025, 512), (300, 256, 1000), (450, 3, 72), (300, 9000, 256), (330, 7001, 130), (70, 2500, 2100), (129, 300, 1280)]


def reference(x, w, y, dtype, dloss=1.0):
    """Values and tolerances: loss, mean, dx, dw."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    T, V, d = len(x), len(w), x.shape[1]
    held = (y >= 0) & (y < V)
    at, n = np.where(held, y, 0), max(int(held.sum()), 1)
    x = np.where(held[:, None], x, 0.0)          # (rows without a target may hold anything)
    l, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    # a logit: at most d / 32 + 32 additions of 32 bits behind one another (a factor 2 for matrix cores that cut instead of
    # rounding); fp32 operands: six products of parts behind one another and the parts left out
    el = 2 * (d / 32 + 32) * U32 * mag * (1 if dtype == "bf16" else 6) + 2 * U32 * mag
    m = l.max(1, keepdims=True)
    s = np.exp(l - m).sum(1, keepdims=True)
    p = np.exp(l - m) / s
    rows = np.arange(T)
    loss = np.where(held, (np.log(s) + m)[:, 0] - l[rows, at], 0.0)
    # exp: 2^-22 and the rounding of its argument; sums over the row: under 200 additions behind one another
    ee = 400 * U32 + 4 * U32 * np.abs(l - m)
    eloss = np.where(held, el.max(1) + el[rows, at] + 400 * U32 + 8 * U32 * np.abs(loss), 0.0)
    g = dloss / n
    P = np.where(held[:, None], p, 0.0) * g
    eP = np.abs(P) * (el + el.max(1, keepdims=True) + ee)
    P[rows[held], y[held]] -= g
    eP = np.where(held[:, None], eP + 4 * U32 * (np.abs(P) + p * abs(g)) + (U16 if dtype == "bf16" else 0) * np.abs(P), 0.0)
    # what is smaller than the smallest normal number of fp32 and bf16, 2^-126, may be lost, of each of three parts: a row that is
    # sure of its target has elements of 1e-100, which no fp32 number is near to
    eP = eP + np.where(held[:, None], 3 * 2.0 ** -126, 0.0)
    dx, dw = P @ w, P.T @ x
    # the products' own sums: over the vocabulary or the tokens
    k = 1 if dtype == "bf16" else 6
    edx = eP @ np.abs(w) + k * 2 * (V / 32 + 48) * U32 * (np.abs(P) @ np.abs(w)) + unit(dtype) * np.abs(dx) * 1.01
    edw = eP.T @ np.abs(x) + k * 2 * (T / 32 + 48) * U32 * (np.abs(P).T @ np.abs(x)) + unit(dtype) * np.abs(dw) * 1.01
    mean = loss.sum() / n
    return dict(loss=(loss, eloss), mean=(mean, eloss.max() + 4 * U32 * abs(mean)), dx=(dx, edx), dw=(dw, edw), n=int(held.sum()))


def run(x, w, y, dtype, shift=0, dloss=None, stats=True):
    (T, d), V = x.shape, len(w)
    c, lib = ctx(), ctx().lib
    b = dict(x=Buf((T, d), dtype, x, shift), w=Buf((V, d), dtype, w, shift), y=Buf((T,), "i32", y, shift), loss=Buf((T,), "f32", shift=shift),
             stats=Buf((2, T), "f32", shift=shift), mean=Buf((2,), "f32", shift=shift), dx=Buf((T, d), dtype, shift=shift), dw=Buf((V, d), dtype, shift=shift))
    p = {k: v.ptr for k, v in b.items()}
    c.check(lib.omega_hip_head_loss_forward(c.handle, p["x"], p["w"], DT[dtype], T, V, d, p["y"], p["loss"], p["stats"] if stats else None, p["mean"]))
    names = ["loss", "mean"]
    if stats:
        db = None if dloss is None else Buf((1,), "f32", [dloss])
        c.check(lib.omega_hip_head_loss_backward(c.handle, p["x"], p["w"], DT[dtype], T, V, d, p["y"], p["stats"], p["mean"], db.ptr if db else None, p["dx"], p["dw"]))
        names += ["dx", "dw", "stats"]
    got = {k: b[k].get() for k in names}
    for v in b.values():
        v.free()
    return got


def targets_of(rng, T, V, pad=0.2):
    y = rng.integers(0, V, T)
    return np.where(rng.random(T) < pad, rng.choice([-1, -100, V, 2 ** 31 - 1], T), y).astype(np.int32)


def check(got, ref, what=""):
    for k in ("loss", "dx", "dw"):
        if k in got:
            within(got[k], ref[k][0], ref[k][1], (k, what))
    assert abs(got["mean"][0] - ref["mean"][0]) <= ref["mean"][1] and got["mean"][1] == ref["n"], what


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,V,d", SHAPES)
def test_against_the_formulas(T, V, d, dtype):
    rng = np.random.default_rng(T + V + d)
    for shift, sure, dloss in ((0, 0.0, None), (1, 6.0, 0.5), (8, 12.0, -3.0)):
        w = normal(rng, V, d, std=d ** -0.5, dtype=dtype)
        y = targets_of(rng, T, V)
        x = rounded(normal(rng, T, d) + np.float32(sure) * w[np.clip(y, 0, V - 1)], dtype)
        got = run(x, w, y, dtype, shift, dloss)
        check(got, reference(x, w, y, dtype, 1.0 if dloss is None else dloss), (shift, sure))
        again = run(x, w, y, dtype, shift, dloss)
        for k in got:
            assert np.array_equal(got[k], again[k]), (k, "the same inputs give other bits")
        served = run(x, w, y, dtype, shift, stats=False)
        assert np.array_equal(served["loss"], got["loss"]) and np.array_equal(served["mean"], got["mean"])


@pytest.mark.parametrize("dtype,V", [("f32", 200001), ("bf16", 600001), ("f32", 400001), ("bf16", 1100001)])
def test_several_pieces_of_the_vocabulary(dtype, V):
    T, d = 20, 24
    rng = np.random.default_rng(V)
    w, y = normal(rng, V, d, std=0.3, dtype=dtype), targets_of(rng, T, V)
    y[:3] = 0, V - 1, V // 2
    x = normal(rng, T, d, dtype=dtype)
    check(run(x, w, y, dtype), reference(x, w, y, dtype))


def test_pieces_of_weights_in_place():
    """More tokens x vocabulary than a piece holds, bf16 rows that are read where they are, a last piece that ends inside a step of 32 rows.
    Some tokens and some rows of W against the formulas of reference(); of the rows' gradients the statistics are the call's own."""
    T, V, d = 2100, 300017, 256
    rng = np.random.default_rng(1)
    w, x, y = normal(rng, V, d, std=d ** -0.5, dtype="bf16"), normal(rng, T, d, dtype="bf16"), targets_of(rng, T, V)
    y[:3] = 0, V - 1, -1
    got = run(x, w, y, "bf16")
    held = (y >= 0) & (y < V)
    n, w = int(held.sum()), w.astype(np.float64)
    assert got["mean"][1] == n and np.isfinite(got["dw"]).all() and np.isfinite(got["dx"]).all()
    toks = np.r_[:16, rng.integers(0, T, 16), T - 1]
    part = reference(x[toks], w, y[toks], "bf16", dloss=float(held[toks].sum()) / n)
    within(got["loss"][toks], *part["loss"], "loss")
    within(got["dx"][toks], *part["dx"], "dx")
    cols = np.r_[:4, V - 40:V, rng.integers(0, V, 60), y[held][:20]]
    x = np.where(held[:, None], x, 0).astype(np.float64)
    l, mag = x @ w[cols].T, np.abs(x) @ np.abs(w[cols]).T
    m, s = (v[:, None].astype(np.float64) for v in got["stats"])
    # (a maximum of 32 bits shifts every exp of its row, and the sum with them: only how far this column's logit is off counts)
    e = 2 * (d / 32 + 32) * U32 * mag + 400 * U32 + 4 * U32 * np.abs(l - m)
    P = np.where(held[:, None], np.exp(l - m) / s, 0.0)
    eP = P * e
    P -= held[:, None] & (y[:, None] == cols)
    eP = (eP + (4 * U32 + U16) * np.abs(P) + 3 * 2.0 ** -126) * held[:, None] / n
    P /= n
    dw = P.T @ x
    within(got["dw"][cols], dw, eP.T @ np.abs(x) + 2 * (T / 32 + 48) * U32 * (np.abs(P).T @ np.abs(x)) + U16 * np.abs(dw) * 1.01, "dw")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [5, 100])
def test_far_logits(T, dtype):
    """Logits of thousands: no exp overflows, and a row that is sure of its target has no gradient to speak of."""
    rng = np.random.default_rng(T)
    V, d = 300, 64
    w, y = normal(rng, V, d, dtype=dtype), rng.integers(0, V, T).astype(np.int32)
    x = rounded(normal(rng, T, d) * 300 + np.float32(100) * w[y], dtype)
    got, ref = run(x, w, y, dtype), reference(x, w, y, dtype)
    assert np.isfinite(got["loss"]).all()
    check(got, ref)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [6, 70, 300])
def test_rows_without_a_target_hold_anything(T, dtype):
    rng = np.random.default_rng(T)
    V, d = 500, 128
    w, y = normal(rng, V, d, std=0.1, dtype=dtype), targets_of(rng, T, V, 0.4)
    y[0], y[1] = -1, 3
    x = normal(rng, T, d, dtype=dtype)
    ref = reference(x, w, y, dtype)
    x[y < 0], x[0, :] = np.nan, np.inf
    x[y >= V] = -np.inf
    got = run(x, w, y, dtype)
    check(got, ref)
    assert not got["dx"][(y < 0) | (y >= V)].any() and not got["loss"][(y < 0) | (y >= V)].any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", [(1, 256), (16, 64), (17, 72), (32, 200), (33, 136), (64, 1000), (65, 40), (100, 68), (128, 132), (129, 72), (5, 63), (40, 33)])
def test_few_tokens_and_a_large_vocabulary(T, d, dtype):
    """Forward passes that stream the head's weights: rows of whole lines, of whole 16-byte pieces and of neither."""
    V = 16384 + 77
    rng = np.random.default_rng(T + d)
    w, y = normal(rng, V, d, std=d ** -0.5, dtype=dtype), targets_of(rng, T, V)
    y[0] = V - 1
    x = rounded(normal(rng, T, d) + np.float32(5) * w[np.clip(y, 0, V - 1)], dtype)
    for shift in (0, 1):
        check(run(x, w, y, dtype, shift, stats=False), reference(x, w, y, dtype), shift)


@pytest.mark.parametrize("dtype,d", [("f32", 260), ("bf16", 260), ("bf16", 256)])
@pytest.mark.parametrize("T,pad", [(600, 0.97), (600, 0.6), (1000, 0.75), (300, 0.997), (300, 1.0), (70, 0.9)])
def test_most_tokens_have_no_target(T, pad, d, dtype):
    """The products work on the others, moved together: fewer rows than tiles, steps and statistics were laid out for."""
    rng = np.random.default_rng(T + d)
    V = 700
    w, y = normal(rng, V, d, std=d ** -0.5, dtype=dtype), targets_of(rng, T, V, pad)
    if pad < 1.0:
        y[-1] = V - 1
    x = normal(rng, T, d, dtype=dtype)
    ref = reference(x, w, y, dtype)
    x[(y < 0) | (y >= V)] = np.nan
    check(run(x, w, y, dtype), ref)


def test_no_target_at_all_and_no_rows():
    rng = np.random.default_rng(0)
    for T in (4, 40):
        x, w = normal(rng, T, 64), normal(rng, 100, 64)
        got = run(x, w, np.full(T, -1, np.int32), "f32")
        assert not got["loss"].any() and np.array_equal(got["mean"], [0, 0]) and not got["dx"].any() and not got["dw"].any()
    c, mean, w, dw = ctx(), Buf((2,), "f32"), Buf((5, 3), "bf16", np.ones((5, 3))), Buf((5, 3), "bf16")
    c.check(c.lib.omega_hip_head_loss_forward(c.handle, None, w.ptr, DT["bf16"], 0, 5, 3, None, None, None, mean.ptr))
    c.check(c.lib.omega_hip_head_loss_backward(c.handle, None, w.ptr, DT["bf16"], 0, 5, 3, None, None, mean.ptr, None, None, dw.ptr))
    assert np.array_equal(mean.get(), [0, 0]) and not dw.get().any()
    for b in (mean, w, dw):
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [4, 80])
def test_no_numbers_stay_in_their_rows(T, dtype):
    """A row of x with a target and an infinity in it has no loss; the others have theirs."""
    rng = np.random.default_rng(T)
    V, d = 200, 64
    w, y = normal(rng, V, d, std=0.1, dtype=dtype), rng.integers(0, V, T).astype(np.int32)
    x = normal(rng, T, d, dtype=dtype)
    ref = reference(x, w, y, dtype)
    x[2, 9] = np.nan
    x[3, 1] = np.inf
    got = run(x, w, y, dtype)
    rest = [t for t in range(T) if t not in (2, 3)]
    within(got["loss"][rest], ref["loss"][0][rest], ref["loss"][1][rest])
    within(got["dx"][rest], ref["dx"][0][rest], ref["dx"][1][rest])
    assert not np.isfinite(got["loss"][[2, 3]]).any() and not np.isfinite(got["mean"][0]) and np.isnan(got["dx"][[2, 3]]).all()


def test_gradients_against_differences():
    """Central differences of the mean loss in 64 bits, for a few elements."""
    rng = np.random.default_rng(9)
    T, V, d, h = 5, 11, 8, 1e-5
    x, w, y = normal(rng, T, d), normal(rng, V, d), np.array([3, -1, 10, 0, 3], np.int32)
    got = run(x, w, y, "f32")

    def f(x, w):
        l = x @ w.T
        l = l - l.max(1, keepdims=True)
        held = y >= 0
        return float((np.log(np.exp(l).sum(1)) - l[np.arange(T), np.where(held, y, 0)])[held].mean())

    args = [x.astype(np.float64), w.astype(np.float64)]
    for k, name in enumerate(("dx", "dw")):
        for at in list(np.ndindex(args[k].shape))[::7]:
            side = []
            for s in (h, -h):
                moved = [a.copy() for a in args]
                moved[k][at] += s
                side.append(f(*moved))
            # h^2 times third derivatives (below 100) and 1e-16 / h; the gradient itself: 1e-6 of its terms
            assert abs((side[0] - side[1]) / (2 * h) - got[name][at]) < 2e-6, (name, at)


@pytest.mark.parametrize("wanted", ["dx", "dw"])
def test_one_gradient_alone(wanted):
    rng = np.random.default_rng(4)
    T, V, d = 90, 600, 256
    c, lib = ctx(), ctx().lib
    x, w, y = normal(rng, T, d, dtype="bf16"), normal(rng, V, d, std=0.1, dtype="bf16"), targets_of(rng, T, V)
    both = run(x, w, y, "bf16")
    b = [Buf((T, d), "bf16", x), Buf((V, d), "bf16", w), Buf((T,), "i32", y), Buf((T,), "f32"), Buf((2, T), "f32"), Buf((2,), "f32"),
         Buf((T, d) if wanted == "dx" else (V, d), "bf16")]
    p = [v.ptr for v in b]
    c.check(lib.omega_hip_head_loss_forward(c.handle, p[0], p[1], DT["bf16"], T, V, d, p[2], p[3], p[4], p[5]))
    c.check(lib.omega_hip_head_loss_backward(c.handle, p[0], p[1], DT["bf16"], T, V, d, p[2], p[4], p[5], None, p[6] if wanted == "dx" else None,
                                             p[6] if wanted == "dw" else None))
    assert np.array_equal(b[6].get(), both[wanted])
    for v in b:
        v.free()
