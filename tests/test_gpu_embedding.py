"""Token embedding and its gradient against plain sums in 64 bits: ids that repeat, are hot, or name no row; odd widths and
addresses; sums added to what the table's gradient holds."""
import numpy as np
import pytest

from tests.lm_util import DT, U32, Buf, ctx, normal, rounded, unit, within

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1, 1), (1, 5, 8), (3, 7, 5), (64, 1000, 256), (65, 513, 100), (257, 512, 1030), (1000, 40, 33), (2999, 1537, 64), (40, 70000, 12)]


def make_ids(rng, T, V, kind):
    ids = rng.integers(0, V, T)
    if kind == "hot":            # one id has most of the tokens, its neighbour some
        ids = np.where(rng.random(T) < 0.8, V // 2, np.where(rng.random(T) < 0.5, min(V // 2 + 1, V - 1), ids))
    if kind == "padded":         # ids outside the table on both sides
        ids = np.where(rng.random(T) < 0.3, rng.choice([-1, -100, V, V + 3, -2 ** 31, 2 ** 31 - 1], T), ids)
    if kind == "none":
        ids = np.full(T, -1)
    return ids.astype(np.int32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,V,d", SHAPES)
def test_lookup(T, V, d, dtype):
    rng = np.random.default_rng(T + V + d)
    for shift, kind, scale in ((0, "any", 1.0), (1, "padded", 45.25), (0, "none", 3.0)):
        table, ids = normal(rng, V, d, dtype=dtype), make_ids(rng, T, V, kind)
        tb, ib, ob = Buf((V, d), dtype, table, shift), Buf((T,), "i32", ids, shift), Buf((T, d), dtype, shift=shift)
        ctx().check(ctx().lib.omega_hip_embedding_forward(ctx().handle, tb.ptr, DT[dtype], V, d, ib.ptr, T, scale, ob.ptr))
        held = (ids >= 0) & (ids < V)
        want = np.where(held[:, None], table[np.where(held, ids, 0)] * np.float32(scale), np.float32(0.0))
        assert np.array_equal(ob.get(), rounded(want, dtype)), (shift, kind)     # one rounding: the same bits
        for b in (tb, ib, ob):
            b.free()


def grad_reference(ids, dout, V, scale):
    """Sums, sums of magnitudes and token counts of every row."""
    ref, mag, n = np.zeros((V, dout.shape[1])), np.zeros((V, dout.shape[1])), np.zeros(V)
    held = (ids >= 0) & (ids < V)
    np.add.at(ref, ids[held], dout[held].astype(np.float64))
    np.add.at(mag, ids[held], np.abs(dout[held].astype(np.float64)))
    np.add.at(n, ids[held], 1)
    return ref * np.float64(np.float32(scale)), mag * abs(np.float64(np.float32(scale))), n


@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("T,V,d", SHAPES)
def test_gradient(T, V, d, dtype, grad):
    rng = np.random.default_rng(T * 3 + V + d)
    for shift, kind, scale, add in ((0, "any", 1.0, 0), (1, "hot", 45.25, 1), (0, "hot", 0.5, 0), (0, "padded", 2.0, 1), (1, "none", 1.0, 0)):
        ids, dout, before = make_ids(rng, T, V, kind), normal(rng, T, d, dtype=dtype), normal(rng, V, d, dtype=grad)
        ref, mag, n = grad_reference(ids, dout, V, scale)
        ib, db = Buf((T,), "i32", ids), Buf((T, d), dtype, dout, shift)
        got = []
        for _ in range(2):
            gb = Buf((V, d), grad, before if add else None, shift)
            ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, ib.ptr, T, db.ptr, DT[dtype], V, d, scale, add, gb.ptr, DT[grad]))
            got.append(gb.get())
            gb.free()
        assert np.array_equal(got[0], got[1]), "the same inputs give other bits"
        want = ref + (before if add else 0)
        # n additions and the scale's product, each within a rounding of the sum of magnitudes; the sum with what was there; the result's rounding
        tol = (n[:, None] + 2) * U32 * mag + (U32 * (np.abs(want) + mag) if add else 0) + unit(grad) * np.abs(want) * (1 + 1e-3)
        within(got[0], want, tol, (shift, kind, add))
        rows = n == 0
        assert np.array_equal(got[0][rows], before[rows] if add else np.zeros_like(got[0][rows])), "rows without tokens"
        for b in (ib, db):
            b.free()


def test_long_runs_meet_every_block_boundary():
    """Runs of 1 .. 70 and of thousands of one id, whose aligned blocks of 32 and of 1024 sorted places are summed apart."""
    rng = np.random.default_rng(5)
    ids = np.concatenate([np.full(n, v) for v, n in enumerate(list(range(1, 71)) + [1024, 2047, 4100, 31, 33])]).astype(np.int32)
    rng.shuffle(ids)
    T, V, d = len(ids), 80, 24
    dout = normal(rng, T, d, dtype="bf16")
    ref, mag, n = grad_reference(ids, dout, V, 1.0)
    ib, db, gb = Buf((T,), "i32", ids), Buf((T, d), "bf16", dout), Buf((V, d), "f32")
    ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, ib.ptr, T, db.ptr, DT["bf16"], V, d, 1.0, 0, gb.ptr, DT["f32"]))
    within(gb.get(), ref, (n[:, None] + 2) * U32 * mag, "runs")
    # no tokens: the gradient is zero, or what it was
    ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, None, 0, None, DT["bf16"], V, d, 1.0, 1, gb.ptr, DT["f32"]))
    within(gb.get(), ref, (n[:, None] + 2) * U32 * mag, "no tokens, added")
    ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, None, 0, None, DT["bf16"], V, d, 1.0, 0, gb.ptr, DT["f32"]))
    assert not gb.get().any()
    for b in (ib, db, gb):
        b.free()


def test_infinities_and_no_numbers_stay_in_their_rows():
    V, d = 9, 16
    ids = np.array([0, 1, 1, -1, 5, V], np.int32)
    dout = np.ones((6, d), np.float32)
    dout[2, 3], dout[3], dout[4, 0], dout[5] = np.nan, np.nan, np.inf, np.inf      # rows 3 and 5 belong to no id
    ib, db, gb = Buf((6,), "i32", ids), Buf((6, d), "f32", dout), Buf((V, d), "f32")
    ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, ib.ptr, 6, db.ptr, DT["f32"], V, d, 1.0, 0, gb.ptr, DT["f32"]))
    got = gb.get()
    assert np.isnan(got[1, 3]) and got[5, 0] == np.inf
    got[1, 3] = got[5, 0] = 0
    want = np.zeros((V, d))
    want[0], want[1], want[5] = 1, 2, 1
    want[1, 3] = want[5, 0] = 0
    assert np.array_equal(got, want)
    for b in (ib, db, gb):
        b.free()
