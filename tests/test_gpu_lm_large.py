"""The operators around the layer at numbers of rows that take several launches, and in tensors whose elements are counted in more than
32 bits.  Large tensors are read and written where it tells: their first and last rows and those around 2^32 elements."""
import numpy as np
import pytest

from tests.lm_util import DT, P, U16, U32, within

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    c = P.Context(0)      # (a workspace of its own, given back behind each test)
    yield c
    c.close()


class Big:
    """A device tensor [n, d] that is written and read by rows."""

    def __init__(self, ctx, n, d, dtype, std=None):
        self.ctx, self.n, self.d, self.dtype = ctx, n, d, dtype
        self.buf = P.DeviceBuffer(ctx, (n, d), dtype)
        if std is not None:
            self.buf.fill_normal(1, 2, std)

    def rows(self, at, n=1):
        return P.DeviceBuffer.wrap(self.ctx, self.buf.ptr.value + at * self.d * self.buf.esize, (n, self.d), self.dtype)

    def put(self, at, values):
        values = np.atleast_2d(values)
        self.rows(at, len(values)).upload(values)

    def get(self, at, n=1):
        return self.rows(at, n).to_numpy()


def some_rows(n, d):
    """Row numbers of a tensor [n, d] where addresses can go wrong."""
    at = {0, 1, n // 2, n - 2, n - 1}
    for bits in (31, 32, 33):
        at |= {r for r in ((1 << bits) // d - 1, (1 << bits) // d, (1 << bits) // d + 1) if 0 <= r < n}
    return sorted(at)


def test_lookup_of_several_launches(ctx):
    rng = np.random.default_rng(0)
    T, V, d = 2 * (1 << 22) + 5, 1000, 2
    table, ids = rng.standard_normal((V, d)).astype(np.float32), rng.integers(-1, V, T).astype(np.int32)
    tb, ib, ob = (P.DeviceBuffer.from_numpy(ctx, table, "f32"), P.DeviceBuffer.from_numpy(ctx, ids, "i32"), P.DeviceBuffer(ctx, (T, d), "f32"))
    ctx.check(ctx.lib.omega_hip_embedding_forward(ctx.handle, tb.ptr, DT["f32"], V, d, ib.ptr, T, 3.0, ob.ptr))
    assert np.array_equal(ob.to_numpy(), np.where(ids[:, None] >= 0, table[ids] * np.float32(3.0), np.float32(0)))
    for b in (tb, ib, ob):
        b.free()


@pytest.mark.parametrize("add", [0, 1])
def test_gradient_of_several_launches(ctx, add):
    rng = np.random.default_rng(1)
    T, V, d = 5000, 2 * (1 << 22) + 21, 5
    ids = rng.integers(0, V, T).astype(np.int32)
    ids[:100], ids[100:200], ids[200:203] = 1 << 22, (1 << 22) - 1, (0, V - 1, V)
    dout, before = rng.standard_normal((T, d)).astype(np.float32), rng.standard_normal((V, d)).astype(np.float32)
    ib, db, gb = (P.DeviceBuffer.from_numpy(ctx, ids, "i32"), P.DeviceBuffer.from_numpy(ctx, dout, "f32"), P.DeviceBuffer.from_numpy(ctx, before, "f32"))
    ctx.check(ctx.lib.omega_hip_embedding_backward(ctx.handle, ib.ptr, T, db.ptr, DT["f32"], V, d, 1.0, add, gb.ptr, DT["f32"]))
    want, mag = (before.astype(np.float64) if add else np.zeros((V, d))), np.zeros((V, d))
    mag += np.abs(want)
    held = ids < V
    np.add.at(want, ids[held], dout[held].astype(np.float64))
    np.add.at(mag, ids[held], np.abs(dout[held]))
    n = np.bincount(ids[held], minlength=V)[:, None]
    within(gb.to_numpy(), want, (n + 1) * U32 * mag * (n > 0))
    for b in (ib, db, gb):
        b.free()


def test_head_of_several_launches(ctx):
    rng = np.random.default_rng(2)
    T, V, d = (1 << 18) + 77, 3, 4
    x, w, y = rng.standard_normal((T, d)).astype(np.float32), rng.standard_normal((V, d)).astype(np.float32), rng.integers(-1, V, T).astype(np.int32)
    b = [P.DeviceBuffer.from_numpy(ctx, x, "f32"), P.DeviceBuffer.from_numpy(ctx, w, "f32"), P.DeviceBuffer.from_numpy(ctx, y, "i32")]
    head = P.HeadLossLayer(V, d, ctx=ctx, weight=b[1])
    loss, dx = head.forward(b[0], b[2]).to_numpy(), head.back().to_numpy()
    x, w, held = x.astype(np.float64), w.astype(np.float64), y >= 0
    l = x @ w.T
    lse = np.log(np.exp(l).sum(1))
    p = np.exp(l - lse[:, None])
    p[held, y[held]] -= 1
    n = held.sum()
    assert tuple(head.mean.to_numpy()[1:]) == (n,)
    # logits of up to 4 terms in six products of parts, exponentials of 2^-21, sums of three
    mag = (np.abs(x) @ np.abs(w).T).max(1)
    within(loss, np.where(held, lse - l[np.arange(T), y], 0.0), np.where(held, 32 * U32 * (mag + 1), 0.0))
    within(dx, np.where(held[:, None], p @ w / n, 0.0), np.where(held, 64 * U32 * (mag + 1), 0.0)[:, None] * np.abs(w).sum(0) / n)
    head.close()
    for v in b:
        v.free()


def test_more_than_32_bits_of_a_table(ctx):
    """Rows looked up in a table of 5e9 elements, and its gradient: those of the tokens, zeros elsewhere."""
    rng = np.random.default_rng(3)
    V, d = 4_900_001, 1030
    some = some_rows(V, d)
    ids = np.repeat(np.array(some, np.int32), 3)
    rng.shuffle(ids)
    T = len(ids)
    table = Big(ctx, V, d, "bf16")
    known = {v: P.bf16_bits_to_f32(P.f32_to_bf16_bits(rng.standard_normal(d))) for v in some}
    for v, row in known.items():
        table.put(v, row)
    ib, ob = P.DeviceBuffer.from_numpy(ctx, ids, "i32"), P.DeviceBuffer(ctx, (T, d), "bf16")
    ctx.check(ctx.lib.omega_hip_embedding_forward(ctx.handle, table.buf.ptr, DT["bf16"], V, d, ib.ptr, T, 1.0, ob.ptr))
    out = ob.to_numpy()
    assert np.array_equal(out, np.stack([known[v] for v in ids]))
    # the gradient of those rows, in the table's place
    for v in some:
        table.put(max(v - 1, 0), np.full(d, np.nan))
    ctx.check(ctx.lib.omega_hip_embedding_backward(ctx.handle, ib.ptr, T, ob.ptr, DT["bf16"], V, d, 2.0, 0, table.buf.ptr, DT["bf16"]))
    for v in some:
        within(table.get(v)[0], 6.0 * known[v].astype(np.float64), (4 * U32 + U16) * 6.0 * np.abs(known[v]))
        for w in (v - 1, v + 1):
            assert not 0 <= w < V or w in known or not table.get(w).any()
    for b in (ib, ob, table.buf):
        b.free()


def test_more_than_32_bits_of_rows(ctx):
    """Layer norm of 5e9 elements, forward and backward."""
    T, d = 610_001, 8192
    some = some_rows(T, d)
    x, dy, out = Big(ctx, T, d, "bf16", 1.5), Big(ctx, T, d, "bf16", 1.0), Big(ctx, T, d, "bf16")
    g, b = (P.DeviceBuffer.from_numpy(ctx, a, "f32") for a in (np.full(d, 2.0), np.full(d, 0.5)))
    stats, dpar = P.DeviceBuffer(ctx, (2, T), "f32"), P.DeviceBuffer(ctx, (2, d), "f32")
    ctx.check(ctx.lib.omega_hip_layernorm_forward(ctx.handle, x.buf.ptr, DT["bf16"], T, d, g.ptr, b.ptr, 1e-5, out.buf.ptr, stats.ptr, stats.ptr.value + 4 * T))
    normed = {}
    for t in some:
        v = x.get(t)[0].astype(np.float64)
        normed[t] = (v - v.mean()) / np.sqrt(v.var() + 1e-5)
        within(out.get(t)[0], 2 * normed[t] + 0.5, 200 * U32 * (np.abs(normed[t]) + 1) + U16 * np.abs(2 * normed[t] + 0.5) * 1.01, t)
    ctx.check(ctx.lib.omega_hip_layernorm_backward(ctx.handle, x.buf.ptr, dy.buf.ptr, DT["bf16"], T, d, g.ptr, stats.ptr, stats.ptr.value + 4 * T, out.buf.ptr,
                                                   dpar.ptr, dpar.ptr.value + 4 * d))
    rstd = stats.to_numpy()[1]
    for t in some:
        q, xh = 2.0 * dy.get(t)[0].astype(np.float64), normed[t]
        want = float(rstd[t]) * (q - q.mean() - xh * (q * xh).mean())
        within(out.get(t)[0], want, 400 * U32 * (np.abs(q) + np.abs(xh) + 1) + U16 * np.abs(want) * 1.01, t)
    for v in (x.buf, dy.buf, out.buf, g, b, stats, dpar):
        v.free()


@pytest.mark.parametrize("T", [3, 150])
def test_more_than_32_bits_of_a_vocabulary(ctx, T):
    """The head over 4.9e9 weights, all zero but a few rows: loss and gradients."""
    rng = np.random.default_rng(T)
    V, d = 2_400_001, 2048
    some = some_rows(V, d)
    w = Big(ctx, V, d, "bf16", 0.0)
    rows = P.bf16_bits_to_f32(P.f32_to_bf16_bits(rng.standard_normal((len(some), d)) * d ** -0.5 * 3))
    for v, row in zip(some, rows):
        w.put(v, row)
    zero = some[2] + 5                                            # a row of zeros that is some tokens' target
    y = rng.choice(np.array(some + [zero], np.int32), T)
    y[0], y[1] = V - 1, -1
    x = P.bf16_bits_to_f32(P.f32_to_bf16_bits(rng.standard_normal((T, d))))
    xb, yb = P.DeviceBuffer.from_numpy(ctx, x, "bf16"), P.DeviceBuffer.from_numpy(ctx, y, "i32")
    head = P.HeadLossLayer(V, d, ctx=ctx, dtype="bf16", weight=w.buf)
    loss = head.forward(xb, yb).to_numpy()
    held = y >= 0
    x, rows = x.astype(np.float64), rows.astype(np.float64)
    l = x @ rows.T
    lse = np.log(np.exp(l).sum(1) + (V - len(some)))
    col = np.array([some.index(t) if t in some else -1 for t in y])
    want = np.where(held, lse - np.where(col >= 0, l[np.arange(T), col], 0.0), 0.0)
    mag = np.abs(x) @ np.abs(rows).T
    el = 2 * (d / 32 + 32) * U32 * mag.max(1) + 800 * U32         # a logit's sum; exponentials and their sum over the vocabulary
    within(loss, want, np.where(held, 2 * el + 8 * U32 * np.abs(want), 0.0))
    dx = head.back().to_numpy()
    n = held.sum()
    p = np.exp(l - lse[:, None])
    e = (el[:, None] + 4 * U32 + U16) * p
    q = p - (col[:, None] == np.arange(len(some)))
    e = np.where(col[:, None] == np.arange(len(some)), e + (U16 + 4 * U32) * np.abs(q), e)
    dxw = np.where(held[:, None], q @ rows, 0.0) / n
    within(dx, dxw, np.where(held[:, None], e @ np.abs(rows) + 400 * U32 * (np.abs(q) @ np.abs(rows)), 0.0) / n + U16 * np.abs(dxw) * 1.01)
    q, e, x = q[held], e[held], x[held]
    dw = Big.__new__(Big)
    dw.ctx, dw.n, dw.d, dw.dtype, dw.buf = ctx, V, d, "bf16", head.diffW
    for k, v in enumerate(some):
        ref = q[:, k] @ x / n
        within(dw.get(v)[0], ref, (e[:, k] @ np.abs(x) + 400 * U32 * (np.abs(q[:, k]) @ np.abs(x))) / n + U16 * np.abs(ref) * 1.01, v)
    p0 = np.exp(-lse[held])
    q0 = p0 - (y[held] == zero)
    for v in (zero, some[3] - 7):                                 # rows of zeros, with and without a target
        q = q0 if v == zero else p0
        ref = q @ x / n
        within(dw.get(v)[0], ref, ((U16 + 2 * el[held] + 8 * U32) * np.abs(q)) @ np.abs(x) / n + U16 * np.abs(ref) * 1.01, v)
    head.close()
    for b in (w.buf, xb, yb):
        b.free()


def test_few_tokens_and_more_rows_than_a_launch_streams(ctx):
    rng = np.random.default_rng(6)
    T, V, d = 2, (1 << 29) + 3, 1
    w = Big(ctx, V, d, "bf16", 0.0)
    w.put(V - 1, [[1.0]])
    w.put(5, [[-2.0]])
    xb, yb = P.DeviceBuffer.from_numpy(ctx, np.array([[2.0], [1.5]]), "bf16"), P.DeviceBuffer.from_numpy(ctx, np.array([V - 1, 7]), "i32")
    head = P.HeadLossLayer(V, d, ctx=ctx, dtype="bf16", weight=w.buf)
    loss = head.forward(xb, yb).to_numpy()
    x = np.array([2.0, 1.5])
    want = np.log(np.exp(x) + np.exp(-2 * x) + V - 2) - np.array([2.0, 0.0])
    within(loss, want, 64 * U32 * want)
    head.close()
    for b in (w.buf, xb, yb):
        b.free()


def test_clip_of_a_tensor_that_takes_several_launches(ctx):
    """A tensor of 2^33 elements and more, whose chunks (2^20 a launch) are in two tables, and one behind it: zeros but for a few elements."""
    d = 4096
    n = (1 << 33) // d + 3
    g, h = Big(ctx, n, d, "bf16", 0.0), Big(ctx, 2, d, "bf16", 0.0)
    at = [0, 1, (1 << 31) // d, (1 << 32) // d - 1, (1 << 32) // d, n - 5, n - 4, n - 3, n - 2, n - 1]
    for k, r in enumerate(at):
        g.put(r, np.full(d, k + 1.0))
    h.put(1, np.full(d, 16.0))
    clip = P.GradClip(ctx, [g.buf, h.buf])
    norm = np.sqrt(d * (sum((k + 1.0) ** 2 for k in range(len(at))) + 256.0))
    got = clip.clip(0.5 * norm).to_numpy()
    coef = float(np.float32(0.5 * norm)) / (norm + 1e-6)
    assert abs(got[0] - norm) <= 2 * U32 * norm and abs(got[1] - coef) <= 2 * U32 * coef
    for k, r in enumerate(at):
        within(g.get(r)[0], np.full(d, (k + 1.0) * coef), (3 * U32 + U16) * (k + 1.0) * coef, r)
    within(h.get(1)[0], np.full(d, 16.0 * coef), (3 * U32 + U16) * 16.0 * coef)
    assert not g.get(2)[0].any() and not g.get(n - 6)[0].any() and not h.get(0)[0].any()
    clip.close()
    g.buf.free()
    h.buf.free()
