"""A training step of a small language model: embedding, MoE block, layer norm, tied head with its loss, all the way back, clipping and
the update; the same for a single token, for several contexts and threads at once, and for batches of changing size."""
import importlib
import threading

import numpy as np
import pytest

from oracle import oracle as O
from oracle import oracle_np as N
from tests import test_gpu_embedding as TE
from tests import test_gpu_head_loss as TH
from tests import test_gpu_layernorm as TN
from tests.lm_util import U32, normal, rounded, unit, within

pytestmark = pytest.mark.gpu
P = importlib.import_module("omega-ai_amd")
L = importlib.import_module("omega-ai_amd._lib")

D, H, V = 256, 128 * 2, 515


class Model:
    """Weights on the host and the layers that hold them."""

    def __init__(self, ctx, dtype, E=4, K=2, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.dtype, self.K = ctx, dtype, K
        self.table = normal(rng, V, D, std=D ** -0.5, dtype=dtype)
        self.gamma, self.beta = normal(rng, D, std=0.1) + np.float32(1), normal(rng, D, std=0.1)
        self.norm = normal(rng, D, std=0.1) + np.float32(1)
        self.Wg = normal(rng, E, D, std=D ** -0.5, dtype=dtype)
        self.W1, self.W3 = normal(rng, E, H, D, std=D ** -0.5, dtype=dtype), normal(rng, E, H, D, std=D ** -0.5, dtype=dtype)
        self.W2 = normal(rng, E, D, H, std=H ** -0.5, dtype=dtype)
        up = lambda a, t: P.DeviceBuffer.from_numpy(ctx, a, t)
        self.weight, self.g, self.b = up(self.table, dtype), up(self.gamma, "f32"), up(self.beta, "f32")
        self.scale = D ** 0.5
        self.emb = P.EmbeddingLayer(V, D, scale=self.scale, ctx=ctx, dtype=dtype, weight=self.weight)
        self.moe = P.MoELayer(D, H, E, K, renorm=True, ctx=ctx, dtype=dtype)
        self.moe.set_gate(self.Wg)
        self.moe.set_norm(self.norm)
        for e in range(E):
            self.moe.set_expert(e, self.W1[e], self.W3[e], self.W2[e])
        self.ln = P.LNLayer(D, ctx=ctx, dtype=dtype, gamma=self.g, beta=self.b)
        self.head = P.HeadLossLayer(V, D, ctx=ctx, dtype=dtype, weight=self.weight)

    def forward(self, ids, y):
        self.ids, self.y = ids, y
        self.e = self.emb.forward(ids)
        self.h = self.moe.forward_block(self.e)
        self.n = self.ln.forward(self.h)
        return self.head.forward(self.n, y)

    def back(self):
        self.dn = self.head.back()
        self.untied = self.head.diffW.to_numpy()
        self.dh = self.ln.back(self.dn)
        self.de = self.moe.back_block(self.dh)
        return self.emb.back(self.de, diffW=self.head.diffW)

    def clip(self):
        return P.GradClip(self.ctx, [self.head.diffW, self.ln.diffGamma, self.ln.diffBeta], [self.moe])

    def close(self):
        for o in (self.emb, self.moe, self.ln, self.head):
            o.close()
        for b in (self.weight, self.g, self.b):
            b.free()


def batch(ctx, rng, T):
    ids, y = rng.integers(0, V, T), rng.integers(0, V, T)
    ids[rng.random(T) < 0.2], y[rng.random(T) < 0.2] = 7, -1      # a token that comes back often; padding
    if T > 8:
        ids[3], ids[5], y[4] = -1, V, V
    y[0] = 2
    return (P.DeviceBuffer.from_numpy(ctx, ids, "i32"), P.DeviceBuffer.from_numpy(ctx, y, "i32"), ids.astype(np.int32), y.astype(np.int32))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 33, 300])
def test_each_link_of_a_step(T, dtype):
    """Every link of the chain against its own formula, from what the link before left on the device, read after the whole step."""
    ctx = P.Context(0)
    m = Model(ctx, dtype)
    idb, yb, ids, y = batch(ctx, np.random.default_rng(T), T)
    m.moe.set_training(True)
    loss = m.forward(idb, yb)
    m.back()
    table, bf = m.table, dtype == "bf16"
    e, h, n, dn, dh, de = (b.to_numpy() for b in (m.e, m.h, m.n, m.dn, m.dh, m.de))
    held = (ids >= 0) & (ids < V)
    assert np.array_equal(e, rounded(np.where(held[:, None], table[np.where(held, ids, 0)] * np.float32(m.scale), np.float32(0)), dtype))
    tol = 1e-2 if bf else 1e-5                                    # the layer's own bounds
    blk = O.block_forward(e, m.norm, m.Wg, None, m.W1, m.W3, m.W2, m.K, True, bf16=bf)
    assert N.rel_l2(h, blk["out"]) <= tol
    ref = TN.reference(h, m.gamma, m.beta, dn)
    within(n, ref["out"][0], ref["out"][1] + unit(dtype) * np.abs(ref["out"][0]) * 1.01, "norm")
    hd = TH.reference(n, table, y, dtype)
    TH.check(dict(loss=loss.to_numpy(), dx=dn, dw=m.untied, mean=m.head.mean.to_numpy()), hd)
    within(dh, ref["dx"][0], ref["dx"][1] + unit(dtype) * np.abs(ref["dx"][0]) * 1.01, "norm's gradient")
    within(m.ln.diffGamma.to_numpy(), *ref["dgamma"], "gamma")
    within(m.ln.diffBeta.to_numpy(), *ref["dbeta"], "beta")
    bw = O.block_backward(e, m.norm, dh, m.Wg, None, m.W1, m.W3, m.W2, m.K, True, bf16=bf)
    assert N.rel_l2(de, bw["dx"]) <= tol
    g, mag, cnt = TE.grad_reference(ids, de, V, m.scale)
    want = m.untied.astype(np.float64) + g
    tied = m.head.diffW.to_numpy()
    within(tied, want, (cnt[:, None] + 4) * U32 * (mag + np.abs(m.untied)) + (cnt > 0)[:, None] * unit(dtype) * np.abs(want) * 1.01, "tied gradient")
    assert np.array_equal(tied[cnt == 0], m.untied[cnt == 0])
    # the clip over all of them and the layer, then the layer's update
    grads = [tied, m.ln.diffGamma.to_numpy(), m.ln.diffBeta.to_numpy()]
    lay = [m.moe.grad(w, g_) for w, g_, _ in m.moe._param_list()] + [m.moe.grad(L.W_NORM)]
    norm = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in grads + lay))
    c = m.clip()
    got = c.clip(0.1 * norm).to_numpy()
    coef = float(np.float32(0.1 * norm)) / (norm + 1e-6)
    assert abs(got[0] - norm) <= 8 * U32 * norm and abs(got[1] - coef) <= 8 * U32 * coef
    for b, a in zip((m.head.diffW, m.ln.diffGamma, m.ln.diffBeta), grads):
        within(b.to_numpy(), a * coef, (16 * U32 + (unit(dtype) * 1.01 if b.dtype == "bf16" else 0)) * np.abs(a) * coef)
    for (w, g_, _), a in zip(m.moe._param_list(), lay):
        within(m.moe.grad(w, g_), a * coef, 16 * U32 * np.abs(a) * coef)
    m.moe.updateAdamW(1e-3, 1)
    assert np.isfinite(m.forward(idb, yb).to_numpy()).all()
    c.close()
    m.close()
    ctx.close()


def loss64(m, ids, y, q):
    """The model's mean loss in 64 bits; q: its parameters (every expert is taken, so that nothing jumps)."""
    held = (ids >= 0) & (ids < V)
    e = np.where(held[:, None], q["table"][np.where(held, ids, 0)] * m.scale, 0.0)
    h = e / np.sqrt((e ** 2).mean(1, keepdims=True) + 1e-6) * q["norm"]
    s = h @ q["Wg"].T
    w = np.exp(s - s.max(1, keepdims=True))
    w /= w.sum(1, keepdims=True)
    o = e.copy()
    for k in range(len(q["Wg"])):
        a, b = h @ q["W1"][k].T, h @ q["W3"][k].T
        o += w[:, k:k + 1] * ((a / (1 + np.exp(-a)) * b) @ q["W2"][k].T)
    mu = o.mean(1, keepdims=True)
    n = (o - mu) / np.sqrt(((o - mu) ** 2).mean(1, keepdims=True) + TN.EPS) * q["gamma"] + q["beta"]
    l = n @ q["table"].T
    at = (y >= 0) & (y < V)
    mx = l.max(1, keepdims=True)
    lse = (np.log(np.exp(l - mx).sum(1, keepdims=True)) + mx)[:, 0]
    return np.where(at, lse - l[np.arange(len(y)), np.where(at, y, 0)], 0.0).sum() / max(at.sum(), 1)


def test_gradients_of_the_whole_step_against_differences():
    """Along its own direction a gradient of length |g| raises the loss by |g|: central differences of the model in 64 bits.  The stages
    keep 1e-5 of their results each, four forward and four back: 1e-4 of |g|."""
    ctx = P.Context(0)
    m = Model(ctx, "f32", E=2, K=2)
    rng = np.random.default_rng(5)
    idb, yb, ids, y = batch(ctx, rng, 40)
    y[7] = ids[7] = 11                                            # one row of the table from both of its sides
    idb.upload(ids)
    yb.upload(y)
    m.forward(idb, yb)
    tied = m.back().to_numpy()
    q = {k: getattr(m, k).astype(np.float64) for k in ("table", "norm", "Wg", "W1", "W3", "W2", "gamma", "beta")}
    assert abs(m.head.mean.to_numpy()[0] - loss64(m, ids, y, q)) <= 1e-5 * loss64(m, ids, y, q)
    row = np.zeros_like(tied)
    row[11] = tied[11]
    grads = dict(table=tied, gamma=m.ln.diffGamma.to_numpy(), beta=m.ln.diffBeta.to_numpy(), norm=m.moe.grad(L.W_NORM),
                 W1=np.stack([m.moe.grad(L.W_W1, e) for e in range(2)]), W2=np.stack([m.moe.grad(L.W_W2, e) for e in range(2)]))
    for what, g in list(grads.items()) + [("table", row)]:
        g = g.astype(np.float64)
        size, step = np.sqrt((g ** 2).sum()), 1e-5
        ends = [loss64(m, ids, y, {**q, what: q[what] + s * step * g / size}) for s in (1, -1)]
        assert abs((ends[0] - ends[1]) / (2 * step) - size) <= 1e-4 * size, what
    m.close()
    ctx.close()


def outcome(m, idb, yb):
    loss = m.forward(idb, yb).to_numpy()
    tied = m.back().to_numpy()
    c = m.clip()
    norm = c.clip(1.0).to_numpy()
    c.close()
    return [loss, tied, norm, m.ln.diffGamma.to_numpy(), m.de.to_numpy(), m.head.diffW.to_numpy()]


def test_batches_of_changing_size_give_the_same_bits():
    """A layer that has seen larger and smaller batches holds nothing of them."""
    ctx = P.Context(0)
    rng = np.random.default_rng(1)
    data = {T: batch(ctx, rng, T) for T in (64, 5, 300, 1)}
    want = {}
    for T, (idb, yb, _, _) in data.items():
        m = Model(ctx, "bf16")
        want[T] = outcome(m, idb, yb)
        m.close()
    m = Model(ctx, "bf16")
    for T in (300, 1, 64, 5, 300, 64):
        for a, b in zip(outcome(m, *data[T][:2]), want[T]):
            assert np.array_equal(a, b), T
    m.close()
    ctx.close()


@pytest.mark.parametrize("shared", [True, False])
def test_threads(shared):
    """Steps from several threads at once, each with its model: on contexts of their own, and on one context, whose workspace the calls
    share one after another."""
    one = P.Context(0)
    rng = np.random.default_rng(2)
    sizes, want = (40, 257, 90), []
    ctxs = [one if shared else P.Context(0) for _ in sizes]
    data = [batch(c, rng, T) for c, T in zip(ctxs, sizes)]
    models = [Model(c, "bf16" if i != 1 else "f32", seed=i) for i, c in enumerate(ctxs)]
    for m, d in zip(models, data):
        want.append(outcome(m, *d[:2]))
    got, errors = [[] for _ in sizes], []

    def work(i):
        try:
            for _ in range(4):
                got[i].append(outcome(models[i], *data[i][:2]))
        except Exception as e:                                    # (a thread's own exception would be lost)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for w, runs in zip(want, got):
        assert len(runs) == 4
        for r in runs:
            for a, b in zip(r, w):
                assert np.array_equal(a, b)
    for m in models:
        m.close()


def test_layers_refuse():
    ctx = P.Context(0)
    m = Model(ctx, "f32")
    rng = np.random.default_rng(3)
    idb, yb, _, _ = batch(ctx, rng, 12)
    x, x16 = P.DeviceBuffer(ctx, (12, D), "f32"), P.DeviceBuffer(ctx, (12, D), "bf16")
    other = P.DeviceBuffer(ctx, (13, D), "f32")
    for call in (lambda: m.emb.back(x), lambda: m.ln.back(x), lambda: m.head.back(),                       # no forward yet
                 lambda: m.emb.forward(x), lambda: m.ln.forward(x16), lambda: m.head.forward(x, x), lambda: m.head.forward(x16, yb),
                 lambda: m.head.forward(other, yb), lambda: P.EmbeddingLayer(V, D, ctx=ctx).forward(idb), lambda: P.LNLayer(D, ctx=ctx).forward(x),
                 lambda: P.HeadLossLayer(V, D, ctx=ctx).forward(x, yb), lambda: P.EmbeddingLayer(V, D, ctx=ctx, dtype="f16"),
                 lambda: P.EmbeddingLayer(V, D + 1, ctx=ctx, weight=m.weight), lambda: P.LNLayer(D, ctx=ctx, gamma=x),
                 lambda: P.HeadLossLayer(V, D, ctx=ctx, dtype="bf16", weight=m.weight), lambda: P.GradClip(ctx, [x], out=[x16]),
                 lambda: P.GradClip(ctx, [idb]), lambda: P.GradClip(ctx, [x], out=[])):
        with pytest.raises(RuntimeError, match="Error code 1"):
            call()
    m.forward(idb, yb)
    m.back()
    for call in (lambda: m.emb.back(other), lambda: m.ln.back(x16), lambda: m.head.back(dloss=x), lambda: m.emb.back(x, diffW=other)):
        with pytest.raises(RuntimeError, match="Error code 1"):
            call()
    c = m.clip()
    m.head.close()
    for call in (lambda: c.clip(1.0), lambda: m.head.back()):     # a gradient whose memory has gone, a closed layer
        with pytest.raises(RuntimeError, match="Error code 1"):
            call()
    c.close()
    c = P.GradClip(ctx, [m.ln.diffGamma, m.ln.diffBeta])
    m.ln.close()
    with pytest.raises(RuntimeError, match="Error code 1"):       # views into a buffer that has gone
        c.clip(1.0)
    c.close()
    # a forward pass that is refused leaves nothing to go back from (its output lies over the table)
    out = m.emb.forward(idb)
    own, out.ptr = out.ptr, m.weight.ptr
    with pytest.raises(RuntimeError, match="Error code 1"):
        m.emb.forward(idb)
    out.ptr = own
    with pytest.raises(RuntimeError, match="without a forward"):
        m.emb.back(x)
    m.close()
    ctx.close()
