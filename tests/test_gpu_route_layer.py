"""A MoE layer with a routing of its own: the choice on its own gate logits against the definition, outputs and gradients against the dense formulas in
64 bits, the step of the bias for balance, and what a caller may do around it."""
import io

import numpy as np
import pytest

from oracle import oracle_np as N
from tests import block_util as B
from tests.lm_util import L, P, U32, ctx, normal, rounded, within

pytestmark = pytest.mark.gpu


class Case:
    """A layer and its weights on the host."""

    def __init__(self, E, K, dtype="f32", d=256, H=256, shared=0, gate_bias=False, mode="exact", seed=0, **route):
        rng = np.random.default_rng(seed)
        self.E, self.K, self.dtype, self.d, self.H, self.shared, self.route = E, K, dtype, d, H, shared, route
        G = E + shared
        self.Wg = normal(rng, E, d, std=1.5 * d ** -0.5, dtype=dtype)
        self.bg = normal(rng, E, std=0.3) if gate_bias else None
        self.W1, self.W3 = normal(rng, G, H, d, std=d ** -0.5, dtype=dtype), normal(rng, G, H, d, std=d ** -0.5, dtype=dtype)
        self.W2 = normal(rng, G, d, H, std=H ** -0.5, dtype=dtype)
        self.biased = route.pop("biased", False)
        self.bias = normal(rng, E, std=0.2 if route.get("sigmoid") else 0.5 / E) if self.biased else None
        self.layer = P.MoELayer(d, H, E, K, nShared=shared, bias=gate_bias, ctx=ctx(), dtype=dtype, router_mode=mode)
        self.layer.set_gate(self.Wg, self.bg)
        for g in range(G):
            self.layer.set_expert(g, self.W1[g], self.W3[g], self.W2[g])
        self.config = P.route_config(E, K, score="sigmoid" if route.get("sigmoid") else "softmax", renorm=route.get("renorm", True), scale=route.get("scale", 1.0),
                                     nGroups=route.get("groups", 1), topGroups=route.get("top"), groupBest=route.get("best", 2))
        self.layer.set_routing(self.config, self.biased)
        if self.biased:
            self.layer.set_balance(self.bias)

    def up(self, a):
        return P.DeviceBuffer.from_numpy(ctx(), a, self.dtype)

    def experts(self, x):
        """Every expert's output for every token in 64 bits [G,T,d] (a rounded to bf16 in a bf16 layer)."""
        x = x.astype(np.float64)
        out = []
        for g in range(self.E + self.shared):
            h1, h3 = x @ self.W1[g].T.astype(np.float64), x @ self.W3[g].T.astype(np.float64)
            a = h1 / (1 + np.exp(-h1)) * h3
            if self.dtype == "bf16":
                a = rounded(a, "bf16").astype(np.float64)
            out.append(a @ self.W2[g].T.astype(np.float64))
        return np.stack(out)

    def wanted(self, logits):
        return B.route(logits, self.bias, self.K, fill=True, **self.route)


CASES = [dict(E=8, K=2, sigmoid=True, biased=True), dict(E=8, K=3, dtype="bf16", renorm=False, scale=2.0), dict(E=16, K=4, groups=4, top=2, dtype="bf16", sigmoid=True),
         dict(E=24, K=6, shared=1, sigmoid=True, renorm=False, biased=True, gate_bias=True), dict(E=64, K=8, dtype="bf16", shared=1, groups=8, top=3, sigmoid=True, biased=True,
                                                                                                 scale=2.5), dict(E=40, K=5, dtype="bf16", mode="fast", groups=5, top=2, best=1),
         dict(E=200, K=7, d=256, groups=20, top=4, best=1, biased=True), dict(E=130, K=3, dtype="bf16", sigmoid=True, renorm=False, biased=True)]


@pytest.mark.parametrize("T", [1, 17, 64, 300])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()))
def test_forward_and_backward(case, T):
    c = Case(**case)
    rng = np.random.default_rng(T)
    x, dout = normal(rng, T, c.d, dtype=c.dtype), normal(rng, T, c.d, dtype=c.dtype)
    xb, db = c.up(x), c.up(dout)
    logits, _ = c.layer.router_probs(xb, T)
    ids, w, counts, s = c.wanted(logits)
    for training in (False, True):
        c.layer.set_training(training)
        out = c.layer.forward(xb).to_numpy()
        r = c.layer.routing()
        assert np.array_equal(r["ids"], ids) and np.array_equal(r["counts"], counts)
        # weights: as in the operator's tests (logits here within 20 of each other)
        within(r["w"], w, 60 * U32 * np.abs(w), "w")
        order = np.argsort(ids.reshape(-1), kind="stable")
        assert np.array_equal(r["offsets"], np.concatenate([[0], np.cumsum(counts)])) and np.array_equal(r["src_row"], order // c.K)
        ys = c.experts(x)
        y = np.take_along_axis(ys[:c.E].transpose(1, 0, 2), ids[:, :, None].astype(np.int64), 1)
        want = (w[:, :, None] * y).sum(1) + ys[c.E:].sum(0)
        assert N.rel_l2(out, want) <= (1e-5 if c.dtype == "f32" else 1e-2)
        dx = c.layer.back(db).to_numpy()
        # the gradient of the weights is that of the layer's own y; of the logits by the definition
        yk = c.layer.workspace("y", T)[r["dst"]].reshape(T, c.K, c.d).astype(np.float64)
        dw = (yk * dout[:, None].astype(np.float64)).sum(2)
        size = (np.abs(yk) * np.abs(dout[:, None])).sum(2)
        args = {k: c.route.get(k, v) for k, v in (("sigmoid", False), ("renorm", True))}
        dz, terms = B.route_back(logits, s, ids, r["w"], dw, c.route.get("scale", 1.0), **args)
        _, over = B.route_back(logits, s, ids, r["w"], size, c.route.get("scale", 1.0), **args)
        reach = np.abs(over) + np.abs(r["w"]).sum(1, keepdims=True) * size.max(1, keepdims=True)
        got = c.layer.workspace("dlogits", T)
        # a product of d terms: d + 8 fp32 roundings of what is summed, which reaches the logits by weights of at most their sum; then the operator's own
        within(got, dz, (c.d + 8) * U32 * 2 * reach + 90 * U32 * terms, "dlogits")
        assert N.rel_l2(c.layer.grad(L.W_GATE), got.astype(np.float64).T @ x.astype(np.float64)) <= 1e-5
        # the input's gradient: through the experts, and through the gate
        if c.dtype == "f32" and T <= 64:
            gx = got.astype(np.float64) @ c.Wg.astype(np.float64)
            x64 = x.astype(np.float64)
            for g in range(c.E + c.shared):
                rows = np.arange(T) if g >= c.E else np.nonzero((ids == g).any(1))[0]
                if not len(rows):
                    continue
                part = np.ones(len(rows)) if g >= c.E else (np.where(ids == g, w, 0).sum(1))[rows]
                W1, W3, W2 = (a[g].astype(np.float64) for a in (c.W1, c.W3, c.W2))
                h1, h3 = x64[rows] @ W1.T, x64[rows] @ W3.T
                sg = 1 / (1 + np.exp(-h1))
                da = (part[:, None] * dout[rows].astype(np.float64)) @ W2
                gx[rows] += (da * h3 * sg * (1 + h1 * (1 - sg))) @ W1 + (da * h1 * sg) @ W3
            assert N.rel_l2(dx, gx) <= 2e-5
    xb.free()
    db.free()
    c.layer.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_block_form_and_stages(dtype):
    c = Case(32, 4, dtype=dtype, sigmoid=True, biased=True, groups=4, top=2)
    rng = np.random.default_rng(1)
    T = 150
    x, gamma = normal(rng, T, c.d, dtype=dtype), normal(rng, c.d, std=0.1) + np.float32(1)
    xb = c.up(x)
    c.layer.set_norm(gamma)
    out = c.layer.forward_block(xb).to_numpy()
    r = c.layer.routing()
    # the same by the stages, on the normalised rows that the block form gathered
    h = np.zeros((T, c.d), np.float32)
    h[r["src_row"]] = c.layer.workspace("xg", T)
    hb, o = c.up(h), P.DeviceBuffer(ctx(), (T, c.d), dtype)
    for name, kw in (("router", dict(x=hb)), ("dispatch", dict(x=hb)), ("experts", dict(x=hb)), ("combine", dict(out=o))):
        c.layer.stage(name, **kw)
    by_stages, again = o.to_numpy(), c.layer.routing()
    assert all(np.array_equal(r[k], again[k]) for k in r)
    assert N.rel_l2(by_stages + x, out) <= (1e-6 if dtype == "f32" else 1e-2)
    assert np.array_equal(c.layer.forward(hb).to_numpy(), by_stages)
    for b in (xb, hb, o):
        b.free()
    c.layer.close()


def test_balance_steps_and_leaves_the_backward_pass_alone():
    c = Case(16, 2, sigmoid=True, biased=True, seed=3)
    rng = np.random.default_rng(2)
    T = 400
    xb, db = c.up(normal(rng, T, c.d)), c.up(normal(rng, T, c.d))
    c.layer.set_balance(np.zeros(16, np.float32))
    for step in range(10):
        c.layer.forward(xb)
        counts = c.layer.routing()["counts"]
        first = c.layer.back(db).to_numpy()
        before = c.layer.balance_bias()
        c.layer.balance(0.02)
        assert np.array_equal(c.layer.balance_bias(), before + np.float32(0.02) * np.sign(T * 2 - counts * 16).astype(np.float32))
        assert np.array_equal(c.layer.back(db).to_numpy(), first)         # of the choice that was made
        c.layer.updateAdamW(0.0, step + 1)                                # no step of an optimiser moves it
    assert np.array_equal(c.layer.balance_bias(), before + np.float32(0.02) * np.sign(T * 2 - counts * 16).astype(np.float32))
    xb.free()
    db.free()
    c.layer.close()


def test_rows_of_no_numbers_stay_in_their_rows():
    for dtype in ("f32", "bf16"):
        c = Case(12, 3, dtype=dtype, sigmoid=True, biased=True, groups=3, top=1)
        rng = np.random.default_rng(4)
        x = normal(rng, 90, c.d, dtype=dtype)
        clean = c.layer.forward(c.up(x)).to_numpy()
        x[5, 7], x[40] = np.nan, np.inf
        out = c.layer.forward(c.up(x)).to_numpy()
        r = c.layer.routing()
        assert np.array_equal(r["ids"][5], [0, 1, 2]) and not r["w"][5].any() and np.isnan(out[5]).any()
        rest = [t for t in range(90) if t not in (5, 40)]
        assert np.array_equal(out[rest], clean[rest]) and (r["ids"] >= 0).all() and (r["ids"] < 12).all()
        c.layer.close()


def test_back_to_the_softmax_top_k_and_checkpoints():
    c = Case(8, 2, sigmoid=True, biased=True, seed=7)
    rng = np.random.default_rng(5)
    xb = c.up(normal(rng, 70, c.d))
    routed = c.layer.forward(xb).to_numpy()
    plain = P.MoELayer(c.d, c.H, 8, 2, ctx=ctx())
    f = io.BytesIO()
    c.layer.saveModel(f)
    assert len(f.getvalue()) == 4 * (8 * c.d + 8 + 8 * 3 * c.H * c.d)     # the bias for balance lies behind the gate
    other = P.MoELayer(c.d, c.H, 8, 2, ctx=ctx())
    other.set_routing(c.config, True)
    f.seek(0)
    other.loadModel(f)
    assert np.array_equal(other.balance_bias(), c.bias) and np.array_equal(other.forward(xb).to_numpy(), routed)
    c.layer.set_routing(None)
    with pytest.raises(RuntimeError, match="Error code 1"):
        c.layer.back(xb)                                                  # the last forward pass was another routing's
    plain.set_gate(c.Wg)
    for e in range(8):
        plain.set_expert(e, c.W1[e], c.W3[e], c.W2[e])
    assert np.array_equal(c.layer.forward(xb).to_numpy(), plain.forward(xb).to_numpy())
    with pytest.raises(RuntimeError, match="Error code 1"):
        c.layer.balance(0.1)
    with pytest.raises(RuntimeError, match="Error code 1"):
        c.layer.balance_bias()
    c.layer.set_routing(c.config, True)
    assert not c.layer.balance_bias().any()                               # a new bias is zeros
    for bad in (P.route_config(9, 2), P.route_config(8, 3), P.route_config(8, 2, nGroups=3), P.route_config(8, 2, scale=0.0), P.route_config(8, 2, scale=np.inf)):
        with pytest.raises(RuntimeError, match="Error code 1"):
            c.layer.set_routing(bad)
    for layer in (c.layer, plain, other):
        layer.close()
    xb.free()
