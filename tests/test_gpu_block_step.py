"""A block's training step with the operators together: norm with the residual's addition that keeps its sum in 8 bits, the routed experts, the
next norm, and all the way back; each link against its formula on what the link before gave, in 64 bits."""
import importlib
import threading

import numpy as np
import pytest

from oracle import oracle_np as N
from tests import block_util as B
from tests import test_gpu_rmsnorm as TR
from tests.lm_util import normal, rounded, within, unit, U32

pytestmark = pytest.mark.gpu
P = importlib.import_module("omega-ai_amd")

D, H, E, K = 256, 256, 16, 4


class Block:
    def __init__(self, ctx, dtype, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.dtype = ctx, dtype
        self.gammas = [normal(rng, D, std=0.1) + np.float32(1) for _ in range(2)]
        self.bufs = [P.DeviceBuffer.from_numpy(ctx, g, "f32") for g in self.gammas]
        self.norm1 = P.RMSLayer(D, ctx=ctx, dtype=dtype, gamma=self.bufs[0], keep8=True)
        self.norm2 = P.RMSLayer(D, ctx=ctx, dtype=dtype, gamma=self.bufs[1])
        self.eight = P.RMSLayer(D, ctx=ctx, dtype=dtype, gamma=self.bufs[1], out8=True)
        self.moe = P.MoELayer(D, H, E, K, ctx=ctx, dtype=dtype)
        self.moe.set_gate(normal(rng, E, D, std=1.5 * D ** -0.5, dtype=dtype))
        for e in range(E):
            self.moe.set_expert(e, normal(rng, H, D, std=D ** -0.5, dtype=dtype), normal(rng, H, D, std=D ** -0.5, dtype=dtype), normal(rng, D, H, std=H ** -0.5, dtype=dtype))
        self.moe.set_routing(P.route_config(E, K, score="sigmoid", scale=2.5, nGroups=4, topGroups=2), bias=True)
        self.moe.set_training(True)

    def step(self, x, res, dout):
        """Host copies of everything that passes between the links."""
        n = lambda b: b.to_numpy()  # noqa: E731
        got = {}
        h = self.norm1.forward(x, res)
        got["h"], got["sum1"] = n(h), n(self.norm1.sum)
        m = self.moe.forward(h)
        got["m"], got["ids"] = n(m), self.moe.routing()["ids"]
        y = self.norm2.forward(m, self.norm1.sum)
        got["y"], got["sum2"] = n(y), n(self.norm2.sum)
        e = self.eight.forward(m, self.norm1.sum)
        got["y8"] = n(self.eight.read8(e))
        d2 = self.norm2.back(dout)
        got["d2"], got["dgamma2"] = n(d2), n(self.norm2.diffGamma)
        dm = self.moe.back(d2)
        got["dm"] = n(dm)
        dx = self.norm1.back(dm, d2)
        got["dx"], got["dgamma1"] = n(dx), n(self.norm1.diffGamma)
        self.moe.balance(0.01)
        self.moe.update(1e-3)
        got["bias"] = self.moe.balance_bias()
        return got

    def close(self):
        for o in (self.norm1, self.norm2, self.eight, self.moe):
            o.close()
        for b in self.bufs:
            b.free()


def inputs(ctx, rng, T, dtype):
    arrays = [normal(rng, T, D, dtype=dtype) for _ in range(3)]
    return arrays, [P.DeviceBuffer.from_numpy(ctx, a, dtype) for a in arrays]


@pytest.fixture(scope="module")
def shared():
    c = P.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T", [1, 40, 300])
def test_each_link(shared, T, dtype):
    block = Block(shared, dtype)
    (x, res, dout), bufs = inputs(shared, np.random.default_rng(T), T, dtype)
    got = block.step(*bufs)
    first = TR.reference(x, res, block.gammas[0], got["dm"], got["d2"], dtype, True)
    second = TR.reference(got["m"], got["sum1"], block.gammas[1], dout, None, dtype, False)
    for ref, names in ((first, dict(out="h", sum="sum1", dx="dx", dgamma="dgamma1")), (second, dict(out="y", sum="sum2", dx="d2", dgamma="dgamma2"))):
        for k, name in names.items():
            want, tol = ref[k]
            within(got[name], want, tol + (unit(dtype) * (1 + 1e-3) if k in ("out", "dx") else U32 if k == "dgamma" else 0) * np.abs(want), name)
    assert np.array_equal(got["y8"], rounded(B.mx_values(*B.mx_codes(second["y"])), "bf16"))
    assert (got["ids"] >= 0).all() and np.isfinite(got["dm"]).all() and np.abs(got["bias"]).max() <= np.float32(0.01)
    for b in bufs:
        b.free()
    block.close()


def test_batches_of_changing_size_give_the_same_bits(shared):
    """Steps of a small, a large and a small batch again: buffers are made anew, and the first batch's results come back."""
    rng = np.random.default_rng(5)
    sets = [inputs(shared, rng, T, "bf16") for T in (30, 700, 30, 1)]
    alone = []
    for _, bufs in sets:
        block = Block(shared, "bf16")
        alone.append(block.step(*bufs))
        block.close()
    block = Block(shared, "bf16")
    block.moe.update = lambda rate: None
    block.moe.balance = lambda rate: None
    for (_, bufs), want in zip(sets, alone):
        got = block.step(*bufs)
        assert all(np.array_equal(got[k], want[k]) for k in want if k != "bias")
    block.close()


def test_contexts_in_threads():
    """Two contexts at once give what each gives alone."""
    out, errors = {}, []

    def work(name, seed, T):
        try:
            c = P.Context(0)
            block = Block(c, "bf16", seed)
            _, bufs = inputs(c, np.random.default_rng(seed), T, "bf16")
            out[name] = [block.step(*bufs) for _ in range(3)]
            block.close()
            for b in bufs:
                b.free()
            c.close()
        except Exception as e:   # (a thread's own)
            errors.append(e)

    for name, seed, T in (("a", 1, 200), ("b", 2, 90)):
        work(name + " alone", seed, T)
    threads = [threading.Thread(target=work, args=a) for a in (("a", 1, 200), ("b", 2, 90))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for name in ("a", "b"):
        for got, want in zip(out[name], out[name + " alone"]):
            assert all(np.array_equal(got[k], want[k]) for k in want)


def test_layers_refuse(shared):
    dtype = "f32"
    block = Block(shared, dtype)
    (x, res, dout), (xb, rb, db) = inputs(shared, np.random.default_rng(3), 5, dtype)
    narrow = P.DeviceBuffer.from_numpy(shared, np.zeros((5, D - 1), np.float32), dtype)
    short = P.DeviceBuffer.from_numpy(shared, np.zeros((4, D), np.float32), dtype)
    half = P.DeviceBuffer.from_numpy(shared, np.zeros((5, D), np.float32), "bf16")
    gone = P.DeviceBuffer.from_numpy(shared, np.zeros((5, D), np.float32), dtype)
    gone.free()
    fresh = P.RMSLayer(D, ctx=shared, dtype=dtype, gamma=block.bufs[0])
    route = P.RoutingLayer(D, 2, ctx=shared)
    keep = P.Keep8Layer(D, ctx=shared, dtype=dtype)
    block.norm2.forward(xb, rb)
    route.forward(xb)
    keep.save(xb)
    calls = [lambda: fresh.back(db), lambda: fresh.forward(narrow), lambda: fresh.forward(half), lambda: fresh.forward(xb, short), lambda: fresh.forward(xb, gone),
             lambda: fresh.forward(gone), lambda: block.norm2.back(short), lambda: block.norm2.back(db, half), lambda: block.norm2.back(db, gone), lambda: block.norm2.back(gone),
             lambda: P.RMSLayer(D, ctx=shared).forward(xb), lambda: P.RMSLayer(D, ctx=shared, gamma=xb), lambda: P.RMSLayer(D, eps=-1.0, ctx=shared, gamma=block.bufs[0]).forward(xb),
             lambda: keep.save(half), lambda: keep.save(narrow), lambda: P.Keep8Layer(D, ctx=shared).load(), lambda: P.Keep8Layer(D, form="e5m2", ctx=shared),
             lambda: route.forward(half), lambda: route.forward(narrow), lambda: route.back(xb), lambda: route.balance(0.1), lambda: P.RoutingLayer(D, 2, ctx=shared).back(xb),
             lambda: P.RoutingLayer(D, 2, ctx=shared, bias=xb), lambda: P.RoutingLayer(D, 65, ctx=shared).forward(xb), lambda: P.RoutingLayer(D, 2, score="tanh", ctx=shared),
             lambda: P.RoutingLayer(D, 4, nGroups=128, topGroups=1, ctx=shared).forward(xb)]
    for k, call in enumerate(calls):
        with pytest.raises(RuntimeError, match="Error code 1:"):
            call()
            print("call", k, "was not refused")
    assert keep.load().to_numpy().shape == (5, D)
    for o in (block, fresh, route, keep):
        o.close()
    with pytest.raises(RuntimeError):
        keep.load()
