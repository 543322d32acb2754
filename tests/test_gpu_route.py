"""Routing to experts against the definition in 64 bits: the choice has to be the same, weights and gradients within their roundings."""
import ctypes as C

import numpy as np
import pytest

from tests import block_util as B
from tests.lm_util import U32, Buf, P, ctx, within

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan
# T, E, K, groups, top, best
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 8, 2, 1, 1, 1), (5, 16, 16, 4, 4, 2), (64, 8, 2, 2, 1, 1), (33, 17, 3, 1, 1, 1), (19, 60, 6, 5, 3, 2), (17, 64, 64, 64, 64, 1),
          (7, 64, 8, 16, 5, 2), (130, 65, 7, 5, 2, 2), (40, 128, 8, 1, 1, 1), (9, 127, 64, 1, 1, 1), (50, 256, 8, 8, 4, 2), (3, 200, 6, 40, 9, 1), (21, 256, 1, 1, 1, 1),
          (11, 512, 16, 64, 8, 2), (6, 511, 5, 7, 3, 2), (2000, 32, 4, 1, 1, 1), (1500, 160, 6, 8, 3, 2)]


def forward(z, b, K, shift=0, **kw):
    T, E = z.shape
    c = ctx()
    cfg = P.route_config(E, K, score="sigmoid" if kw.get("sigmoid") else "softmax", renorm=kw.get("renorm", True), scale=kw.get("scale", 1.0), nGroups=kw.get("groups", 1),
                         topGroups=kw.get("top"), groupBest=kw.get("best", 2))
    zb, bb = Buf((T, E), "f32", z, shift), None if b is None else Buf((E,), "f32", b, shift)
    ids, w, n = Buf((T, K), "i32", shift=shift), Buf((T, K), "f32", shift=shift), Buf((E,), "i32", shift=shift)
    c.check(c.lib.omega_hip_route_forward(c.handle, C.byref(cfg), zb.ptr, T, bb.ptr if bb else None, ids.ptr, w.ptr, n.ptr))
    got = ids.get(), w.get(), n.get()
    for o in (zb, ids, w, n) + ((bb,) if bb else ()):
        o.free()
    return got


def backward(z, ids, w, dw, shift=0, **kw):
    T, E = z.shape
    c, K = ctx(), ids.shape[1]
    cfg = P.route_config(E, K, score="sigmoid" if kw.get("sigmoid") else "softmax", renorm=kw.get("renorm", True), scale=kw.get("scale", 1.0), nGroups=kw.get("groups", 1),
                         topGroups=kw.get("top"), groupBest=kw.get("best", 2))
    zb, ib, wb, db, out = Buf((T, E), "f32", z, shift), Buf((T, K), "i32", ids), Buf((T, K), "f32", w, shift), Buf((T, K), "f32", dw), Buf((T, E), "f32", shift=shift)
    c.check(c.lib.omega_hip_route_backward(c.handle, C.byref(cfg), zb.ptr, T, ib.ptr, wb.ptr, db.ptr, out.ptr))
    got = out.get()
    for o in (zb, ib, wb, db, out):
        o.free()
    return got


def check(z, b, K, dw=None, shift=0, **kw):
    ids, w, counts, s = B.route(z, b, K, **kw)
    got = forward(z, b, K, shift, **kw)
    other = np.nonzero((got[0] != ids).any(1))[0]
    if len(other) and kw.get("groups", 1) > 1:      # what 64 bits leave open (block_util.GROUPS_OPEN)
        assert all(B.choices(z, b, K, got[0][t], t, **kw) for t in other), (kw, other[:4])
        z, got = np.delete(z, other, 0), tuple(np.delete(a, other, 0) for a in got[:2]) + (B.route(np.delete(z, other, 0), b, K, **kw)[2],)
        dw = None if dw is None else np.delete(dw, other, 0)
        ids, w, counts, s = B.route(z, b, K, **kw)
        assert len(other) <= 0.05 * (len(z) + len(other)) + 1
    assert np.array_equal(got[0], ids), (kw, np.argwhere(got[0] != ids)[:4])
    assert np.array_equal(got[2], counts)
    # a weight: e^x, its rounded argument of up to 100 below the largest, the sum and the division; scores below 2^-120 are lost without renorm
    with np.errstate(invalid="ignore"):
        near = np.abs(np.where(np.isfinite(z), z, 0).max(1, keepdims=True) - np.take_along_axis(np.where(np.isfinite(z), z, 0), np.maximum(ids, 0), 1))
    size = 4 if kw.get("sigmoid") else 4 + np.minimum(near, 200)
    within(got[1], w, (size + 24) * U32 * np.abs(w) + kw.get("scale", 1.0) * 2.0 ** -120, ("w", kw))
    if dw is not None:
        args = {k: kw.get(k, d) for k, d in (("sigmoid", False), ("renorm", True))}
        dz, terms = B.route_back(z, s, got[0], got[1], dw, kw.get("scale", 1.0), **args)
        back = backward(z, got[0], got[1], dw, shift, **kw)
        # (scores again: their own roundings; sums of up to 64 terms)
        depth = 70 + (4 + np.minimum(np.abs(np.where(np.isfinite(z), z, 0) - np.where(np.isfinite(z), z, 0).max(1, keepdims=True)), 200))
        within(back, dz, depth * U32 * terms + 2.0 ** -120, ("dlogits", kw))
    return got


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("T,E,K,groups,top,best", SHAPES)
def test_against_the_definition(T, E, K, groups, top, best, sigmoid, biased):
    rng = np.random.default_rng(T * E + K)
    for renorm, scale, shut, shift in ((True, 1.0, 0.0, 0), (False, 2.5, 0.1, 1), (True, 0.5, 0.6, 2), (False, 1.0, 0.0, 3)):
        z = (rng.standard_normal((T, E)) * 1.5 + rng.standard_normal(E)).astype(np.float32)
        z[rng.random((T, E)) < shut] = -INF
        if shut:
            z[rng.random(T) < 0.2] = -INF         # tokens without an expert
        b = (rng.standard_normal(E) * (0.2 if sigmoid else 1.0 / E)).astype(np.float32) if biased else None
        dw = rng.standard_normal((T, K)).astype(np.float32)
        check(z, b, K, dw, shift, sigmoid=sigmoid, renorm=renorm, scale=scale, groups=groups, top=top, best=best)


@pytest.mark.parametrize("E", [12, 64, 96, 256, 400])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_worths_that_fp32_cannot_tell_apart(E, sigmoid):
    """Few different logits and few different biases, and logits that differ in their last places: the first of equal ones, the larger of nearly equal
    ones."""
    rng = np.random.default_rng(E)
    T, K = 200, min(8, E // 2)
    pool = rng.standard_normal(3).astype(np.float32)
    z = rng.choice(pool, (T, E))
    near = rng.random((T, E)) < 0.5
    z[near] = (z[near].view(np.int32) + rng.integers(-2, 3, near.sum(), dtype=np.int32)).view(np.float32)
    z[:3] = 0.25                                     # all equal
    for b in (None, np.zeros(E, np.float32), rng.choice(np.float32([0.0, 0.125]), E), (1e-7 * rng.standard_normal(E)).astype(np.float32)):
        for groups, top in ((1, 1), (4, 2)):
            for best in (1, 2):
                check(z, b, K, sigmoid=sigmoid, groups=groups, top=top, best=best)


def test_biases_that_cancel_scores():
    """Worths that are equal in 64 bits but for what fp32 rounds off: b = -s for half of the experts, so that all their worths are near 0."""
    rng = np.random.default_rng(8)
    T, E = 1, 256
    for _ in range(20):
        z = rng.standard_normal((T, E)).astype(np.float32)
        s = 1.0 / (1.0 + np.exp(-z[0].astype(np.float64)))
        check(z, (-s).astype(np.float32), 8, sigmoid=True)
        e = np.exp(z[0].astype(np.float64))
        check(z, (-e / e.sum()).astype(np.float32), 8)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("E,groups", [(8, 1), (60, 5), (256, 8), (512, 1)])
def test_closed_and_extreme_logits(E, groups, sigmoid):
    rng = np.random.default_rng(E)
    K = 4
    z = rng.standard_normal((12, E)).astype(np.float32)
    z[0] = -INF
    z[1] = NAN
    z[2, :-1] = -INF                                  # one open, the last
    z[3, 3], z[3, 5] = INF, NAN
    z[4, [1, 6]] = INF
    z[5] = np.finfo(np.float32).min                   # a mask of the lowest value: open, and all equal
    z[6, ::2] = np.finfo(np.float32).min
    z[7] *= 60
    z[8] = -200 + rng.standard_normal(E)
    z[9] = 90 + rng.standard_normal(E)
    z[10, 2:] = -INF
    b = (rng.standard_normal(E) * 0.1).astype(np.float32)
    odd = b.copy()
    odd[[0, 3]] = -INF
    odd[1], odd[2] = NAN, INF
    dw = rng.standard_normal((12, K)).astype(np.float32)
    for bias in (None, b, odd):
        for renorm in (True, False):
            check(z, bias, K, dw, sigmoid=sigmoid, renorm=renorm, groups=groups, top=max(1, groups // 2))


def test_gradient_against_differences():
    """Central differences of sum(w dw) in 64 bits with the choice held."""
    rng = np.random.default_rng(4)
    T, E, K, step = 3, 12, 4, 1e-5
    z, dw, b = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal(E).astype(np.float32)
    for sigmoid in (False, True):
        for renorm in (False, True):
            kw = dict(sigmoid=sigmoid, renorm=renorm, scale=1.5)
            ids, w, _ = forward(z, b, K, **kw)
            back = backward(z, ids, w, dw, **kw)

            def f(z):
                s = 1 / (1 + np.exp(-z)) if sigmoid else np.exp(z) / np.exp(z).sum(1, keepdims=True)
                v = np.take_along_axis(s, ids, 1)
                return float((v / (v.sum(1, keepdims=True) if renorm else 1.0) * 1.5 * dw).sum())

            for at in np.ndindex(T, E):
                side = []
                for h in (step, -step):
                    moved = z.astype(np.float64)
                    moved[at] += h
                    side.append(f(moved))
                assert abs((side[0] - side[1]) / (2 * step) - back[at]) < 2e-6, (sigmoid, renorm, at)   # step^2 and 1e-16 / step: 1e-10; fp32 roundings of the rest


def test_ids_that_are_none_and_no_tokens():
    c, T, E, K = ctx(), 9, 30, 3
    rng = np.random.default_rng(2)
    z, dw = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, K)).astype(np.float32)
    ids, w, _ = forward(z, None, K, renorm=False)
    odd = ids.copy()
    odd[0, 1], odd[1, 0], odd[2, 2] = -1, E, 2 ** 30          # outside: no part
    got = backward(z, odd, w, dw, renorm=False)
    w2 = np.where((odd < 0) | (odd >= E), 0, w)
    assert np.array_equal(got, backward(z, ids, w2, dw, renorm=False))
    cfg, counts = P.route_config(E, K), Buf((E,), "i32")
    c.check(c.lib.omega_hip_route_forward(c.handle, C.byref(cfg), None, 0, None, None, None, counts.ptr))
    assert not counts.get().any()
    c.check(c.lib.omega_hip_route_forward(c.handle, C.byref(cfg), None, 0, None, None, None, None))
    c.check(c.lib.omega_hip_route_backward(c.handle, C.byref(cfg), None, 0, None, None, None, None))
    counts.free()


def test_many_tokens_and_counts():
    rng = np.random.default_rng(6)
    T, E, K = 40001, 24, 3
    z = rng.standard_normal((T, E)).astype(np.float32)
    c, zb = ctx(), None
    layer = P.RoutingLayer(E, K, ctx=c, bias=P.DeviceBuffer.from_numpy(c, np.zeros(E, np.float32), "f32"))
    zb = P.DeviceBuffer.from_numpy(c, z, "f32")
    w = layer.forward(zb).to_numpy()
    order = np.argsort(-z, 1, kind="stable")[:, :K]
    assert np.array_equal(layer.ids.to_numpy(), order)
    counts = np.bincount(order.reshape(-1), minlength=E)
    assert np.array_equal(layer.counts.to_numpy(), counts)
    e = np.exp(np.take_along_axis(z, order, 1).astype(np.float64))
    within(w, e / e.sum(1, keepdims=True), 1e-6)
    layer.balance(0.01)
    assert np.array_equal(layer.bias.to_numpy(), np.float32(0.01) * np.sign(T * K - counts * E).astype(np.float32))
    layer.close()
    zb.free()


def test_balance():
    c = ctx()
    rng = np.random.default_rng(9)
    for E in (1, 7, 256, 1000):
        counts, bias = rng.integers(0, 5, E).astype(np.int32), rng.standard_normal(E).astype(np.float32)
        cb, bb = Buf((E,), "i32", counts), Buf((E,), "f32", bias)
        c.check(c.lib.omega_hip_route_balance(c.handle, cb.ptr, E, 0.25, bb.ptr))
        step = np.float32(0.25) * np.sign(counts.sum() - counts.astype(np.int64) * E).astype(np.float32)
        assert np.array_equal(bb.get(), bias + step)
        cb.free()
        bb.free()
    big = np.full(2, 2 ** 31 - 1, np.int32)            # sums past 32 bits
    big[1] -= 1
    cb, bb = Buf((2,), "i32", big), Buf((2,), "f32", np.zeros(2, np.float32))
    c.check(c.lib.omega_hip_route_balance(c.handle, cb.ptr, 2, 1.0, bb.ptr))
    assert list(bb.get()) == [-1.0, 1.0]
