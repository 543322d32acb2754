"""Refusals of the Python layers around the MoE layer, without a GPU: the C ABI compiled for the host against stand-ins, whose log says
what would have been launched."""
import ctypes as C

import numpy as np
import pytest

from tests.conftest import load_pkg
from tests.test_ops_host_logic import lib  # noqa: F401  (the host's build of the C ABI)

P, L = load_pkg(), load_pkg("_lib")


@pytest.fixture
def ctx(lib, monkeypatch):  # noqa: F811
    lib.host_live_bytes.restype = C.c_size_t
    monkeypatch.setattr(L, "_lib", lib)
    c = P.Context(0)
    lib.host_take_ops()
    yield c
    c.close()


def buf(ctx, *shape, dtype="f32"):
    return P.DeviceBuffer.from_numpy(ctx, np.zeros(shape, np.float32), dtype)


def refused(ctx, call, match):
    ctx.lib.host_take_ops()
    with pytest.raises(RuntimeError, match="Error code 1:.*" + match):
        call()
    assert ctx.lib.host_take_ops() == b""                       # nothing was launched


T, V, D = 6, 20, 8


def test_parameters_that_are_set_later(ctx):
    """A table, gamma or beta set behind the constructor is read with the layer's sizes: another shape or type would be read beyond its end."""
    ids, y, x = buf(ctx, T, dtype="i32"), buf(ctx, T, dtype="i32"), buf(ctx, T, D)
    small, half, freed = buf(ctx, V - 1, D), buf(ctx, V, D, dtype="bf16"), buf(ctx, V, D)
    freed.free()
    good, one, short = buf(ctx, V, D), buf(ctx, D), buf(ctx, D - 1)
    gone = buf(ctx, D)
    gone.free()
    emb, head, ln = P.EmbeddingLayer(V, D, ctx=ctx), P.HeadLossLayer(V, D, ctx=ctx), P.LNLayer(D, ctx=ctx)
    for call, layer in ((lambda: emb.forward(ids), emb), (lambda: head.forward(x, y), head)):
        refused(ctx, call, "no weight")
        for w in (small, half, freed, x):
            refused(ctx, lambda: setattr(layer, "weight", w), "weight")
            refused(ctx, call, "no weight")                     # (it has none still)
        layer.weight = good
        refused(ctx, lambda: setattr(layer, "weight", small), "weight")
        call()
        assert layer.weight is good and ctx.lib.host_take_ops().count(b"\n") == 1
        layer.weight = None
        refused(ctx, call, "no weight")
    refused(ctx, lambda: ln.forward(x), "no gamma")
    for name in ("gamma", "beta"):
        for b in (short, gone, good):
            refused(ctx, lambda: setattr(ln, name, b), name)
        setattr(ln, name, one)
    ln.forward(x)
    ln.back(x)
    # freed behind the layer's back: the call itself refuses
    emb.weight = head.weight = good
    head.forward(x, y)
    good.free()
    one.free()
    for call in (lambda: emb.forward(ids), head.back, lambda: head.forward(x, y), lambda: ln.back(x), lambda: ln.forward(x)):
        refused(ctx, call, "NULL")
    for w in (small, half, freed):
        refused(ctx, lambda: P.EmbeddingLayer(V, D, ctx=ctx, weight=w), "weight")
        refused(ctx, lambda: P.HeadLossLayer(V, D, ctx=ctx, weight=w), "weight")
    refused(ctx, lambda: P.LNLayer(D, ctx=ctx, gamma=gone), "gamma")
    for b in (ids, y, x, small, half, short):
        b.free()
    for layer in (emb, head, ln):
        layer.close()


def test_a_freed_factor_of_the_loss(ctx):
    """No address stands for a factor of 1: a buffer that has been freed has none either."""
    x, y, w, factor = buf(ctx, T, D), buf(ctx, T, dtype="i32"), buf(ctx, V, D), buf(ctx, 1)
    head = P.HeadLossLayer(V, D, ctx=ctx, weight=w)
    head.forward(x, y)
    head.back(factor)
    head.back()
    factor.free()
    refused(ctx, lambda: head.back(factor), "dloss")
    head.close()
    for b in (x, y, w):
        b.free()


def test_a_closed_clip(ctx):
    """It has no norm to return: nothing is scaled either."""
    g = buf(ctx, 100)
    clip = P.GradClip(ctx, [g])
    clip.clip(1.0)
    clip.close()
    refused(ctx, lambda: clip.clip(1.0), "closed")
    g.free()
