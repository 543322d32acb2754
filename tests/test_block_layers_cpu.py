"""Refusals of the Python layers around the experts, without a GPU: the C ABI compiled for the host against stand-ins, whose log says what would
have been launched."""
import numpy as np
import pytest

from tests.conftest import load_pkg
from tests.test_block_host_logic import lib  # noqa: F401  (the host's build of the C ABI)

P, L = load_pkg(), load_pkg("_lib")
T, D, E, K = 6, 200, 16, 4


@pytest.fixture
def ctx(lib, monkeypatch):  # noqa: F811
    monkeypatch.setattr(L, "_lib", lib)
    c = P.Context(0)
    lib.host_take_block()
    yield c
    c.close()
    assert lib.host_live_bytes() == 0


def buf(ctx, *shape, dtype="f32"):
    return P.DeviceBuffer.from_numpy(ctx, np.zeros(shape, np.float32), dtype)


def gone(ctx, *shape, dtype="f32"):
    b = buf(ctx, *shape, dtype=dtype)
    b.free()
    return b


def refused(ctx, call, match):
    ctx.lib.host_take_block()
    with pytest.raises(RuntimeError, match="Error code 1:.*" + match):
        call()
    assert ctx.lib.host_take_block() == b""                              # nothing was launched


def launched(ctx, call, what):
    ctx.lib.host_take_block()
    r = call()
    assert ctx.lib.host_take_block() == what
    return r


def free(*bufs):
    for b in bufs:
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rms_layer(ctx, dtype):
    other = "bf16" if dtype == "f32" else "f32"
    x, r, dy, g = buf(ctx, T, D, dtype=dtype), buf(ctx, T, D, dtype=dtype), buf(ctx, T, D, dtype=dtype), buf(ctx, D)
    wrong = [buf(ctx, T, D, dtype=other), buf(ctx, T, D - 1, dtype=dtype), buf(ctx, T + 1, D, dtype=dtype), buf(ctx, D, dtype=dtype)]
    freed = gone(ctx, T, D, dtype=dtype)
    layer = P.RMSLayer(D, ctx=ctx, dtype=dtype)
    refused(ctx, lambda: layer.forward(x), "no gamma")
    for bad in (wrong[3] if dtype == "bf16" else buf_of(wrong, ctx), gone(ctx, D)):
        refused(ctx, lambda: setattr(layer, "gamma", bad), "gamma")
    refused(ctx, lambda: layer.back(dy), "without a forward")
    layer.gamma = g
    for bad in (wrong[0], wrong[1], wrong[3]):
        refused(ctx, lambda: layer.forward(bad), "input")
    for bad in (wrong[0], wrong[1], wrong[2], freed):
        refused(ctx, lambda: layer.forward(x, bad), "residual")
    refused(ctx, lambda: layer.forward(freed), "NULL")
    refused(ctx, lambda: layer.back(dy), "without a forward")            # a refused forward leaves none behind
    out = launched(ctx, lambda: layer.forward(x, r), b"rms\n")
    assert out.shape == (T, D) and out.dtype == dtype and layer.sum.shape == (T, D) and layer.input is layer.sum
    for bad in wrong:
        refused(ctx, lambda: layer.back(bad), "delta")
        refused(ctx, lambda: layer.back(dy, bad), "dsum")
    refused(ctx, lambda: layer.back(dy, freed), "dsum")
    launched(ctx, lambda: layer.back(dy, dy), b"rms_back ws\n")
    layer.gamma = None
    refused(ctx, lambda: layer.back(dy), "no gamma")
    layer.gamma = g
    layer.sum.free()
    refused(ctx, lambda: layer.forward(x, r), "sum")                     # (no address would mean none)
    layer.forward(x)
    assert layer.sum is None and layer.input is x
    free(g)
    refused(ctx, lambda: layer.forward(x), "NULL")
    layer.close()
    refused(ctx, lambda: layer.back(dy), "without a forward")
    free(x, r, dy, *wrong)


def buf_of(wrong, ctx):
    b = buf(ctx, D - 1)
    wrong.append(b)
    return b


def test_rms_layer_in_8_bits(ctx):
    x, g, dy = buf(ctx, T, D, dtype="bf16"), buf(ctx, D), buf(ctx, T, D, dtype="bf16")
    layer = P.RMSLayer(D, ctx=ctx, dtype="bf16", gamma=g, out8=True, keep8=True)
    rows = launched(ctx, lambda: layer.forward(x), b"rms\n")
    assert rows.form == "mx" and rows.codes.shape == (T, D) and rows.scales.shape == (T, 7) and layer.kept.scales.shape == (T, 2)
    assert launched(ctx, lambda: layer.read8(rows), b"load\n").dtype == "bf16"
    refused(ctx, lambda: layer.read8(rows, "i32"), "dtype")
    free(x)                                                              # the backward pass needs the kept rows alone
    launched(ctx, lambda: layer.back(dy), b"rms_back ws\n")
    assert layer.forward(dy) is rows                                     # the same buffers for a batch of the same size
    more = buf(ctx, T + 1, D, dtype="bf16")
    assert layer.forward(more) is not rows
    refused(ctx, lambda: layer.read8(rows), "NULL")                      # the smaller batch's have gone
    codes, scales = buf(ctx, T, D, dtype="u8"), buf(ctx, T, 7, dtype="u8")
    launched(ctx, lambda: layer.read8(P.Rows8("mx", (T, D), codes, scales), "f32"), b"load\n")
    for form, shape, c, s in (("mx", (T + 1, D), codes, scales), ("mx", (T, D), scales, scales), ("int8", (T, D), codes, scales), ("fp4", (T, D), codes, scales),
                              ("mx", (T, D), dy, scales), ("mx", (T * D,), codes, scales)):
        refused(ctx, lambda: P.Rows8(form, shape, c, s), "")
    layer.close()
    free(g, dy, more, codes, scales)


@pytest.mark.parametrize("form", ["int8", "mx"])
def test_keep8_layer(ctx, form):
    x, wrong = buf(ctx, T, D), [buf(ctx, T, D, dtype="bf16"), buf(ctx, T, D + 1), buf(ctx, D)]
    refused(ctx, lambda: P.Keep8Layer(D, form="fp4", ctx=ctx), "form")
    layer = P.Keep8Layer(D, form=form, ctx=ctx)
    refused(ctx, layer.load, "without a save")
    launched(ctx, lambda: layer.save(x), b"save\n")
    for bad in wrong:
        refused(ctx, lambda: layer.save(bad), "input")
    launched(ctx, layer.load, b"load\n")                                 # what was refused leaves the last rows
    refused(ctx, lambda: layer.save(gone(ctx, T, D)), "NULL")
    refused(ctx, layer.load, "without a save")
    layer.close()
    refused(ctx, layer.load, "without a save")
    free(x, *wrong)


def test_routing_layer(ctx):
    z, dw, bias = buf(ctx, T, E), buf(ctx, T, K), buf(ctx, E)
    wrong = [buf(ctx, T, E + 1), buf(ctx, T, E, dtype="bf16"), buf(ctx, E)]
    refused(ctx, lambda: P.RoutingLayer(E, K, score="linear", ctx=ctx), "score")
    layer = P.RoutingLayer(E, K, ctx=ctx)
    refused(ctx, lambda: layer.back(dw), "without a forward")
    refused(ctx, lambda: layer.balance(0.1), "without")
    for bad in (wrong[0], gone(ctx, E)):
        refused(ctx, lambda: setattr(layer, "bias", bad), "bias")
    for bad in wrong:
        refused(ctx, lambda: layer.forward(bad), "logits")
    w = launched(ctx, lambda: layer.forward(z), b"route ws\n")
    assert w.shape == layer.ids.shape == (T, K) and layer.ids.dtype == "i32" and layer.counts.shape == (E,)
    refused(ctx, lambda: layer.balance(0.1), "without")
    for bad in wrong:
        refused(ctx, lambda: layer.back(bad), "delta")
    launched(ctx, lambda: layer.back(dw), b"route_back\n")
    layer.bias = bias
    launched(ctx, lambda: layer.forward(z), b"route ws\n")
    launched(ctx, lambda: layer.balance(0.1), b"balance\n")
    for rate in (-0.1, float("nan"), float("inf")):
        refused(ctx, lambda: layer.balance(rate), "rate")
    free(bias)
    refused(ctx, lambda: layer.forward(z), "freed")                      # (no address would mean no bias)
    refused(ctx, lambda: layer.balance(0.1), "NULL")
    layer.close()
    refused(ctx, lambda: layer.back(dw), "without a forward")
    for kw in (dict(nGroups=3), dict(nGroups=4, topGroups=5), dict(nGroups=4, groupBest=3), dict(nGroups=8, topGroups=1), dict(scale=0.0)):
        bad = P.RoutingLayer(E, K, ctx=ctx, **kw)
        refused(ctx, lambda: bad.forward(z), "")
        bad.close()
    free(z, dw, *wrong)
