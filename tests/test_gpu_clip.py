"""Clipping by the global norm of many tensors against 64 bits: in place and into other buffers, both types, tensors of every
alignment and length, a MoE layer's gradients among them, norms that overflow fp32 squares."""
import ctypes as C

import numpy as np
import pytest

from tests.lm_util import L, P, U32, Buf, ctx, normal, unit, within

pytestmark = pytest.mark.gpu


def make(rng, sizes, std=1.0):
    out = []
    for i, n in enumerate(sizes):
        dtype = "bf16" if i % 3 == 1 else "f32"
        out.append((normal(rng, n, std=std * (1 + i % 5), dtype=dtype), dtype, i % 4))
    return out


@pytest.mark.parametrize("sizes", [[1], [5, 0, 3], [16384], [16385, 7, 40000, 1, 100001], [3] * 97, list(range(1, 260)), [200003] * 5])
@pytest.mark.parametrize("place", ["in", "out", "crooked"])
def test_tensors(sizes, place):
    rng = np.random.default_rng(len(sizes))
    data = make(rng, sizes)
    norm = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a, _, _ in data))
    for limit in (0.5 * norm, 2.0 * norm, 0.0, np.inf):
        src = [Buf((len(a),), dt, a, sh) for a, dt, sh in data]
        dst = src if place == "in" else [Buf((len(a),), dt, None, sh + (place == "crooked")) for a, dt, sh in data]
        clip = P.GradClip(ctx(), [b.buf for b in src], out=None if place == "in" else [b.buf for b in dst])
        got = clip.clip(limit).to_numpy()
        coef = 1.0 if np.isinf(limit) else min(1.0, float(np.float32(limit)) / (norm + 1e-6))
        assert abs(got[0] - norm) <= 2 * U32 * norm and abs(got[1] - coef) <= 2 * U32 * coef
        for (a, dt, _), s, d in zip(data, src, dst):
            # the coefficient's rounding, the product's and the result's
            within(d.get(), a.astype(np.float64) * coef, (3 * U32 + unit(dt)) * np.abs(a) * coef, (limit, len(a), dt))
            if place != "in":
                assert np.array_equal(s.get(), a)
        clip.close()
        for b in src + (dst if place != "in" else []):
            b.free()


def test_extremes():
    """Squares beyond fp32, values that only count together, infinities and no numbers, no tensors at all."""
    big, small = np.full(1000, 3e37, np.float32), np.full(50000, 1e-22, np.float32)
    b = Buf((1000,), "f32", big), Buf((50000,), "f32", small)
    clip = P.GradClip(ctx(), [b[0].buf])
    got = clip.clip(1.0).to_numpy()
    norm = np.float64(np.float32(3e37)) * np.sqrt(1000.0)
    # 9.5e38 is beyond fp32 (3.4e38): as a float it is infinite; the coefficient 1.05e-39, formed from the double, is a denormal of
    # fp32, whose half step 2^-150 is 7e-7 of it
    assert got[0] == np.inf and abs(got[1] - 1.0 / norm) <= 2.0 ** -150
    within(b[0].get(), big / norm, 8e-7 * big / norm)
    clip.close()
    few = Buf((100,), "f32", big[:100])                   # the same with a norm of 3e38
    clip = P.GradClip(ctx(), [few.buf])
    got = clip.clip(1.0).to_numpy()
    assert abs(got[0] - np.float64(big[0]) * 10) <= 4 * U32 * 3e38
    clip.close()
    few.free()
    clip = P.GradClip(ctx(), [b[1].buf])
    got = clip.clip(1.0).to_numpy()                       # squares of 1e-44: a denormal in fp32, none in double
    want = float(np.float32(1e-22)) * np.sqrt(50000.0)
    assert abs(got[0] - want) <= 4 * U32 * want and got[1] == 1.0 and np.array_equal(b[1].get(), small)
    clip.close()
    for bad, coef in ((np.inf, 0.0), (np.nan, np.nan)):
        a = np.ones(100, np.float32)
        a[7] = bad
        t = Buf((100,), "f32", a)
        clip = P.GradClip(ctx(), [t.buf])
        got = clip.clip(1.0).to_numpy()
        assert np.array_equal(got, np.array([abs(bad), coef], np.float32), equal_nan=True)
        assert np.array_equal(t.get(), a * np.float32(coef), equal_nan=True)
        clip.close()
        t.free()
    clip = P.GradClip(ctx(), [])
    assert np.array_equal(clip.clip(1.0).to_numpy(), [0.0, 1.0])
    clip.close()
    for x in b:
        x.free()


@pytest.mark.parametrize("accumulated", [False, True])
def test_with_the_gradients_of_layers(accumulated):
    """A network's norm over its MoE layers and other tensors, against the layers' own sums and scaling."""
    from tests import gpu_util as G
    from tests.synth import C as cfgs, make_inputs, scaled
    cfg = scaled(cfgs.CONFIGS["c1_tiny_f32"], T=64)
    rng = np.random.default_rng(2)
    layers, grads = [], []
    for seed in (1, 2):
        layer = G.build_layer(cfg, make_inputs(cfg, seed))
        layer.ctx.sync()
        x = P.DeviceBuffer.from_numpy(G.ctx(), make_inputs(cfg, seed)["x"], cfg.dtype)
        dout = P.DeviceBuffer.from_numpy(G.ctx(), normal(rng, cfg.T, cfg.d), cfg.dtype)
        layer.forward(x)
        layer.back(dout)
        if accumulated:
            layer.accGrad(1.0)
        layers.append(layer)
        grads.append([layer.grad(w, g) for w, g, _ in layer._param_list()])
    other = normal(rng, 5000)
    t = P.DeviceBuffer.from_numpy(G.ctx(), other, "f32")
    norm = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for gs in grads for g in gs) + (other.astype(np.float64) ** 2).sum())
    clip = P.GradClip(G.ctx(), [t], layers=layers)
    got = clip.clip(0.25 * norm).to_numpy()
    coef = float(np.float32(0.25 * norm)) / (norm + 1e-6)
    assert abs(got[0] - norm) <= 4 * U32 * norm and abs(got[1] - coef) <= 2 * U32 * coef
    within(t.to_numpy(), other * coef, 4 * U32 * np.abs(other) * coef)
    for layer, gs in zip(layers, grads):
        if accumulated:
            # the accumulators hold the scaled gradients, the gradients themselves are what they were
            assert abs(layer.gradSumSq() - sum((g.astype(np.float64) ** 2).sum() for g in gs) * coef ** 2) <= 1e-5 * layer.gradSumSq()
            for (w, g, _), a in zip(layer._param_list(), gs):
                assert np.array_equal(layer.grad(w, g), a)
        else:
            for (w, g, _), a in zip(layer._param_list(), gs):
                within(layer.grad(w, g), a * coef, 4 * U32 * np.abs(a) * coef)
        layer.close()
    with pytest.raises(RuntimeError, match="layer"):
        clip.clip(1.0)                                    # a closed layer
    clip.close()
    t.free()


def test_refusals():
    a, b = Buf((100,), "f32", np.ones(100)), Buf((100,), "f32", np.ones(100))
    lib, h = ctx().lib, ctx().handle
    T = L.GradTensorStruct

    def call(*tensors, limit=1.0, norm=None):
        return lib.omega_hip_clip_grad_norm(h, (T * max(len(tensors), 1))(*tensors), len(tensors), None, 0, limit, norm)

    pa, pb = a.ptr.value, b.ptr.value
    assert call(T(pa, pa, 100, 0, 0), T(pb, pb, 100, 0, 0)) == 0
    assert call(T(pa, pa, 100, 0, 0), T(pa, pa, 100, 0, 0)) == 1          # the same tensor twice
    assert call(T(pa, pa, 100, 0, 0), T(pa + 396, pa + 396, 1, 0, 0)) == 1
    assert call(T(pa, pb, 100, 0, 0), T(pa, pb, 100, 0, 0)) == 1          # one destination for two
    assert call(T(pa, pa + 4, 50, 0, 0)) == 1                             # a destination that overlaps its source
    assert call(T(pa, pb, 100, 0, 0), T(pb, pb, 100, 0, 0)) == 1
    assert call(T(pa, pa, 100, 7, 0)) == 1 and call(T(pa, pa, 100, 0, 5)) == 1 and call(T(None, pa, 100, 0, 0)) == 1
    assert call(T(pa + 1, pa + 1, 10, 0, 0)) == 1 and call(T(pa, pa, 100, 0, 0), limit=-1.0) == 1 and call(T(pa, pa, 100, 0, 0), limit=float("nan")) == 1
    assert call(T(pa, pa, 100, 0, 0), norm=C.c_void_p(pa + 8)) == 1
    assert np.allclose(a.get(), 0.07071, atol=1e-4)                       # only the first call ran: 1 / sqrt(200)
    a.free()
    b.free()
