"""The operators around the experts at numbers of rows that take several launches, and in tensors whose elements are counted in more than 32 bits.
Large tensors are read and written where it tells."""
import ctypes as C
import importlib

import numpy as np
import pytest

from tests.lm_util import DT, P, U32, unit, within
from tests.test_gpu_lm_large import Big, ctx, some_rows  # noqa: F401

L = importlib.import_module("omega-ai_amd._lib")
pytestmark = pytest.mark.gpu


def free(*bufs):
    for b in bufs:
        b.buf.free()


def test_norm_of_more_than_32_bits(ctx):  # noqa: F811
    d, dtype = 1001, "bf16"
    T = (1 << 32) // d + 3000
    rng = np.random.default_rng(0)
    gamma = (1 + 0.1 * rng.standard_normal(d)).astype(np.float32)
    gb = P.DeviceBuffer.from_numpy(ctx, gamma, "f32")
    x, out, codes = Big(ctx, T, d, dtype, 1.0), Big(ctx, T, d, dtype), Big(ctx, T, d, "u8")
    scales, rstd = Big(ctx, T, 8, "f32"), Big(ctx, T, 1, "f32")
    ctx.check(ctx.lib.omega_hip_rmsnorm_forward(ctx.handle, x.buf.ptr, None, DT[dtype], T, d, gb.ptr, 1e-6, None, out.buf.ptr, None, None, codes.buf.ptr, scales.buf.ptr,
                                                rstd.buf.ptr))
    at = some_rows(T, d)
    for t in at:
        v = x.get(t)[0].astype(np.float64)
        q = 1 / np.sqrt((v * v).mean() + np.float64(np.float32(1e-6)))
        want = v * q * gamma
        within(out.get(t)[0], want, (unit(dtype) + 4 * U32) * np.abs(want), t)
        within(rstd.get(t)[0], [q], 2 * U32 * q, t)
        s = np.repeat(scales.get(t)[0].astype(np.float64), 128)[:d]
        back = codes.get(t)[0].astype(np.int8) * s
        assert (np.abs(back - v) <= 0.5 * s).all(), t    # (the nearest whole number of scales)
    # back: a gradient in those rows and their neighbours alone
    dout, dx = Big(ctx, T, d, dtype, 0.0), out
    for t in at:
        dout.put(t, rng.standard_normal((1, d)).astype(np.float32))
    dg = P.DeviceBuffer(ctx, (d,), "f32")
    ctx.check(ctx.lib.omega_hip_rmsnorm_backward(ctx.handle, x.buf.ptr, None, None, dout.buf.ptr, None, DT[dtype], T, d, gb.ptr, rstd.buf.ptr, dx.buf.ptr, dg.ptr))
    want_g, mag = np.zeros(d), np.zeros(d)
    for t in at:
        v, dy, q = x.get(t)[0].astype(np.float64), dout.get(t)[0].astype(np.float64), float(rstd.get(t)[0, 0])
        g, xh = dy * gamma, v * q
        m = (g * xh).mean()
        # (the mean of 1001 products: eight in a lane, then a tree of 64, four roundings each)
        within(dx.get(t)[0], q * (g - xh * m), (unit(dtype) + 4 * U32) * np.abs(q * (g - xh * m)) + q * (6 * U32 * (np.abs(g) + np.abs(xh * m)) + 24 * U32 * np.abs(xh) * np.abs(g * xh).mean()), t)
        want_g, mag = want_g + dy * xh, mag + np.abs(dy * xh)
    within(dg.to_numpy(), want_g, (len(at) + 2) * U32 * mag)
    free(x, out, codes, scales, rstd, dout)
    gb.free()
    dg.free()


def test_rows_in_8_bits_of_several_launches(ctx):  # noqa: F811
    d, dtype = 9, "bf16"
    T = (1 << 29) + 5
    x, codes, scales, out = Big(ctx, T, d, dtype, 1.0), Big(ctx, T, d, "u8"), Big(ctx, T, 1, "f32"), Big(ctx, T, d, dtype)
    ctx.check(ctx.lib.omega_hip_keep8_save(ctx.handle, x.buf.ptr, DT[dtype], T, d, L.KEEP8_INT8, codes.buf.ptr, scales.buf.ptr))
    ctx.check(ctx.lib.omega_hip_keep8_load(ctx.handle, codes.buf.ptr, scales.buf.ptr, L.KEEP8_INT8, T, d, out.buf.ptr, DT[dtype]))
    launches = {(k << 26) + n for k in range(1, 9) for n in (-2, -1, 0, 1)}    # where one of the launches ends and another begins
    for t in sorted(launches | set(some_rows(T, d))):
        v = x.get(t)[0].astype(np.float64)
        s = float(scales.get(t)[0, 0])
        within([s], [np.abs(v).max() / 127], 2 * U32 * s, t)
        kept = codes.get(t)[0].astype(np.int8) * s
        assert (np.abs(kept - v) <= 0.5 * s).all(), t
        within(out.get(t)[0], kept, (unit(dtype) + U32) * np.abs(kept), t)
    free(x, codes, scales, out)


def route(ctx, cfg, z, T, ids, w, counts=None):  # noqa: F811
    ctx.check(ctx.lib.omega_hip_route_forward(ctx.handle, C.byref(cfg), z.buf.ptr, T, None, ids.buf.ptr, w.buf.ptr, counts.ptr if counts else None))


def test_routing_of_more_than_32_bits(ctx):  # noqa: F811
    T, E, K = (1 << 23) + 5, 512, 2
    z, ids, w, dw, dz = Big(ctx, T, E, "f32", 1.0), Big(ctx, T, K, "i32"), Big(ctx, T, K, "f32"), Big(ctx, T, K, "f32", 1.0), Big(ctx, T, E, "f32")
    counts, cfg = P.DeviceBuffer(ctx, (E,), "i32"), P.route_config(E, K)
    route(ctx, cfg, z, T, ids, w, counts)
    ctx.check(ctx.lib.omega_hip_route_backward(ctx.handle, C.byref(cfg), z.buf.ptr, T, ids.buf.ptr, w.buf.ptr, dw.buf.ptr, dz.buf.ptr))
    assert counts.to_numpy().astype(np.int64).sum() == T * K
    for t in some_rows(T, E):
        v = z.get(t)[0].astype(np.float64)
        order = np.argsort(-v, kind="stable")[:K]
        assert np.array_equal(ids.get(t)[0], order), t
        e = np.exp(v[order] - v[order[0]])
        p = e / e.sum()
        within(w.get(t)[0], p, 12 * U32 * p, t)
        g, want, mag = dw.get(t)[0].astype(np.float64), np.zeros(E), np.zeros(E)
        want[order] = p * (g - (p * g).sum())
        mag[order] = p * (np.abs(g) + (p * np.abs(g)).sum())
        within(dz.get(t)[0], want, 40 * U32 * mag, t)
    free(z, ids, w, dw, dz)
    counts.free()


def test_gradient_of_the_logits_of_several_launches(ctx):  # noqa: F811
    T, E, K = (1 << 26) + 77, 2, 1
    z, ids, w, dw, dz = Big(ctx, T, E, "f32", 1.0), Big(ctx, T, K, "i32"), Big(ctx, T, K, "f32"), Big(ctx, T, K, "f32", 1.0), Big(ctx, T, E, "f32")
    cfg = P.route_config(E, K, score="sigmoid", renorm=False)
    route(ctx, cfg, z, T, ids, w)
    ctx.check(ctx.lib.omega_hip_route_backward(ctx.handle, C.byref(cfg), z.buf.ptr, T, ids.buf.ptr, w.buf.ptr, dw.buf.ptr, dz.buf.ptr))
    for at in (0, (1 << 26) - 8, T - 8):
        v, g = z.get(at, 8).astype(np.float64), dw.get(at, 8)[:, 0].astype(np.float64)
        best, row = v.argmax(1), np.arange(8)
        s = 1 / (1 + np.exp(-v[row, best]))
        assert np.array_equal(ids.get(at, 8)[:, 0], best)
        within(w.get(at, 8)[:, 0], s, 12 * U32 * s)
        want = np.zeros((8, E))
        want[row, best] = s * g / (1 + np.exp(v[row, best]))
        within(dz.get(at, 8), want, 24 * U32 * np.abs(want))
    free(z, ids, w, dw, dz)
