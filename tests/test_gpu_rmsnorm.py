"""RMS norm with the residual's addition, forward and backward, whole and in 8 bits, against the formulas in 64 bits and against differences."""
import numpy as np
import pytest

from tests import block_util as B
from tests.lm_util import DT, U32, Buf, ctx, normal, rounded, unit, within
from tests.test_gpu_keep8 import Bytes

pytestmark = pytest.mark.gpu

EPS = np.float64(np.float32(1e-6))
SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (4, 512), (7, 513), (64, 1000), (9, 2050), (3, 4096), (2, 8192), (2, 8200), (3, 9001), (600, 96), (2500, 40),
          (2100, 768), (1100, 130), (1200, 1024), (700, 2048)]
ADDS = 60     # no fp32 sum over a row has more additions behind one another: 40 elements a lane, six steps in a wave, sixteen waves at most


def reference(x, res, gamma, dy, dsum, dtype, kept):
    """Formulas in 64 bits, with what each may be off by before it is rounded."""
    h = x if res is None else rounded(x + res, dtype)                # fp32 addition, rounded to the type
    v, gamma, dy = (np.asarray(a, np.float64) for a in (h, gamma, dy))
    q = 1.0 / np.sqrt((v * v).mean(1, keepdims=True) + EPS)
    y = v * q * gamma
    u = B.int8_values(*B.int8_codes(h)).astype(np.float64) if kept else v
    xh, g = u * q, dy * gamma
    m = (g * xh).mean(1, keepdims=True)
    dx = q * (g - xh * m)
    # q: a rounding to fp32; xh one more; a product with gamma or dy one each; the mean's additions
    em = (ADDS + 6) * U32 * np.abs(g * xh).mean(1, keepdims=True)
    edx = q * (4 * U32 * np.abs(g) + np.abs(xh) * em + 5 * U32 * np.abs(xh * m))
    if dsum is not None:
        dx = dx + dsum
        edx = edx + U32 * (np.abs(dx) + np.abs(dsum))
    n = len(x)
    return dict(sum=(h, 0.0), out=(y, 4 * U32 * np.abs(y)), rstd=(q[:, 0], U32 * q[:, 0]), dx=(dx, edx),
                dgamma=((dy * xh).sum(0), (n + 24) * U32 * np.abs(dy * xh).sum(0)), y=y)


def run(x, res, gamma, dy, dsum, dtype, shift=0, kept=False, out8=False, in_place=False):
    T, d = x.shape
    c, lib = ctx(), ctx().lib
    dt = DT[dtype]
    b = dict(x=Buf((T, d), dtype, x, shift), gamma=Buf((d,), "f32", gamma, shift), dy=Buf((T, d), dtype, dy, shift), rstd=Buf((T,), "f32"),
             out=Buf((T, d), dtype, shift=shift), dx=Buf((T, d), dtype, shift=shift), dgamma=Buf((d,), "f32", shift=shift))
    if res is not None:
        b["res"], b["sum"] = Buf((T, d), dtype, res, shift), Buf((T, d), dtype, shift=shift)
        if in_place:
            b["sum"].free()
            b["sum"] = b["res"]
    if dsum is not None:
        b["dsum"] = Buf((T, d), dtype, dsum, shift)
        if in_place:
            b["dx"].free()
            b["dx"] = b["dsum"]
    if kept:
        b["keep"], b["keep_s"] = Bytes((T, d), shift=shift), Buf((T, -(-d // 128)), "f32", shift=shift)
    if out8:
        b["out8"], b["out8_s"] = Bytes((T, d), shift=shift), Bytes((T, -(-d // 32)), shift=shift)
    p = {k: v.ptr for k, v in b.items()}
    at = p.get
    c.check(lib.omega_hip_rmsnorm_forward(c.handle, p["x"], at("res"), dt, T, d, p["gamma"], EPS, at("sum"), p["out"], at("out8"), at("out8_s"), at("keep"),
                                          at("keep_s"), p["rstd"]))
    got = {k: b[k].get() for k in ("out", "rstd", "sum", "keep", "keep_s", "out8", "out8_s") if k in b}
    h = None if kept else p["x"] if res is None else p["sum"]
    c.check(lib.omega_hip_rmsnorm_backward(c.handle, h, at("keep"), at("keep_s"), p["dy"], at("dsum"), dt, T, d, p["gamma"], p["rstd"], p["dx"], p["dgamma"]))
    got.update(dx=b["dx"].get(), dgamma=b["dgamma"].get())
    for v in {id(v): v for v in b.values()}.values():
        v.free()
    return got


def inputs(rng, T, d, dtype, residual=True):
    x = rounded(rng.standard_normal((T, d)) * np.exp(rng.standard_normal((T, 1))), dtype)
    res = normal(rng, T, d, dtype=dtype) if residual else None
    return x, res, normal(rng, d) + np.float32(1), normal(rng, T, d, dtype=dtype), normal(rng, T, d, dtype=dtype) if residual else None


def check(got, ref, dtype, what):
    for k in ("sum", "out", "rstd", "dx", "dgamma"):
        if k in got:
            want, tol = ref[k]
            if k == "sum":
                assert np.array_equal(got[k], want), what
            else:
                within(got[k], want, tol + (unit(dtype) * (1 + 1e-3) if k in ("out", "dx") else U32) * np.abs(want), (k, what))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", SHAPES)
def test_against_the_formulas(T, d, dtype):
    rng = np.random.default_rng(T + d)
    for shift, residual, kept in ((0, True, False), (1, False, False), (2, True, True), (4, False, True)):
        x, res, gamma, dy, dsum = inputs(rng, T, d, dtype, residual)
        ref = reference(x, res, gamma, dy, dsum, dtype, kept)
        got = run(x, res, gamma, dy, dsum, dtype, shift, kept)
        check(got, ref, dtype, (shift, residual, kept))
        if kept:
            codes, scales = B.int8_codes(ref["sum"][0])
            assert np.array_equal(got["keep"].view(np.int8), codes) and np.array_equal(got["keep_s"], scales)
        for k, v in run(x, res, gamma, dy, dsum, dtype, shift, kept, in_place=True).items():
            assert np.array_equal(got[k], v), (k, "the same inputs, or sums in place, give other bits")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", SHAPES)
def test_output_in_8_bits(T, d, dtype):
    """Codes and scales of y in 64 bits, bit for bit: a y in doubt is formed again in double, whose own error of some 2^-50 reaches a border with a
    probability of 2^-45 an element."""
    rng = np.random.default_rng(T * 7 + d)
    for shift, residual in ((0, True), (1, False)):
        x, res, gamma, dy, dsum = inputs(rng, T, d, dtype, residual)
        got = run(x, res, gamma, dy, dsum, dtype, shift, out8=True)
        ref = reference(x, res, gamma, dy, dsum, dtype, False)
        codes, scales = B.mx_codes(ref["y"])
        assert np.array_equal(got["out8_s"], scales) and np.array_equal(got["out8"], codes)
        check(got, ref, dtype, "out beside out8")


def test_output_in_8_bits_on_its_borders():
    """Rows whose y are borders of their codes exactly but for the root mean square's error: gamma = 1, elements multiples of a number, so that a
    fp32 q would put thousands of them on either side."""
    rng = np.random.default_rng(11)
    T, d = 200, 1024
    for _ in range(3):
        x = rng.choice((B.E4M3[8:] + B.E4M3[7:-1]) / 2, (T, d)).astype(np.float32) * np.float32(rng.random() + 0.5)
        x[:, ::32] = 449.0
        gamma = rounded(np.sqrt((x.astype(np.float64) ** 2).mean(0)), "f32")
        x[:, 1::2] *= -1
        got = run(x, None, gamma, x, None, "f32", out8=True)
        ref = reference(x, None, gamma, x, None, "f32", False)
        codes, scales = B.mx_codes(ref["y"])
        assert np.array_equal(got["out8_s"], scales) and np.array_equal(got["out8"], codes)


def test_gradients_against_differences():
    """Central differences of sum(y * dy) + sum(h * dsum) in 64 bits, for a few elements of x and of gamma."""
    rng = np.random.default_rng(3)
    T, d, step = 3, 10, 1e-6
    x, gamma, dy, dsum = normal(rng, T, d), normal(rng, d) + np.float32(1), normal(rng, T, d), normal(rng, T, d)
    got = run(x, np.zeros_like(x), gamma, dy, dsum, "f32")

    def f(x, gamma):
        y = x / np.sqrt((x * x).mean(1, keepdims=True) + EPS) * gamma
        return float((y * dy.astype(np.float64)).sum() + (x * dsum.astype(np.float64)).sum())

    args = [a.astype(np.float64) for a in (x, gamma)]
    for k, name in enumerate(("dx", "dgamma")):
        for at in list(np.ndindex(args[k].shape))[::3]:
            side = []
            for s in (step, -step):
                moved = [a.copy() for a in args]
                moved[k][at] += s
                side.append(f(*moved))
            # differences: step^2 times a third derivative (of order 10) and cancellation 1e-15 / step; the gradient itself: 1e-5 of its terms
            assert abs((side[0] - side[1]) / (2 * step) - got[name][at]) < 3e-5, (name, at)


def test_zeros_and_no_rows():
    T, d = 4, 100
    x = np.zeros((T, d), np.float32)
    got = run(x, None, np.ones(d, np.float32), np.ones((T, d), np.float32), None, "f32", out8=True)
    assert not got["out"].any() and not got["dgamma"].any() and not got["out8"].any() and not got["out8_s"].any()
    want = np.float64(1.0) / np.sqrt(EPS)
    within(got["dx"], np.full((T, d), want), 4 * U32 * want)
    c, dg = ctx(), Buf((d,), "f32")
    c.check(c.lib.omega_hip_rmsnorm_forward(c.handle, None, None, 0, 0, d, None, EPS, None, None, None, None, None, None, None))
    c.check(c.lib.omega_hip_rmsnorm_backward(c.handle, None, None, None, None, None, 0, 0, d, None, None, None, dg.ptr))
    assert not dg.get().any()
    dg.free()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("d", [96, 1500, 9001])
def test_no_numbers_stay_in_their_rows(d, kept):
    rng = np.random.default_rng(d)
    x, dy = normal(rng, 6, d), normal(rng, 6, d)
    x[2, 5] = np.inf
    x[4, 0] = np.nan
    one = np.ones(d, np.float32)
    got = run(x, None, one, dy, None, "f32", kept=kept, out8=True)
    rows = [0, 1, 3, 5]
    clean = run(x[rows], None, one, dy[rows], None, "f32", kept=kept, out8=True)
    for k in ("out", "dx"):
        assert np.array_equal(got[k][rows], clean[k]) and np.isnan(got[k][[2, 4]]).any(1).all()
    assert np.array_equal(got["out8"][rows], clean["out8"]) and np.array_equal(got["out8_s"][rows], clean["out8_s"])
    assert got["out8_s"][2, 0] == 255 and (got["out8_s"][4] == 255).all()
