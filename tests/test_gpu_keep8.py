"""Rows in 8 bits: codes, scales and values against the definition, bit for bit (it leaves no room)."""
import numpy as np
import pytest

from tests import block_util as B
from tests.lm_util import DT, L, Buf, P, ctx, rounded

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 128), (2, 7), (3, 31), (3, 33), (5, 127), (4, 129), (2, 1000), (9, 256), (600, 40), (3, 8200), (33, 2050)]


class Bytes(Buf):
    """Buf of single bytes."""

    def __init__(self, shape, values=None, shift=0):
        n = int(np.prod(shape, dtype=np.int64))
        self.shape, self.dtype, self.at = tuple(shape), "u8", 64 + shift
        self.host = np.full(n + 128 + shift, 99, np.uint8)
        self.host[:self.at], self.host[self.at + n:] = 7, 7
        if values is not None:
            self.host[self.at:self.at + n] = np.asarray(values).reshape(-1)
        self.all = P.DeviceBuffer.from_numpy(ctx(), self.host, "u8")
        self.buf = P.DeviceBuffer.wrap(ctx(), self.all.ptr.value + self.at, self.shape, "u8")
        self.ptr = self.buf.ptr


def hold(x, dtype, form, shift=0):
    """Codes, scales, and the values in both types."""
    T, d = x.shape
    c, lib = ctx(), ctx().lib
    kind = {"int8": L.KEEP8_INT8, "mx": L.KEEP8_MX}[form]
    src, codes = Buf((T, d), dtype, x, shift), Bytes((T, d), shift=shift)
    scales = Buf((T, -(-d // 128)), "f32", shift=shift) if form == "int8" else Bytes((T, -(-d // 32)), shift=shift)
    c.check(lib.omega_hip_keep8_save(c.handle, src.ptr, DT[dtype], T, d, kind, codes.ptr, scales.ptr))
    got = [codes.get(), scales.get()]
    for to in ("f32", "bf16"):
        out = Buf((T, d), to, shift=shift)
        c.check(lib.omega_hip_keep8_load(c.handle, codes.ptr, scales.ptr, kind, T, d, out.ptr, DT[to]))
        got.append(out.get())
        out.free()
    for b in (src, codes, scales):
        b.free()
    return got


def check(x, dtype, form, shift=0):
    codes, scales, v32, v16 = hold(x, dtype, form, shift)
    want_codes, want_scales = B.int8_codes(x) if form == "int8" else B.mx_codes(x)
    assert np.array_equal(scales, want_scales, equal_nan=form == "int8")
    good = np.repeat(np.isfinite(want_scales) if form == "int8" else want_scales != 255, 128 if form == "int8" else 32, 1)[:, :x.shape[1]]
    got = codes.view(np.int8) if form == "int8" else codes
    assert np.array_equal(got[good], want_codes[good]), np.argwhere(got != want_codes)[:3]
    want = B.int8_values(want_codes, want_scales) if form == "int8" else B.mx_values(want_codes, want_scales).astype(np.float32)
    assert np.array_equal(v32, want, equal_nan=True) and np.isnan(v32[~good]).all()
    with np.errstate(invalid="ignore"):
        assert np.array_equal(v16[good], rounded(want, "bf16")[good]) and np.isnan(v16[~good]).all()


@pytest.mark.parametrize("form", ["int8", "mx"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", SHAPES)
def test_against_the_definition(T, d, dtype, form):
    rng = np.random.default_rng(T * 10000 + d)
    for shift, spread in ((0, 0.0), (1, 3.0), (3, 20.0)):
        x = rng.standard_normal((T, d)) * np.exp(rng.standard_normal((T, 1)) * spread)
        x[:, rng.random(d) < 0.02] *= 50.0
        check(rounded(x, dtype), dtype, form, shift)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quotients_on_and_next_to_a_half(dtype):
    """Whole and half multiples of a scale, and their neighbours in fp32: every code and border."""
    for most in (127.0, 127.0 * 2.0 ** -20, 254.0 * 3.0, 1.0, 3.3e38, 2.0 ** -118):
        s = np.float32(np.float32(most) * np.float32(1.0 / 127.0))
        near = (np.arange(-253, 254) * 0.5 * np.float64(s)).astype(np.float32)
        x = np.concatenate([near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(-np.inf))])
        x = x[np.abs(x) < most]
        x = np.pad(x, (0, -len(x) % 127)).reshape(-1, 127)
        x = np.concatenate([np.full((len(x), 1), most, np.float32), x], 1)
        check(rounded(x, dtype), dtype, "int8")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_borders_of_e4m3(dtype):
    """Every value of the format, the middle of every two and the neighbours of those, at several scales; largest magnitudes around 448 2^k."""
    mid = (B.E4M3[1:] + B.E4M3[:-1]) / 2
    for k in (0, 5, -30, -100, 110):
        near = (np.concatenate([B.E4M3, mid]) * 2.0 ** k).astype(np.float32)
        x = np.concatenate([near, np.nextafter(near, np.float32(np.inf)), np.nextafter(near, np.float32(0))])
        x = x[x < 448.0 * 2.0 ** k]
        x = np.pad(np.concatenate([x, -x]), (0, -2 * len(x) % 31)).reshape(-1, 31)
        check(rounded(np.concatenate([np.full((len(x), 1), 448.0 * 2.0 ** k), x], 1), dtype), dtype, "mx")
    top = np.float32(448.0) * np.exp2(np.arange(-120, 117)).astype(np.float32)
    top = np.concatenate([top, np.nextafter(top, np.float32(np.inf)), np.nextafter(top, np.float32(0))])
    check(rounded(np.concatenate([top[:, None], top[:, None] * np.linspace(-1, 1, 31, dtype=np.float32)], 1), dtype), dtype, "mx")


@pytest.mark.parametrize("form", ["int8", "mx"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_zeros_tiny_values_and_no_numbers(dtype, form):
    rng = np.random.default_rng(5)
    x = rounded(rng.standard_normal((6, 300)), dtype)
    x[0] = 0
    x[1] *= np.float32(2.0 ** -126)     # below the least scale, some of them subnormal
    x[2, 5] = np.inf
    x[3, 200] = -np.inf
    x[4, 299] = np.nan
    x[5] = np.float32(3.38e38) * np.sign(x[5])
    check(rounded(x, dtype), dtype, form)


def test_no_rows_and_more_than_the_caches_hold():
    c = ctx()
    for form in (L.KEEP8_INT8, L.KEEP8_MX):
        c.check(c.lib.omega_hip_keep8_save(c.handle, None, 0, 0, 5, form, None, None))
        c.check(c.lib.omega_hip_keep8_load(c.handle, None, None, form, 0, 5, None, 0))
    T, d = 70000, 4096                  # 2^28 elements and more, 0.6 GB of bf16
    x = P.DeviceBuffer(c, (T, d), "bf16")
    x.fill_normal(3, 1, 1.0)
    layer = P.Keep8Layer(d, ctx=c, dtype="bf16")
    layer.save(x)
    back = layer.load()
    at = [0, 1, 40000, 65535, 65536, T - 1]
    row = lambda b, t: P.DeviceBuffer.wrap(c, b.ptr.value + t * d * 2, (1, d), "bf16").to_numpy()  # noqa: E731
    for t in at:
        src = row(x, t)
        assert np.array_equal(row(back, t), rounded(B.int8_values(*B.int8_codes(src)), "bf16"))
    layer.close()
    x.free()
