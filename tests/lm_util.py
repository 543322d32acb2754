"""Helpers of the tests of the operators around the layer: buffers between guard bands, bf16 rounding, units of rounding."""
import importlib

import numpy as np

P = importlib.import_module("omega-ai_amd")
L = importlib.import_module("omega-ai_amd._lib")

U32 = 2.0 ** -24    # a rounding to fp32, relative
U16 = 2.0 ** -8     # ... to bf16
DT = {"f32": L.DTYPE_F32, "bf16": L.DTYPE_BF16}
GUARD = 64          # elements in front of and behind a buffer

_ctx = None


def ctx():
    global _ctx
    if _ctx is None:
        _ctx = P.Context(0)
    return _ctx


def unit(dtype):
    return U16 if dtype == "bf16" else U32


def rounded(a, dtype):
    """fp32 values that the dtype holds."""
    a = np.ascontiguousarray(a, np.float32)
    return P.bf16_bits_to_f32(P.f32_to_bf16_bits(a)) if dtype == "bf16" else a


def normal(rng, *shape, std=1.0, dtype="f32"):
    return rounded(rng.standard_normal(shape) * std, dtype)


class Buf:
    """A device buffer of `shape` in the middle of a larger one whose other elements hold a pattern; `shift` elements further on, so
    that the address is aligned to nothing but its element."""

    def __init__(self, shape, dtype, values=None, shift=0, fill=float("nan")):
        self.shape, self.dtype = tuple(shape), dtype
        n = int(np.prod(shape, dtype=np.int64))
        self.at = GUARD + shift
        self.host = np.full(n + 2 * GUARD + shift, 7 if dtype == "i32" else fill, np.int32 if dtype == "i32" else np.float32)
        self.host[:self.at], self.host[self.at + n:] = 7, 7
        if values is not None:
            self.host[self.at:self.at + n] = np.asarray(values).reshape(-1)
        self.all = P.DeviceBuffer.from_numpy(ctx(), self.host, dtype)
        es = 2 if dtype == "bf16" else 4
        self.buf = P.DeviceBuffer.wrap(ctx(), self.all.ptr.value + self.at * es, self.shape, dtype)
        self.ptr = self.buf.ptr

    def get(self):
        """The values; fails if an element outside the buffer has changed."""
        got, n = self.all.to_numpy(), int(np.prod(self.shape, dtype=np.int64))
        assert (got[:self.at] == 7).all() and (got[self.at + n:] == 7).all(), "written outside the buffer"
        return got[self.at:self.at + n].reshape(self.shape)

    def free(self):
        self.all.free()


def within(got, ref, tol, what=""):
    """Every element within its tolerance of the 64-bit reference; no number where the reference has one fails."""
    got, ref, tol = np.asarray(got, np.float64), np.asarray(ref, np.float64), np.broadcast_to(np.asarray(tol, np.float64), np.shape(ref))
    bad = ~(np.abs(got - ref) <= tol)
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} off, first at {at}: got {got[at]!r}, want {ref[at]!r} +- {tol[at]!r}")
