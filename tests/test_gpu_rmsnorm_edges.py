"""RMS norm: rows whose mean is 0 or infinite, and batches around the numbers of rows whose gradient of gamma one workgroup forms."""
import numpy as np
import pytest

from tests import test_gpu_rmsnorm as R
from tests.lm_util import DT, Buf, ctx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [40, 700, 3000, 8300])
def test_means_of_zero_and_infinity(d, dtype):
    """1 / sqrt(infinity) = 0: what is finite in such a row becomes 0; without eps a row of zeros has an infinite factor, and no numbers."""
    rng = np.random.default_rng(d)
    x = np.asarray(R.normal(rng, 4, d, dtype=dtype)).copy()
    x[1, d // 2], x[2] = -np.inf, 0
    c, gamma = ctx(), np.full(d, 2, np.float32)
    for eps, factor in ((0.0, np.inf), (1e-6, 1e3)):
        xb, gb, ob, rb = Buf((4, d), dtype, x), Buf((d,), "f32", gamma), Buf((4, d), dtype), Buf((4,), "f32")
        c.check(c.lib.omega_hip_rmsnorm_forward(c.handle, xb.ptr, None, DT[dtype], 4, d, gb.ptr, eps, None, ob.ptr, None, None, None, None, rb.ptr))
        out, rstd = ob.get(), rb.get()
        assert rstd[1] == 0 and np.isnan(out[1, d // 2]) and not np.delete(out[1], d // 2).any()
        assert (np.isinf(rstd[2]) and np.isnan(out[2]).all()) if eps == 0 else (abs(rstd[2] / factor - 1) < 1e-6 and not out[2].any())
        for t in (0, 3):
            v = x[t].astype(np.float64)
            want = 2 * v / np.sqrt((v * v).mean() + np.float64(np.float32(eps)))
            R.within(out[t], want, (R.unit(dtype) * (1 + 1e-3) + 4 * R.U32) * np.abs(want), t)
        for b in (xb, gb, ob, rb):
            b.free()


@pytest.mark.parametrize("kept", [False, True])
@pytest.mark.parametrize("d,most", [(100, 16), (1000, 16), (2000, 4), (4000, 4), (8192, 4), (8201, 4)])
def test_rows_that_one_workgroup_takes(d, most, kept):
    for T in (2, most - 1, most, most + 1):
        rng = np.random.default_rng(T + d)
        x, res, gamma, dy, dsum = R.inputs(rng, T, d, "bf16")
        R.check(R.run(x, res, gamma, dy, dsum, "bf16", 0, kept), R.reference(x, res, gamma, dy, dsum, "bf16", kept), "bf16", T)
