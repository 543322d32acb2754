"""Gradient of the embedding where one id has many tokens: whole blocks of 64 sorted places, which are summed apart in batches that have
two of them or more, against plain sums in 64 bits."""
import numpy as np
import pytest

from tests.lm_util import DT, U32, Buf, ctx, normal, unit, within
from tests.test_gpu_embedding import grad_reference

pytestmark = pytest.mark.gpu


def check(ids, V, d, dtype="f32", grad="f32", add=0, scale=1.0, shift=0):
    """The gradient of random rows for these ids, and that a second run gives the same bits."""
    ids = np.asarray(ids, np.int32)
    T = len(ids)
    rng = np.random.default_rng(T + V + d)
    dout, before = normal(rng, T, d, dtype=dtype), normal(rng, V, d, dtype=grad)
    ref, mag, n = grad_reference(ids, dout, V, scale)
    ib, db = Buf((T,), "i32", ids), Buf((T, d), dtype, dout, shift)
    got = []
    for _ in range(2):
        gb = Buf((V, d), grad, before if add else None, shift)
        ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, ib.ptr, T, db.ptr, DT[dtype], V, d, scale, add, gb.ptr, DT[grad]))
        got.append(gb.get())
        gb.free()
    assert np.array_equal(got[0], got[1]), "the same inputs give other bits"
    want = ref + (before if add else 0)
    # n additions and the scale's product, each within a rounding of the sum of magnitudes; the sum with what was there; the result's rounding
    tol = (n[:, None] + 2) * U32 * mag + (U32 * (np.abs(want) + mag) if add else 0) + unit(grad) * np.abs(want) * (1 + 1e-3)
    within(got[0], want, tol, (T, V, d, dtype, grad, add))
    rows = n == 0
    assert np.array_equal(got[0][rows], before[rows] if add else np.zeros_like(got[0][rows])), "rows without tokens"
    for b in (ib, db):
        b.free()


@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("T", [63, 64, 65, 100, 127, 128, 130])
def test_a_batch_of_a_block_or_two(T, dtype, grad):
    """As a batch padded with one id is: its block of 64 places has a sum of its own from 128 tokens on, below they are added one by one."""
    first = min(T, 64)
    runs = ([0] * T, [3] * T, [0] * first + [5] * (T - first), [5] * (T - first) + [0] * first, [2] * (T - first) + [7] * first, [-1] * (T - first) + [19] * first)
    for k, ids in enumerate(runs):
        for add in (0, 1):
            check(ids, 20, (3, 12, 130, 1030)[(k + T) % 4], dtype, grad, add, scale=2.5, shift=k % 3)
    check([0] * T, 1, 8, dtype, grad)           # a table of one row
