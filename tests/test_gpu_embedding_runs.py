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


def shuffled(rng, runs, pad=0):
    """Ids 0, 1, ... with the given numbers of tokens and `pad` tokens that have none, in any order."""
    ids = np.concatenate([np.full(n, v) for v, n in enumerate(runs)] + [rng.choice([-1, len(runs), 2 ** 31 - 1], pad)])
    rng.shuffle(ids)
    return ids.astype(np.int32)


# one block of 64 and one of 4096 places and what is next to them; runs that begin on a block's border and in its middle, long ones over
# several blocks of 4096, a last one that ends the list inside a block
RUNS = [[4096, 8192, 63, 64, 65, 4095, 4097, 127, 128, 129, 1, 3 * 4096 + 70, 200],
        [70, 20000, 0, 5, 16384, 4030, 4096],
        [1] * 300 + [40000] + [2] * 100,
        [32768], [65537]]


@pytest.mark.parametrize("runs", range(len(RUNS)))
@pytest.mark.parametrize("d,dtype,grad,add,pad", [(24, "bf16", "f32", 0, 0), (37, "f32", "f32", 1, 1000), (3, "bf16", "bf16", 0, 33), (260, "bf16", "bf16", 1, 4096)])
def test_blocks_of_blocks(runs, d, dtype, grad, add, pad):
    """From 32768 tokens on, 64 blocks of one id are summed once more."""
    rng = np.random.default_rng(runs + d)
    ids = shuffled(rng, RUNS[runs], pad)
    assert len(ids) >= 32768
    check(ids, len(RUNS[runs]), d, dtype, grad, add, scale=0.5)


@pytest.mark.parametrize("V", [300, 512, 600, 2000])
def test_many_tokens_of_few_ids(V):
    """More tokens of 512 neighbouring ids in a wave's share of the batch than it notes, for all waves, for some, and for some ids."""
    T = 40000
    rng = np.random.default_rng(V)
    ids = rng.integers(0, V, T)
    ids[T // 2:] = rng.integers(0, 100 if V == 2000 else V, T - T // 2)
    ids[rng.random(T) < 0.1] = -1
    check(ids, V, 20, "bf16", "f32")
    check(np.sort(ids), V, 9, "f32", "f32", add=1)


@pytest.mark.parametrize("V,d,grad", [(25000, 1030, "f32"), (50001, 1030, "bf16"), (8500000, 3, "f32"), (6300000, 8, "bf16")])
def test_a_gradient_larger_than_the_caches(V, d, grad):
    """96 MiB and more are written past them."""
    rng = np.random.default_rng(d)
    T, n = 700, V * d
    assert n * (2 if grad == "bf16" else 4) >= 96 << 20
    ids = np.where(rng.random(T) < 0.3, 5, rng.integers(0, V, T)).astype(np.int32)
    ids[:2] = 0, V - 1
    dout = normal(rng, T, d, dtype="bf16")
    some, at = np.unique(ids, return_inverse=True)
    ref, mag, cnt = grad_reference(at, dout, len(some), 3.0)
    ib, db, gb = Buf((T,), "i32", ids), Buf((T, d), "bf16", dout), Buf((V, d), grad)
    ctx().check(ctx().lib.omega_hip_embedding_backward(ctx().handle, ib.ptr, T, db.ptr, DT["bf16"], V, d, 3.0, 0, gb.ptr, DT[grad]))
    got = gb.get()
    within(got[some], ref, (cnt[:, None] + 2) * U32 * mag + unit(grad) * np.abs(ref) * (1 + 1e-3))
    got[some] = 0
    assert not got.any()                        # (no number left of what was there either)
    for b in (ib, db, gb):
        b.free()
