"""Clipping of more than the caches hold, which is written past them, and of lists around the number of chunks that every workgroup adds
up for itself."""
import numpy as np
import pytest

from tests.lm_util import P, U32, Buf, ctx, normal, unit, within

pytestmark = pytest.mark.gpu


def clip_and_check(data, place, share):
    """data: (values, dtype, shift) of every tensor; the limit is `share` of the norm."""
    norm = np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a, _, _ in data))
    src = [Buf((len(a),), dt, a, sh) for a, dt, sh in data]
    dst = src if place == "in" else [Buf((len(a),), dt, None, sh + (place == "crooked")) for a, dt, sh in data]
    clip = P.GradClip(ctx(), [b.buf for b in src], out=None if place == "in" else [b.buf for b in dst])
    got = clip.clip(share * norm).to_numpy()
    coef = min(1.0, float(np.float32(share * norm)) / (norm + 1e-6))
    assert abs(got[0] - norm) <= 2 * U32 * norm and abs(got[1] - coef) <= 2 * U32 * coef
    for (a, dt, _), d in zip(data, dst):
        # the coefficient's rounding, the product's and the result's
        within(d.get(), a.astype(np.float64) * coef, (3 * U32 + unit(dt)) * np.abs(a) * coef, (len(a), dt))
    clip.close()
    for b in src + (dst if place != "in" else []):
        b.free()


@pytest.mark.parametrize("place", ["in", "out", "crooked"])
def test_larger_than_the_caches(place):
    """102 MB in both types, not aligned to 16 bytes."""
    rng = np.random.default_rng(1)
    clip_and_check([(normal(rng, 21_000_003), "f32", 1), (normal(rng, 9_000_001, dtype="bf16"), "bf16", 3), (normal(rng, 17), "f32", 0)], place, 0.5)


@pytest.mark.parametrize("chunks", [1023, 1024, 1025])
def test_around_the_number_of_chunks_that_is_few(chunks):
    rng = np.random.default_rng(chunks)
    n = chunks * 8192 - 100
    clip_and_check([(normal(rng, n - 50), "f32", 0)], "in", 0.25)
    # the same number of chunks in more tensors than a launch's table holds
    sizes = [8192] * 100 + [(chunks - 100) * 8192 - 5]
    clip_and_check([(normal(rng, k, dtype="bf16"), "bf16", i % 2) for i, k in enumerate(sizes)], "in", 2.0)
