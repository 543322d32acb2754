"""Products of the fp32 head: three bf16 parts of each factor hold its 24 bits, and what the six products of parts leave out of a term is at
most 2^-24 of it."""
import numpy as np
import pytest

from tests.lm_util import U32, normal, within
from tests.test_gpu_head_loss import reference, run

pytestmark = pytest.mark.gpu


LOW = np.float32(1 + 2.0 ** -7 - 2.0 ** -23)   # seven zeros and sixteen ones behind the point: cut into parts, most of it is in the lower two


@pytest.mark.parametrize("T,V,d", [(200, 300, 256), (200, 300, 72), (150, 300, 2100), (140, 5000, 64)])
def test_a_term_keeps_its_bits(T, V, d):
    """Logits of one term a row: 0 but for row 0 of W, whose logit of 64 to 130 is the loss of every other target (the others' exponentials
    are below 2^-80 of its own)."""
    rng = np.random.default_rng(d)
    k = rng.integers(0, d)
    x, w = np.zeros((T, d), np.float32), np.zeros((V, d), np.float32)
    x[:, k] = np.where(rng.random(T) < 0.5, LOW + rng.integers(0, 4, T) * 2.0 ** -7, 1 + rng.random(T))
    x[:2, k] = LOW, np.nextafter(np.float32(2), np.float32(0))
    w[0, k] = 64 * LOW
    y = rng.integers(1, V, T).astype(np.int32)
    want = x[:, k].astype(np.float64) * w[0, k].astype(np.float64)
    assert want.min() > 60
    # what is left out 1, the last of the six additions 2 (a matrix core may cut instead of rounding), those before it 2^-6 of that
    within(run(x, w, y, "f32", stats=False)["loss"], want, 3.1 * U32 * want)


@pytest.mark.parametrize("T", [130, 300])
def test_factors_near_the_ends_of_fp32(T):
    """Factors of 3.4e38, whose leading part would round to infinity, against small ones, and factors of 1e-33 (2^-110 and less), which
    lose up to 2^-134: here nothing that counts."""
    rng = np.random.default_rng(T)
    V, d = 260, 64
    x, w = normal(rng, T, d), normal(rng, V, d, std=0.1)
    big = np.float32(3.4028235e38)
    x[:, 5], w[:, 5] = big, normal(rng, V) * np.float32(2e-39)              # (denormals)
    x[:, 9], w[:, 9] = normal(rng, T) * np.float32(2e-33), np.float32(1e30)
    x[1, 5], x[2, 5] = -big, np.float32(3.3961775e38)                       # (the last is 2^128 (1 - 2^-9) - 1 unit: rounds to infinity or not)
    y = rng.integers(0, V, T).astype(np.int32)
    y[0] = -1
    got, ref = run(x, w, y, "f32", stats=False), reference(x, w, y, "f32")
    # denormals of 2e-39 keep 2^-134 / 2e-39 = 2^-5.4 of themselves at worst, in products of up to 0.7: absolute errors of up to 3.4e38 x 2^-134
    e = 2 * float(big) * 2.0 ** -134 * 1.01 + 2 * 1e30 * 2.0 ** -134
    within(got["loss"], ref["loss"][0], np.where(y >= 0, ref["loss"][1] + e, 0.0))
