"""RMS norm with its output in 8 bits where fp32 products of the row, its factor and gamma lose places below 2^-126: codes are those of 64 bits all the same."""
import numpy as np
import pytest

from tests import block_util as B
from tests import test_gpu_rmsnorm as R

pytestmark = pytest.mark.gpu


def check(x, gamma, dtype, what):
    ref = R.reference(x, None, gamma, np.zeros_like(x), None, dtype, False)
    got = R.run(x, None, gamma, np.zeros_like(x), None, dtype, out8=True)
    codes, scales = B.mx_codes(ref["y"])
    assert np.array_equal(got["out8_s"], scales), what
    assert np.array_equal(got["out8"], codes), (what, int((got["out8"] != codes).sum()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", [(600, 1000), (300, 2050), (80, 8200)])
def test_outputs_below_the_least_normal_number(T, d, dtype):
    rng = np.random.default_rng(d)
    x = R.rounded(rng.standard_normal((T, d)), dtype)
    for power in (-126, -132, -136, -142):
        check(x, (rng.standard_normal(d) * 2.0 ** power).astype(np.float32), dtype, power)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("T,d", [(600, 1000), (300, 2050), (80, 8200)])
def test_rows_far_below_their_largest_element(T, d, dtype):
    """x q below 2^-126, as it is and with a large gamma."""
    rng = np.random.default_rng(d + 1)
    x = R.rounded(rng.standard_normal((T, d)) * 2.0 ** -66, dtype)
    x[:, 5] = 2.0 ** 66
    one = (rng.standard_normal(d) + 1).astype(np.float32)
    for power in (0, 9, 40):
        check(x, (one * 2.0 ** power).astype(np.float32), dtype, power)
    x[:, 5] = 2.0 ** 96
    for power in (0, 100, 110):
        check(x, (one * 2.0 ** power).astype(np.float32), dtype, power)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_factors_below_the_least_normal_number(dtype):
    rng = np.random.default_rng(2)
    x = R.rounded(np.where(rng.random((400, 1500)) < 0.5, 1.0, -1.0) * (2.0 ** 127 * (1.2 + 0.79 * rng.random((400, 1500)))), dtype)
    check(x, (rng.standard_normal(1500) + 1).astype(np.float32), dtype, "")
