"""Rows in 8 bits whose scale is next to the least one: half of a scale below 2^-125 is not always a number of fp32."""
import numpy as np
import pytest

from tests import block_util as B
from tests import test_gpu_keep8 as K

pytestmark = pytest.mark.gpu


def test_quotients_next_to_a_half_of_the_least_scales():
    """Scales S 2^-149 with S odd, elements one 2^-149 from one and a half or from half of it: codes -2 .. 2, the nearest."""
    rng = np.random.default_rng(1)
    least = 2.0 ** -149
    S = rng.integers(2 ** 22, 2 ** 24 // 3, 4000) * 2 + 1            # (one and a half of it is a whole multiple of 2^-149 below 2^24)
    # the largest magnitude whose product with 1 / 127 rounds to the scale
    most = (127.0 * S * least).astype(np.float32)
    fits = (most * np.float32(1.0 / 127.0)).astype(np.float64) == S * least
    S, most = S[fits], most[fits]
    assert len(S) > 500
    x = np.zeros((len(S), 128), np.float32)
    x[:, 0] = most
    at = np.stack([S + (S - 1) // 2, S + (S + 1) // 2, (S - 1) // 2, (S + 1) // 2], 1)
    x[:, 1:9] = np.concatenate([at, -at], 1) * least
    assert np.array_equal(x[:, 1:5].astype(np.float64), at * least)
    codes, scales = B.int8_codes(x)
    assert np.array_equal(scales[:, 0].astype(np.float64), S * least) and (codes[:, 1:9] == [1, 2, 0, 1, -1, -2, 0, -1]).all()
    K.check(x, "f32", "int8")
