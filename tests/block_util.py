"""Plain forms of the operators around the experts, in 64 bits, for their tests."""
import numpy as np

INT8_GROUP, MX_GROUP = 128, 32
# the magnitudes that e4m3 holds: eighths of the powers of two from 2^-6 to 2^8 (but 480), multiples of 2^-9 below
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1])


def grouped(x, n):
    T, d = x.shape
    g = np.zeros((T, -(-d // n) * n), np.float64)
    g[:, :d] = x
    return g.reshape(T, -1, n)


def nearest_even(q):
    return np.rint(q)   # (NumPy's: halves to even)


def int8_codes(x):
    """Codes [T,d] (int8) and scales [T,groups] (fp32) of the definition; groups that hold no numbers: scale NaN, code 0."""
    g = grouped(np.asarray(x, np.float64), INT8_GROUP)
    with np.errstate(invalid="ignore", over="ignore"):
        most = np.abs(g).max(2)
        s = np.maximum(np.float32(most) / np.float32(127.0), np.float32(2.0 ** -126)).astype(np.float32)
        bad = ~np.isfinite(most)
        q = nearest_even(g / s.astype(np.float64)[:, :, None])
    q[bad] = 0
    s[bad] = np.nan
    return q.reshape(len(x), -1)[:, :x.shape[1]].astype(np.int8), s


def int8_values(codes, s):
    """fp32 products, as the definition says."""
    return (codes.astype(np.float32) * np.repeat(s, INT8_GROUP, 1)[:, :codes.shape[1]]).astype(np.float32)


def mx_exponents(most):
    k = np.full(most.shape, -127, np.int64)
    with np.errstate(invalid="ignore"):
        for _ in range(300):
            k += most > 448.0 * np.exp2(k.astype(np.float64))
    return k


def mx_codes(x):
    """Codes (e4m3 bits, uint8) and scale bytes of the definition."""
    x = np.asarray(x, np.float64)
    g = grouped(x, MX_GROUP)
    bad = ~np.isfinite(g).all(2)
    g[bad] = 0
    k = mx_exponents(np.abs(g).max(2))
    u = np.abs(g) * np.exp2(-k.astype(np.float64))[:, :, None]
    up = np.searchsorted(E4M3, u).clip(max=len(E4M3) - 1)
    low = (up - 1).clip(min=0)
    a, b = u - E4M3[low], E4M3[up] - u
    at = np.where((a < b) | ((a == b) & (low % 2 == 0)), low, up)
    codes = (at | np.where(np.signbit(g), 128, 0)).astype(np.uint8)
    return codes.reshape(len(x), -1)[:, :x.shape[1]], np.where(bad, 255, k + 127).astype(np.uint8)


def mx_values(codes, scales):
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    v = E4M3[np.minimum(codes & 127, len(E4M3) - 1)] * np.where(codes & 128, -1.0, 1.0)
    return v * np.repeat(s, MX_GROUP, 1)[:, :codes.shape[1]]
