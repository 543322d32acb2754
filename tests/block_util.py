"""Plain forms of the operators around the experts, in 64 bits, for their tests."""
import itertools

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
        s = np.maximum(np.float32(most) * np.float32(1.0 / 127.0), np.float32(2.0 ** -126)).astype(np.float32)
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


# Two evaluations in 64 bits of a group's worth differ by up to 2^-49 of it: each by an exponential (1 unit of 2^-53; the two sides: 2), a quotient
# (a half; 1) and the addition of two (a half; 1) - the sum of a softmax is the same for all groups of a token -, with twice that for the spread between two
# groups.  Sums like e^(x+2u) + e^x against 2 e^(x+u), u a last place of fp32, are nearer to each other than that; which of those groups stays is open.
GROUPS_OPEN = 2.0 ** -48


def choices(z, b, K, ids, t, **kw):
    """Whether a token's ids follow from the definition with one of the sets of groups that 64 bits leave open (of groups with the same logits
    and biases the first)."""
    groups, top = kw["groups"], kw["top"]
    of, best = group_worths(z[t:t + 1], b, kw.get("sigmoid", False), groups, kw["best"])
    of, best = of[0], best[0]
    edge = np.sort(of)[::-1][top - 1]
    sure = [g for g in range(groups) if of[g] > edge + GROUPS_OPEN * abs(edge)]
    maybe = [g for g in range(groups) if abs(of[g] - edge) <= GROUPS_OPEN * abs(edge)]
    for more in itertools.combinations(maybe, top - len(sure)):
        if any(g not in more and g < h and best[g] == best[h] for h in more for g in maybe):
            continue
        shut = ~np.isin(np.arange(z.shape[1]) // (z.shape[1] // groups), sure + list(more))
        zt = np.where(shut, -np.inf, z[t])
        key = zt if b is None else np.where(shut, -np.inf, worths(z[t:t + 1], b, kw.get("sigmoid", False))[0][0])
        order = np.argsort(-key, kind="stable")[:K]
        if np.array_equal(np.where(key[order] > -np.inf, order, -1), ids):
            return True
    return False


def worths(z, b, sigmoid):
    """Worths (-inf: closed) and scores."""
    z = np.asarray(z, np.float64)
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max))
    shut = z == -np.inf
    with np.errstate(all="ignore"):
        if sigmoid:
            s = 1.0 / (1.0 + np.exp(-z))
        else:
            e = np.where(shut, 0.0, np.exp(z - z.max(1, keepdims=True)))
            s = e / np.where(shut.all(1), 1.0, e.sum(1))[:, None]
        worth = s if b is None else s + np.asarray(b, np.float64)
        return np.where(shut | np.isnan(worth), -np.inf, worth), s


def group_worths(z, b, sigmoid, groups, n):
    """Worths of a token's groups, and what they were made of."""
    worth, _ = worths(z, b, sigmoid)
    T, E = worth.shape
    v = -np.sort(-worth.reshape(T, groups, -1), 2)[:, :, :n]
    of = np.where(v[:, :, 0] > -np.inf, np.where(v > -np.inf, v, 0.0).sum(2), -np.inf)
    zb = np.stack([np.asarray(z, np.float64), np.broadcast_to(0.0 if b is None else np.asarray(b, np.float64), (T, E))], 2).reshape(T, groups, -1, 2)
    at = np.argsort(-worth.reshape(T, groups, -1), 2, kind="stable")[:, :, :n]
    made = [[sorted(map(tuple, zb[t, g, at[t, g]].tolist())) for g in range(groups)] for t in range(T)]
    return of, made


def route(z, b, K, sigmoid=False, renorm=True, scale=1.0, groups=1, top=None, best=2, fill=False):
    """ids, w, counts of the definition, and s (scores), token by token in 64 bits."""
    z = np.asarray(z, np.float64)
    T, E = z.shape
    top = groups if top is None else top
    z = np.where(np.isnan(z), -np.inf, np.minimum(z, np.finfo(np.float32).max))
    shut = z == -np.inf
    with np.errstate(all="ignore"):
        if sigmoid:
            s = 1.0 / (1.0 + np.exp(-z))
        else:
            e = np.where(shut, 0.0, np.exp(z - z.max(1, keepdims=True)))
            s = e / np.where(shut.all(1), 1.0, e.sum(1))[:, None]
        worth = s if b is None else s + np.asarray(b, np.float64)
        worth = np.where(shut | np.isnan(worth), -np.inf, worth)
    key = z.copy() if b is None else worth.copy()
    ids, w = np.full((T, K), -1, np.int32), np.zeros((T, K))
    for t in range(T):
        if groups > 1:
            of = np.empty(groups)
            for g in range(groups):
                v = np.sort(worth[t].reshape(groups, -1)[g])[::-1][:best]
                of[g] = v[v > -np.inf].sum() if v[0] > -np.inf else -np.inf
            stays = np.argsort(-of, kind="stable")[:top]
            key[t][~np.isin(np.arange(E) // (E // groups), stays)] = -np.inf
        order = np.argsort(-key[t], kind="stable")[:K]
        held = key[t][order] > -np.inf
        n = int(held.sum())
        ids[t, :n] = order[:n]
        if fill and n < K:
            ids[t, n:] = [e for e in range(E) if e not in set(order[:n])][:K - n]
        if n:
            if not renorm:
                w[t, :n] = s[t, order[:n]]
            else:   # e^-c more of every score: where all of them vanish their ratios do not
                zz = z[t, order[:n]]
                c = zz.max() if not sigmoid else min(zz.max(), 0.0)
                with np.errstate(over="ignore"):
                    v = np.exp(zz - c) if not sigmoid else np.where(zz > 0, 1.0 / (1.0 + np.exp(-zz)), np.exp(np.minimum(zz, 0) - c) / (1.0 + np.exp(np.minimum(zz, 0))))
                w[t, :n] = v / v.sum()
    counts = np.bincount(ids[ids >= 0], minlength=E).astype(np.int32)
    return ids, w * scale, counts, s


def route_back(z, s, ids, w, dw, scale, sigmoid, renorm):
    """dlogits of the definition in 64 bits, and the size of the terms of each (for its tolerance)."""
    T, E = s.shape
    with np.errstate(over="ignore"):
        rest = 1.0 / (1.0 + np.exp(np.asarray(z, np.float64)))    # 1 - s for sigmoid: the difference itself loses all its places at s = 1
    s, w, dw = (np.asarray(a, np.float64) for a in (s, w, dw))
    dz, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        at = np.nonzero((ids[t] >= 0) & (w[t] != 0))[0]
        e, u, d = ids[t, at], w[t, at] / scale, dw[t, at]
        if renorm:
            g = ((d[:, None] - d[None]) * u[None]).sum(1)
            m = (np.abs(d[:, None] - d[None]) * u[None]).sum(1)
            f = w[t, at] * (rest[t, e] if sigmoid else 1.0)
            dz[t, e], size[t, e] = f * g, f * m
        elif sigmoid:
            dz[t, e] = w[t, at] * d * rest[t, e]
            size[t, e] = np.abs(dz[t, e])
        else:
            dot, m = (w[t, at] * d).sum(), np.abs(w[t, at] * d).sum()
            dz[t], size[t] = -s[t] * dot, s[t] * m
            dz[t, e] += w[t, at] * d
            size[t, e] += np.abs(w[t, at] * d)
    return dz, size
