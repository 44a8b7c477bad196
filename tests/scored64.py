"""Group norm, 8-bit integer rows and attention with changed scores in float64 (numpy), from their definitions, with bounds on
what fp32 arithmetic and one rounding may add."""
import numpy as np

import rows64 as ref

E = ref.E


def group_norm(x, at, gamma, beta, groups, eps, act):
    """(value, bound, rows in a sequence).  Sums are of 64 bits and the mean has two parts, so what is left is fp32's: two
    subtractions, the inverse root, its product with gamma and the product with that (5 roundings of t = (x - m) / s * gamma),
    the sum with beta (one of z).  Activations: slopes up to 1.13; their own error some 16 roundings, and of the exponential's
    argument (up to 1.6 |z| + 0.08 |z|^3, three roundings; erfc: z^2 / 2) no more than 4 z^2 + 4 |z|."""
    n, c = x.shape
    y, tol, inside = np.zeros((n, c)), np.zeros((n, c)), np.zeros(n, bool)
    g = np.ones(c) if gamma is None else gamma
    b = np.zeros(c) if beta is None else beta
    for s in range(len(at) - 1):
        rows = slice(at[s], at[s + 1])
        inside[rows] = True
        if at[s + 1] == at[s]:
            continue
        v = x[rows].reshape(at[s + 1] - at[s], groups, -1)
        mean = v.mean((0, 2), keepdims=True)
        d = v - mean
        t = (d / np.sqrt((d * d).mean((0, 2), keepdims=True) + eps)).reshape(-1, c) * g
        z = t + b
        y[rows] = ref.activate(z, act)
        tol[rows] = 1.13 * E * (5 * np.abs(t) + 2 * np.abs(z))
        if act != "none":
            tol[rows] += (16 + 4 * z * z + 4 * np.abs(z)) * E * np.abs(y[rows])
    return y, tol, inside


def int8_rows(v):
    """(codes, scales) of rows; v float64 values whose product with 127 float64 holds."""
    most = np.abs(v).max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        codes = np.where(most > 0, np.rint(127 * v / most), 0)
    return codes, most / 127


def int8_linear(codes, scales, w, b, act, r, fp32):
    """(value, bound): sums are exact; their conversion, two products with scales (each rounded itself) and the bias take six
    roundings.  Activations as in rows64.linear_act."""
    wc, ws = int8_rows(w)
    t = (codes @ wc.T) * scales * ws.T
    z = t + (0 if b is None else b)
    err = E * (6 * np.abs(t) + 2 * np.abs(z))
    if act != "none":
        err = 1.13 * err + 2.0 ** (-21 if fp32 else -19) * np.abs(z)
    y = ref.activate(z, act)
    if r is not None:
        y = y + r
        err = err + E * np.abs(y)
    return y, err


def distances(q_xyz, k_xyz):
    d = q_xyz[:, None, 1:].astype(np.float64) - k_xyz[None, :, 1:]
    return np.sqrt((d * d).sum(2))


def attention(q, k, v, scale, group, q_at, k_at, half_p, cap=0.0, slopes=None, q_xyz=None, k_xyz=None, causal=False,
              prefix=None):
    """As rows64.attention.  A score's error d has besides: the tanh's (8 E of the cap: its value is one less a quotient of
    two parts in 2^23) and the distance's and its product's (6 E of it); all scores of a row are rounded at the size of their
    terms.  What is not seen is left out."""
    nq, heads, dim = q.shape
    y, tol = np.zeros((nq, heads, dim)), np.zeros((nq, heads, dim))
    inside = np.zeros(nq, bool)
    for s in range(len(q_at) - 1):
        qs, ks = slice(q_at[s], q_at[s + 1]), slice(k_at[s], k_at[s + 1])
        inside[qs] = True
        m, nk = q_at[s + 1] - q_at[s], k_at[s + 1] - k_at[s]
        if nk == 0 or m == 0:
            continue
        place = (np.arange(m) + nk - m)[:, None]
        seen = np.ones((m, nk), bool)
        if causal:
            seen = (np.arange(nk) <= place) | (np.arange(nk) < (0 if prefix is None else prefix[s]))
        far = np.abs(place - np.arange(nk)) if q_xyz is None else distances(q_xyz[qs], k_xyz[ks])
        for h in range(heads):
            kk, vv, qq = k[ks, h // group], v[ks, h // group], q[qs, h]
            some = seen.any(0)  # (a key that no query sees may hold anything)
            kk, vv = np.where(some[:, None], kk, 0), np.where(some[:, None], vv, 0)
            z = scale * (qq @ kk.T)
            size = np.abs(z)
            if cap:
                z = cap * np.tanh(z / cap)
                size = np.minimum(size, cap) + 8 * cap
            if slopes is not None:
                z = z - slopes[h] * far
                size = size + 6 * np.abs(slopes[h]) * far
            z = np.where(seen, z, -np.inf)
            top = z.max(1, keepdims=True)
            top = np.where(np.isfinite(top), top, 0)
            p = np.exp(z - top)
            total = p.sum(1, keepdims=True)
            p = p / np.where(total > 0, total, 1)
            y[qs, h] = p @ vv
            walk = abs(scale) * 8 * np.sqrt(dim) * E * np.sqrt((qq * qq) @ (kk * kk).T)
            # A score matters as its weight does: what is far below the top may be off by more.
            matters = p > 2.0 ** -40
            size = np.where(matters, size + np.abs(np.where(seen, z, 0)) + np.abs(top), 0)
            d = np.max(np.where(matters, walk, 0) + 4 * E * size + 4 * E, 1, keepdims=True)
            most = (d + half_p) * (p @ np.abs(vv))
            rms = np.sqrt((p * p) @ (vv * vv))
            tol[qs, h] = np.minimum(most, 8 * (d + half_p) * rms + d * np.abs(y[qs, h])) + \
                8 * np.sqrt(nk) * E * (rms + np.abs(y[qs, h])) + 4 * E * np.abs(y[qs, h]) + 2.0 ** -30 * np.abs(vv).max()
    return y, tol, inside
