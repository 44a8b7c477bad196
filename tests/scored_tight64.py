"""Attention with changed scores in float64 (numpy), from its definition, with bounds that follow a score's own size: a cap's
tanh is off by a part of its value, not of the cap, but where the caller grants the latter."""
import numpy as np

import rows64 as ref

E = ref.E


def attention(q, k, v, scale, half, cap=0.0, slopes=None, q_xyz=None, k_xyz=None, causal=False, prefix=0, of_cap=0.0):
    """One sequence; q [nq][heads][dim], k, v [nk][kv_heads][dim] -> (value, bound before the output's rounding).

    A product of q and k is a sum of dim terms, a walk of 8 sqrt(dim) E of their root sum of squares.  The score's scale takes
    2 roundings of it; a tanh 16 of its value (the exponential 2, its argument 4.4, a sum, a difference, a reciprocal and two
    products; the series below 0.35 less), or of_cap of the cap; a distance and its product 6 of theirs; the sum with the
    distance one of itself, the exponent's argument two of itself and of the reference.  A weight is then off by d, relative, d
    the largest of those of the row's weights that matter, and rounded to `half`; sums as in rows64.attention."""
    nq, heads, dim = q.shape
    nk, group = k.shape[0], heads // k.shape[1]
    place = (np.arange(nq) + nk - nq)[:, None]
    j = np.arange(nk)
    seen = (j <= place) | (j < prefix) if causal else np.ones((nq, nk), bool)
    if q_xyz is None:
        far = np.abs(place - j).astype(np.float64)
    else:
        off = q_xyz[:, None, 1:].astype(np.float64) - k_xyz[None, :, 1:]
        far = np.sqrt((off * off).sum(2))
    y, tol = np.zeros((nq, heads, dim)), np.zeros((nq, heads, dim))
    for h in range(heads):
        qq, kk, vv = q[:, h], k[:, h // group], v[:, h // group]
        z = scale * (qq @ kk.T)
        err = abs(scale) * 8 * np.sqrt(dim) * E * np.sqrt((qq * qq) @ (kk * kk).T) + 2 * E * np.abs(z)
        if cap:
            z = cap * np.tanh(z / cap)
            err = err + 16 * E * np.abs(z) + of_cap * cap
        if slopes is not None:
            d = slopes[h] * far
            z = z - d
            err = err + 6 * E * np.abs(d) + E * np.abs(z)
        z = np.where(seen, z, -np.inf)
        top = z.max(1, keepdims=True)
        top = np.where(np.isfinite(top), top, 0.0)
        p = np.exp(z - top)
        total = p.sum(1, keepdims=True)
        p = p / np.where(total > 0, total, 1)
        y[:, h] = p @ vv
        matters = p > 2.0 ** -40
        err = err + 2 * E * (np.abs(np.where(seen, z, 0)) + np.abs(top) + 1)
        d = np.max(np.where(matters, err, 0), 1, keepdims=True)
        most = (d + half) * (p @ np.abs(vv))
        rms = np.sqrt((p * p) @ (vv * vv))
        tol[:, h] = np.minimum(most, 8 * (d + half) * rms + d * np.abs(y[:, h])) + \
            8 * np.sqrt(nk) * E * (rms + np.abs(y[:, h])) + 4 * E * np.abs(y[:, h]) + 2.0 ** -30 * np.abs(vv).max()
    return y, tol
