"""The row operators of transformer blocks in float64 (numpy), from their definitions, with bounds on what fp32
arithmetic and one rounding may add: the oracle of test_gpu_rows.py and test_gpu_attention.py."""
import numpy as np

import sparse_hip as sh

E = 2.0 ** -24  # half a step of fp32, relative
HALF = {sh.F32: E, sh.F16: 2.0 ** -11, sh.BF16: 2.0 ** -8}  # half a step of the storage type, relative
TINY = {sh.F32: 2.0 ** -149, sh.F16: 2.0 ** -25, sh.BF16: 2.0 ** -133}  # half a step of its subnormals


def check(got, exp, tol, what=""):
    """|got - exp| <= tol element by element; NaN where the oracle has NaN."""
    got, exp = np.asarray(got, np.float64), np.asarray(exp, np.float64)
    assert got.shape == exp.shape
    bad = ~(np.abs(got - exp) <= tol) & ~(np.isnan(got) & np.isnan(exp)) & ~((got == exp) & np.isinf(exp))
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(np.abs(got - exp), nan=np.inf), -1)), got.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} off; at {at} got {got[at]!r}, expected {exp[at]!r} "
                             f"+- {np.broadcast_to(tol, got.shape)[at]!r}")


def stored(exp, dtype):
    """What the one rounding to the storage type may add."""
    return HALF[dtype] * np.abs(exp) + TINY[dtype]


def rms_norm(s, gamma, eps):
    y = s / np.sqrt(np.mean(s * s, -1, keepdims=True) + eps)
    return y if gamma is None else y * gamma


def rms_slack(c):
    """fp32 error of a norm, relative.  The sum of squares (positive terms) passes at most c / 64 + 64 additions in a lane
    and 6 across lanes, one rounding each; the root halves it; square, mean, eps, root, reciprocal, the sum x + residual
    and two products add at most 10 more."""
    return ((c / 64 + 70) / 2 + 10) * E


def block_exponent(v):
    """Per 32 channels (the last block may be short) the least e >= -126 with max|v| <= 448 * 2^e; 0 for zeros; NaN where
    the block is not finite.  Shape [n][blocks]."""
    n, c = v.shape
    b = np.zeros((n, -(-c // 32) * 32))
    b[:, :c] = np.abs(v)
    most = b.reshape(n, -1, 32).max(2)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.ceil(np.log2(most / 448))
    e = np.where(most == 0, 0, np.maximum(e, -126))
    return np.where(np.isfinite(most), e, np.nan)


def rows8(v):
    """The values that 8-bit rows hold of v, v fp32 values in float64."""
    e = np.repeat(block_exponent(v), 32, 1)[:, :v.shape[1]]
    with np.errstate(divide="ignore", invalid="ignore"):
        u = v / 2.0 ** e
        power = np.maximum(np.floor(np.log2(np.maximum(np.abs(u), 2.0 ** -30))), -6)
    step = 2.0 ** (power - 3)
    return np.rint(u / step) * step * 2.0 ** e


def rows8_slack(v, err):
    """How far codes of values within err of v may be from v: half a step of e4m3 (2^-4 relative, or half of 2^-9 scales),
    the scale one power of two higher where err carries the maximum over a border."""
    e = np.repeat(block_exponent(v), 32, 1)[:, :v.shape[1]] + 1
    return err + np.maximum(2.0 ** -4 * (np.abs(v) + err), 2.0 ** -10 * 2.0 ** e)


def activate(z, act):
    if act == "silu":
        with np.errstate(over="ignore"):
            return z / (1 + np.exp(-z))
    if act == "gelu":
        from scipy.special import erf
        return 0.5 * z * (1 + erf(z / np.sqrt(2)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    return z


def linear_act(x, w, b, act, r, from8=False):
    """(value, bound on the fp32 error).  A sum of K products takes K roundings, each within E of a partial sum; partial
    sums stay within some root-sum-square of the products, and roundings are as often up as down: 8 standard deviations of
    that walk, 8 sqrt(K) E.  Activations have slopes up to 1.13, and their own error is 2^-19 |z| (fp32 outputs: 2^-21): erf
    1.5e-7 = 2^-22.7, an exponential and a reciprocal 2^-21 each, the exponential's argument (up to 20 before the result
    drops below 1e-8 of z) 20 E.  From 8-bit rows the matrix unit cuts each product at 2^-13 of the largest of its eight
    neighbours in K (towards zero, so as often up as down; measured with single products, largest * 2^-13 stays and
    largest * 2^-14 goes): up to 7 cuts below 2^-13 M a group, M at most the group's largest |x| times its largest |w|,
    or 8 standard deviations of their sum, each uniform: 8 / sqrt(3) 2^-13 sqrt(7 sum M^2)."""
    z = x @ w.T + (0 if b is None else b)
    walk = np.sqrt((x * x) @ (w * w).T + (0 if b is None else b * b))
    err = 8 * np.sqrt(x.shape[1]) * E * walk + 2 * E * np.abs(z)
    if from8:
        top = lambda a: np.pad(np.abs(a), ((0, 0), (0, -a.shape[1] % 8))).reshape(a.shape[0], -1, 8).max(2)  # noqa: E731
        mx, mw = top(x), top(w)
        err = err + 2.0 ** -13 * np.minimum(7 * (mx @ mw.T), 8 / np.sqrt(3) * np.sqrt(7 * ((mx * mx) @ (mw * mw).T)))
    err = 1.2 * err
    if act != "none":
        err = err + 2.0 ** -19 * np.abs(z)
    y = activate(z, act)
    if r is not None:
        y = y + r
        err = err + E * np.abs(y)
    return y, err


def rotary(x, coords, pairs, base, split, gamma=None, eps=None):
    """x [n][heads][dim] -> (value, bound).  Angles in turns are off by half a step of [1/4, 1/2), 2^-26, or 1.6 E in radians;
    sine and cosine by two steps of 1 (2 E each); products and their sum 3 E: 8 E of |a| + |b|."""
    n, heads, dim = x.shape
    slack = 0.0
    if eps is not None:
        x = rms_norm(x, gamma, eps)
        slack = rms_slack(dim)
    j = np.concatenate([np.arange(p) / p for p in pairs if p]) if sum(pairs) else np.zeros(0)
    axis = np.repeat([1, 2, 3], pairs)
    angle = coords[:, axis].astype(np.float64) * base ** -j
    full = np.zeros((n, dim // 2))
    full[:, :angle.shape[1]] = angle
    c, s = np.cos(full)[:, None], np.sin(full)[:, None]
    if split:
        a, b = x[..., :dim // 2], x[..., dim // 2:]
    else:
        a, b = x[..., 0::2], x[..., 1::2]
    ya, yb = a * c - b * s, a * s + b * c
    e = (8 * E + slack) * (np.abs(a) + np.abs(b))
    if split:
        return np.concatenate([ya, yb], 2), np.concatenate([e, e], 2)
    return np.stack([ya, yb], 3).reshape(n, heads, dim), np.stack([e, e], 3).reshape(n, heads, dim)


def attention(q, k, v, scale, group, q_at, k_at, half_p):
    """q [nq][heads][dim], k, v [nk][kv_heads][dim], offsets -> (value, bound, rows in a sequence).  With weights p: scores
    are sums of dim products (a walk of 8 sqrt(dim) E as in linear_act), which with the rounding of the exponent's argument
    scale a weight by 1 + d, d the natural exponent's error; a weight is rounded to half_p (half a step, relative; E for
    fp32) before it meets v.  Those errors differ from key to key: at most (d + half_p) sum p |v|, and 8 standard deviations,
    8 (d + half_p) sqrt(sum p^2 v^2); sums over nk keys add a walk of 8 sqrt(nk) E of the latter and of the sum of weights."""
    nq, heads, dim = q.shape
    y, tol = np.zeros((nq, heads, dim)), np.zeros((nq, heads, dim))
    inside = np.zeros(nq, bool)
    for s in range(len(q_at) - 1):
        qs, ks = slice(q_at[s], q_at[s + 1]), slice(k_at[s], k_at[s + 1])
        inside[qs] = True
        nk = k_at[s + 1] - k_at[s]
        if nk == 0 or q_at[s + 1] == q_at[s]:
            continue
        for h in range(heads):
            kk, vv, qq = k[ks, h // group], v[ks, h // group], q[qs, h]
            z = scale * (qq @ kk.T)
            m = z.max(1, keepdims=True)
            p = np.exp(z - m)
            p /= p.sum(1, keepdims=True)
            y[qs, h] = p @ vv
            walk = abs(scale) * 8 * np.sqrt(dim) * E * np.sqrt((qq * qq) @ (kk * kk).T)
            d = np.max(walk + 4 * E * (np.abs(z) + np.abs(m)) + 4 * E, 1, keepdims=True)
            most = (d + half_p) * (p @ np.abs(vv))
            rms = np.sqrt((p * p) @ (vv * vv))
            tol[qs, h] = np.minimum(most, 8 * (d + half_p) * rms + d * np.abs(y[qs, h])) + \
                8 * np.sqrt(nk) * E * (rms + np.abs(y[qs, h])) + 4 * E * np.abs(y[qs, h])
    return y, tol, inside
