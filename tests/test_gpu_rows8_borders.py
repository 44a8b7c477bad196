"""Norms to 8-bit rows where the norm lies beside a border between two codes: the codes are those of the exact value."""
import numpy as np
import pytest

import rows64 as ref
import sparse_hip as sh

pytestmark = pytest.mark.gpu


def beside_borders(s, eps):
    """gamma for rows s [n][c]: channel i's norm in row i % n lands on the fp32 multiplier whose product is next to a border
    between codes, one step below, at or above (in turn)."""
    n, c = s.shape
    y = s / np.sqrt(np.mean(s * s, 1, keepdims=True) + eps)
    e = np.repeat(ref.block_exponent(y), 32, 1)[:, :c]
    i = np.arange(c)
    v, scale = y[i % n, i], 2.0 ** e[i % n, i]
    u = np.abs(v) / scale
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(u, 2.0 ** -20))), -6) - 3)
    border = (np.floor(u / step) + 0.5) * step
    g = np.where(u > 0, border / np.maximum(u, 1e-9), 1.0).astype(np.float32)
    away = np.array([-np.inf, 0, np.inf], np.float32)[i // n % 3]
    return np.where(away == 0, g, np.nextafter(g, away)).astype(np.float32)


def plain(s, g, eps):
    """The norm in fp32 with its usual roundings (the sum is exact here)."""
    f = np.float32
    inv = f(1) / np.sqrt((np.sum(s * s, 1, keepdims=True).astype(f) / f(s.shape[1]) + f(eps)).astype(f))
    return ((s.astype(f) * inv).astype(f) * g).astype(f).astype(np.float64)


def check_codes(dtype, x, r, eps, least):
    """The norm of x + r to 8-bit rows, gamma beside borders: the float64 norm's codes, which fp32's roundings miss at `least`
    places or more."""
    n, c = x.shape
    s = x.astype(np.float64) + r
    g = beside_borders(s, float(np.float32(eps)))
    exp = ref.rows8(ref.rms_norm(s, g.astype(np.float64), float(np.float32(eps))))
    be = sh.Backend(0, dtype)
    try:
        q, y, t = be.alloc_rows8(n, c), be.alloc(n * c), be.alloc(n * c)
        be.rms_norm(be.upload(x), g, q, n, c, eps, residual=be.upload(r), total=t)
        be.expand_rows8(q, y, n, c)
        got = be.download(y).reshape(n, c).astype(np.float64)
        assert np.array_equal(got, sh.storage_round(exp.astype(np.float32), dtype))
        assert np.array_equal(be.download(t).reshape(n, c), sh.storage_round(s.astype(np.float32), dtype))
        assert (ref.rows8(plain(s, g, eps)) != exp).sum() > least
    finally:
        be.destroy()


WIDTHS = [64, 128, 256, 512, 1000, 1024, 2048, 4096, 1001, 4100]


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("c", WIDTHS)
def test_norms_beside_borders(dtype, c):
    """Rows of small whole numbers, whose squares' sums are exact, so that the norm in two floats is right to 2^-45 and the
    border at least some 2^-36 away: every code is that of the float64 norm (no tolerance), where a norm with fp32's
    roundings gives the code on the other side at many of these places."""
    rng, n = np.random.default_rng(c), 21
    x, r = (rng.integers(-8, 9, (n, c)).astype(np.float32) for _ in range(2))
    s = x.astype(np.float64) + r
    s[:, 0] += s[:, 0] == 0
    x[:, 0] = s[:, 0] - r[:, 0]
    check_codes(dtype, x, r, 1e-6, c / 10)


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("c", WIDTHS + [330])
def test_norms_beside_borders_of_many_digits(dtype, c):
    """Rows whose sums x + r are exact (multiples of 2^-8, 2^-10, 2^-12) but whose squares, or their sums, have more digits
    than fp32: those of the norm are exact too."""
    rng, n = np.random.default_rng(c + 1), 21
    step = {sh.BF16: 2.0 ** -8, sh.F16: 2.0 ** -10, sh.F32: 2.0 ** -12}[dtype]
    x, r = (sh.storage_round((np.rint(rng.standard_normal((n, c)) / step) * step).astype(np.float32), dtype)
            for _ in range(2))
    check_codes(dtype, x, r, 1e-6, c / 20)
