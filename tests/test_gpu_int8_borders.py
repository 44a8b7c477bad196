"""Codes of integer rows beside the borders between two of them, where an estimate in fp32 may fall on the wrong side: rows, and
norms of sums that fp32 does not hold, with codes near 127 most of all."""
import numpy as np
import pytest

import sparse_hip as sh

pytestmark = pytest.mark.gpu


def codes_of(be, rows, n, c, scale):
    y = be.alloc(n * c)
    be.expand_rows8(rows, y, n, c)
    return np.rint(be.download(y).reshape(n, c).astype(np.float64) / scale)


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("c", [128, 512, 2048])
def test_norms_of_sums(seed, c):
    """fp32 rows and residuals of like size: their sum has up to 30 bits, its product with a gamma of 23 is exact in float64.
    Each value is placed at a border k + 1/2 of its row, k up to 126, within 6e-5 of a code."""
    be, rng, n = sh.Backend(0, sh.F32), np.random.default_rng(seed), 400
    try:
        g = (1 + rng.random(c)).astype(np.float32)
        r = (0.25 * rng.uniform(-1, 1, (n, c))).astype(np.float32)
        top = (1 + rng.random(n)).astype(np.float32).astype(np.float64)
        k = np.where(rng.random((n, c)) < 0.7, rng.integers(120, 127, (n, c)), rng.integers(0, 127, (n, c)))
        want = (k + 0.5 + rng.choice([0.0, 1e-8, 1e-6, 1e-5, 4e-5, 6e-5], (n, c)) * rng.choice([-1, 1], (n, c)))
        t = want / 127 * top[:, None] * rng.choice([-1, 1], (n, c))
        t[:, 0] = top
        x = (t / g - r).astype(np.float32)
        gamma = g.astype(np.float64)
        v = (x.astype(np.float64) + r) * gamma
        most = np.abs(v).max(1, keepdims=True)
        codes = np.rint(127 * v / most)
        gap = np.abs(127 * v / most - codes)
        assert (gap > 0.4999).mean() > 0.5 and (gap > 0.4999999).sum() > 100
        sure = gap < 0.5 - 1e-12  # (where float64's own rounding cannot turn it)
        rows = be.alloc_rows_int8(n, c)
        be.rms_norm(be.upload(x), g, rows, n, c, 1e-5, residual=be.upload(r))
        s = x.astype(np.float64) + r
        scale = most / np.sqrt((s * s).mean(1, keepdims=True) + float(np.float32(1e-5))) / 127
        got = codes_of(be, rows, n, c, scale)
        assert np.array_equal(got[sure], codes[sure])
    finally:
        be.destroy()


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("c", [128, 512, 1000, 2048])
def test_rows_as_they_are(dtype, c):
    """127 v against k times the largest, both exact in float64, and halves to the even code."""
    be, rng, n = sh.Backend(0, dtype), np.random.default_rng(c), 400
    try:
        top = sh.storage_round((1 + rng.random((n, 1))).astype(np.float32), dtype).astype(np.float64)
        x = sh.storage_round(((rng.integers(-127, 127, (n, c)) + 0.5) / 127 * top).astype(np.float32), dtype)
        x[:, :1] = top
        v = x.astype(np.float64)
        k = np.floor(127 * v / top)
        rest = 2 * (127 * v - k * top)
        codes = k + np.where(rest > top, 1, np.where(rest == top, np.abs(k) % 2, 0))
        rows = be.alloc_rows_int8(n, c)
        be.pack_rows8(be.upload(x), rows, n, c)
        assert np.array_equal(codes_of(be, rows, n, c, top / 127), codes)
    finally:
        be.destroy()


@pytest.mark.parametrize("dtype", [sh.F16, sh.BF16])
def test_sums_are_the_same_at_every_width(dtype):
    """x + residual of 16-bit rows where fp32 has no such number: a width that is a whole number of chunks and one that is not
    (a zero more) give the same codes, those of the sum in fp32."""
    be, rng, n, c = sh.Backend(0, dtype), np.random.default_rng(1), 50, 1000
    try:
        x = (rng.integers(-63, 63, (n, c)) + 0.5).astype(np.float32)
        x[:, 0] = 127
        r = (2.0 ** -20 * rng.choice([-1, 1], (n, c))).astype(np.float32)
        r[:, 0] = 0
        codes = np.rint(x + r)  # (where |x| is 16 or more the sum is x, half way between two codes)
        assert (np.rint(x.astype(np.float64) + r) != codes).mean() > 0.2
        for wide in (0, 1):
            m = c + wide
            xs, rs = (np.concatenate([a, np.zeros((n, wide), np.float32)], 1) for a in (x, r))
            rows = be.alloc_rows_int8(n, m)
            be.rms_norm(be.upload(xs), None, rows, n, m, 1e-5, residual=be.upload(rs))
            got = codes_of(be, rows, n, m, 1 / np.sqrt((xs.astype(np.float64) ** 2).mean(1, keepdims=True) + 1e-5))
            np.testing.assert_array_equal(got[:, :c], codes)
    finally:
        be.destroy()
