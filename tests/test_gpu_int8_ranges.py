"""Integer rows and their linear at the ends of fp32's range, where a product on the way may leave it though the output does
not; a row's outputs are the same bits alone, beside rows of every size, and in every kernel."""
import numpy as np
import pytest

import rows64 as ref
import scored64 as more
import sparse_hip as sh

pytestmark = pytest.mark.gpu
WIDE = [sh.F32, sh.BF16]  # (fp16's largest is 65,504)


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in [sh.F32, sh.F16, sh.BF16]}
    yield bes
    for b in bes.values():
        b.destroy()


def linear(be, x, w, b, act="none", residual=None):
    (n, ci), co = x.shape, w.shape[0]
    rows, y = be.alloc_rows_int8(n, ci), be.alloc(n * co)
    be.pack_rows8(be.upload(x), rows, n, ci)
    be.linear_act(rows, w, b, y, n, ci, co, act=act, residual=None if residual is None else be.upload(residual))
    return be.download(y).reshape(n, co)


@pytest.mark.parametrize("n", [1, 2, 4, 5, 40, 300, 3000])
@pytest.mark.parametrize("ci,co", [(64, 64), (1024, 128), (300, 77), (2048, 256)])
@pytest.mark.parametrize("dtype", WIDE)
def test_large_rows_and_small_weights(backends, dtype, n, ci, co):
    """Rows from 1e-30 to 1e38 through weights whose outputs stay within the range: sums of 1e6 codes times a scale of 1e34 do
    not.  Some channels' weights are so large that their outputs of large rows are infinite, of zeros zero."""
    be, rng = backends[dtype], np.random.default_rng(n + ci)
    size = 10.0 ** rng.choice([-30, -3, 0, 20, 28, 30, 35, 37], (n, 1))
    x = np.clip(rng.standard_normal((n, ci)), -3, 3) * size
    if n > 4:
        x[3] = 0
    x = sh.storage_round(x.astype(np.float32), dtype)
    w = (np.abs(rng.standard_normal((co, ci))) * 1e-4 / ci).astype(np.float32)
    w[::2] *= -1
    w[5] = 0
    b = rng.standard_normal(co).astype(np.float32)
    exp, tol = more.int8_linear(*more.int8_rows(x.astype(np.float64)), w.astype(np.float64), b.astype(np.float64), "none", None,
                                dtype == sh.F32)
    got = linear(be, x, w, b)
    assert np.abs(exp).max() < 1e35
    ref.check(got, exp, tol + ref.stored(exp, dtype), f"{n} {ci} {co}")
    for i in range(0, n, max(1, n // 7)):
        np.testing.assert_array_equal(linear(be, x[i:i + 1], w, b)[0], got[i])


@pytest.mark.parametrize("n", [3, 200])
@pytest.mark.parametrize("dtype", WIDE)
def test_both_scales_large(backends, dtype, n):
    """Rows and weights at 1e36: outputs are infinite, but where the sum is zero."""
    be, ci, co = backends[dtype], 128, 32
    x = np.full((n, ci), 1e36, np.float32)
    x[:, ::2] *= -1
    w = np.full((co, ci), 1e36, np.float32)
    w[1::2, ::2] *= -1
    got = linear(be, x, w, np.ones(co, np.float32))
    assert np.all(got[:, ::2] == 1) and np.all(got[:, 1::2] == np.inf)
    w = w.copy()  # (weights are known by their address)
    w[3, 3] = np.nan
    got = linear(be, x, w, None)
    assert np.isnan(got[:, 3]).all() and np.all(got[:, ::2] == 0)


@pytest.mark.parametrize("dtype", WIDE)
def test_large_rows_in_many_tiles(backends, dtype):
    """Blocks of every width, activations and residuals among ordinary rows and large ones."""
    be, rng = backends[dtype], np.random.default_rng(3)
    for n, ci, co, act in ((9001, 256, 768, "gelu"), (6000, 1024, 514, "none")):
        x = rng.standard_normal((n, ci)) * np.where(rng.random((n, 1)) < 0.3, 1e34, 1.0)
        x = sh.storage_round(x.astype(np.float32), dtype)
        w = (rng.standard_normal((co, ci)) * 1e-3).astype(np.float32)
        r = sh.storage_round(rng.standard_normal((n, co)).astype(np.float32), dtype)
        d = lambda a: a.astype(np.float64)  # noqa: E731
        exp, tol = more.int8_linear(*more.int8_rows(d(x)), d(w), None, act, d(r), dtype == sh.F32)
        ref.check(linear(be, x, w, None, act, r), exp, tol + ref.stored(exp, dtype), f"{n} {ci} {co} {act}")


@pytest.mark.parametrize("c", [64, 300, 512, 1000, 1024])
@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
def test_norms_with_tiny_gammas(backends, dtype, c):
    """Products of values and gammas below fp32's range, whose norms are not; gammas of zero, and rows of zeros among others."""
    be, rng, n = backends[dtype], np.random.default_rng(c), 33
    size = rng.choice({sh.F32: [1e-30, 1e-14, 1e-3, 1.0, 0.0], sh.F16: [2e-6, 1e-3, 1.0, 0.0],
                       sh.BF16: [1e-30, 1e-14, 1e-3, 1.0, 0.0]}[dtype], (n, 1))
    x = sh.storage_round((np.clip(rng.standard_normal((n, c)), -3, 3) * size).astype(np.float32), dtype)
    for eps, g in ((1e-30, 1e-32), (1e-38, 1e-30), (1e-5, 1e-37), (1e-12, 1e-36), (1e-5, 0.0)):
        gamma = (g * np.exp(rng.standard_normal(c))).astype(np.float32)
        rows, y = be.alloc_rows_int8(n, c), be.alloc(n * c)
        be.rms_norm(be.upload(x), gamma, rows, n, c, eps)
        be.expand_rows8(rows, y, n, c)
        s = x.astype(np.float64)
        codes, scales = more.int8_rows(s * gamma.astype(np.float64))
        exp = codes * scales / np.sqrt((s * s).mean(1, keepdims=True) + float(np.float32(eps)))
        # (A scale below fp32's normal numbers is off by up to half of 2^-149, a value by 127 times that.)
        ref.check(be.download(y).reshape(n, c), exp, 4 * ref.E * np.abs(exp) + ref.stored(exp, dtype) + 128 * 2.0 ** -149,
                  f"{c} {eps} {g}")
