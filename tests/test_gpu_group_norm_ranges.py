"""Group norm of values at the ends of fp32's range, whose differences from the mean or inverse deviations fp32 does not hold as
they are, and of ordinary groups beside them."""
import numpy as np
import pytest

import rows64 as ref
import scored64 as more
import sparse_hip as sh

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in [sh.F32, sh.F16, sh.BF16]}
    yield bes
    for b in bes.values():
        b.destroy()


@pytest.mark.parametrize("n", [3, 40, 20000])
@pytest.mark.parametrize("c,groups", [(64, 8), (70, 7), (128, 32), (24, 24)])
@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
def test_ends_of_the_range(backends, dtype, n, c, groups):
    """Groups of deviations from 1e-37 to 3e38, some with a mean as large; gammas of 1e-3 and of 1.  fp32 has no steps below
    2^-149: the mean's lower part is rounded to half a step of that, and so are the two differences, which is up to
    3 x 2^-150 of x - m and reaches the output times gamma over the deviation."""
    be, rng = backends[dtype], np.random.default_rng(n + c)
    top = {sh.F32: 3.4e38, sh.F16: 65000.0, sh.BF16: 3.38e38}[dtype]
    size = c // groups
    x = rng.uniform(-1, 1, (n, c))
    spread = np.resize([top, 1.0, top / 2.0, 1e-3 * top, 1e-37 if dtype != sh.F16 else 1e-6, 1e-20, 0.3 * top], groups)
    mean = np.resize([0, 5.0, top / 2.0, 0, 0, 0, -0.7 * top], groups)
    x = sh.storage_round(np.clip(x * np.repeat(spread, size) + np.repeat(mean, size), -top, top).astype(np.float32), dtype)
    for g, eps in ((None, 1e-5), (np.full(c, 1e-3, np.float32), 1e-5), (None, 1e-38)):
        y = be.alloc(n * c)
        be.group_norm(be.upload(x), g, None, y, n, c, groups, eps)
        exp, tol, _ = more.group_norm(x.astype(np.float64), [0, n], None if g is None else g.astype(np.float64), None, groups,
                                      float(np.float32(eps)), "none")
        v = x.reshape(n, groups, size).astype(np.float64)
        root = np.sqrt(((v - v.mean((0, 2), keepdims=True)) ** 2).mean((0, 2)) + float(np.float32(eps)))
        tol = tol + 2.0 ** -148 * np.repeat(1 / root, size) * (1.0 if g is None else 1e-3)
        assert np.abs(exp).max() < 1e6 and np.isfinite(exp).all()
        ref.check(be.download(y).reshape(n, c), exp, tol + ref.stored(exp, dtype), f"{n} {c}/{groups} {eps}")


@pytest.mark.parametrize("n", [40, 20000])
@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_equal_values_at_the_end_of_the_range(backends, dtype, n):
    """Their mean is that value, and the result beta, whatever eps."""
    be, c = backends[dtype], 64
    b = np.arange(c, dtype=np.float32)
    x = np.full((n, c), 3e38 if dtype == sh.F32 else 2.0 ** 127, np.float32)
    for eps in (1e-5, 1e-45):
        y = be.alloc(n * c)
        be.group_norm(be.upload(x), None, b, y, n, c, 8, eps)
        np.testing.assert_array_equal(be.download(y).reshape(n, c), np.tile(sh.storage_round(b, dtype), (n, 1)))
