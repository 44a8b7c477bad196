"""Group norm of voxel rows against float64: widths and group sizes that are whole chunks and that are not, one row and many,
uneven and empty sequences, rows in no sequence, means far above the deviations, in place, refusals."""
import ctypes

import numpy as np
import pytest

import rows64 as ref
import scored64 as more
import sparse_hip as sh

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in DTYPES}
    yield bes
    for b in bes.values():
        b.destroy()


def run_case(be, dtype, lengths, c, groups, act="silu", extra=0, affine=True, mean=0.0, spread=1.0, whole=False, inplace=False,
             eps=1e-5, seed=0):
    """Sequences of the given lengths, and `extra` more rows behind the last."""
    rng = np.random.default_rng(seed + sum(lengths) + 3 * c + 7 * groups)
    n = sum(lengths) + extra
    x = (mean * rng.standard_normal((1, c)) + spread * rng.standard_normal((n, c))).astype(np.float32)
    x = sh.storage_round(x, dtype)
    if extra:
        x[-extra:] = np.nan
    g = (1 + 0.2 * rng.standard_normal(c)).astype(np.float32) if affine else None
    b = rng.standard_normal(c).astype(np.float32) if affine else None
    at = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    bx = be.upload(x)
    y = bx if inplace else be.upload(np.full(n * c, 7, np.float32))
    be.group_norm(bx, g, b, y, n, c, groups, eps, act=act, offsets=None if whole else be.upload_i32(at))
    got = be.download(y).reshape(n, c)
    d = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    exp, tol, inside = more.group_norm(d(x), at, d(g), d(b), groups, float(np.float32(eps)), act)
    left = x if inplace else np.full((n, c), 7.0)
    np.testing.assert_array_equal(got[~inside], left[~inside])
    ref.check(got[inside], exp[inside], (tol + ref.stored(exp, dtype))[inside], f"group_norm {lengths} {c}/{groups} {act}")


@pytest.mark.parametrize("c,groups", [(32, 32), (64, 32), (128, 32), (256, 32), (512, 32), (1024, 32), (2048, 16), (300, 10),
                                      (96, 3), (40, 5), (7, 1), (77, 11), (1, 1), (520, 65), (512, 1), (4100, 41),
                                      (24, 24), (100, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_widths(backends, dtype, c, groups):
    run_case(backends[dtype], dtype, [131], c, groups, whole=True)
    run_case(backends[dtype], dtype, [1000, 37], c, groups, act="none")


@pytest.mark.parametrize("lengths", [[1], [2], [3, 0, 1], [0], [0, 0, 5, 0], [63, 64, 65], [127, 1, 129, 0, 255], [1] * 70,
                                     [5000], [20, 9000, 0, 3]])
@pytest.mark.parametrize("c,groups", [(64, 16), (128, 32), (30, 5)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences(backends, dtype, lengths, c, groups):
    """Rows behind the last sequence hold NaN, which reaches nothing, and stay as they were in the output."""
    run_case(backends[dtype], dtype, lengths, c, groups, extra=3)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations(backends, dtype, act):
    run_case(backends[dtype], dtype, [700, 300], 128, 32, act=act)
    run_case(backends[dtype], dtype, [40], 128, 32, act=act, affine=False, inplace=True)


@pytest.mark.parametrize("n", [20, 3000, 60000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_means(backends, dtype, n):
    """Means a thousand and more deviations away (in 16 bits as far as the type can hold the deviations)."""
    far = {sh.F32: 3000.0, sh.F16: 30.0, sh.BF16: 4.0}[dtype]
    be, rng, c, groups = backends[dtype], np.random.default_rng(n), 64, 8
    x = sh.storage_round((far + rng.standard_normal((n, c))).astype(np.float32), dtype)
    y = be.alloc(n * c)
    be.group_norm(be.upload(x), None, None, y, n, c, groups, 1e-5)
    exp, tol, _ = more.group_norm(x.astype(np.float64), [0, n], None, None, groups, float(np.float32(1e-5)), "none")
    ref.check(be.download(y).reshape(n, c), exp, tol + ref.stored(exp, dtype), "large means")


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows(backends, dtype):
    run_case(backends[dtype], dtype, [30011, 0, 20000, 1], 128, 32, extra=5)
    run_case(backends[dtype], dtype, [20011], 300, 10, act="none", inplace=True)


@pytest.mark.parametrize("n", [50, 20000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_values_and_special_ones(backends, dtype, n):
    """Where all values are equal the result is beta; a NaN or an infinity makes its own group of its own sequence NaN."""
    be, c, groups = backends[dtype], 64, 8
    b = np.arange(c, dtype=np.float32) / 64
    x = np.full((n, c), 0.1, np.float32)
    at = be.upload_i32(np.array([0, n // 2, n], np.int32))
    y = be.alloc(n * c)
    be.group_norm(be.upload(x), None, b, y, n, c, groups, 1e-5, offsets=at)
    np.testing.assert_array_equal(be.download(y).reshape(n, c), np.tile(sh.storage_round(b, dtype), (n, 1)))
    rng = np.random.default_rng(1)
    for bad in (np.nan, np.inf, -np.inf):
        x = sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype)
        be.group_norm(be.upload(x), None, b, y, n, c, groups, 1e-5, offsets=at)
        base = be.download(y).reshape(n, c)
        x[n - 3, 17] = bad
        be.group_norm(be.upload(x), None, b, y, n, c, groups, 1e-5, offsets=at)
        got = be.download(y).reshape(n, c)
        hit = np.zeros((n, c), bool)
        hit[n // 2:, 16:24] = True
        assert np.isnan(got[hit]).all()
        np.testing.assert_array_equal(got[~hit], base[~hit])


@pytest.mark.parametrize("dtype", DTYPES)
def test_repeats_its_bits(backends, dtype):
    be, rng, n, c = backends[dtype], np.random.default_rng(2), 40000, 128
    x, y = be.upload(rng.standard_normal((n, c)).astype(np.float32)), be.alloc(n * c)
    first = None
    for _ in range(5):
        be.group_norm(x, None, None, y, n, c, 32, 1e-5, act="silu")
        got = be.download_raw(y)
        first = got if first is None else first
        np.testing.assert_array_equal(got, first)


def test_offsets_outside_the_rows(backends):
    """Offsets are clamped to the rows that there are; falling ones leave their sequence empty."""
    be, n, c = backends[sh.F32], 300, 32
    rng = np.random.default_rng(3)
    x = rng.standard_normal((n, c)).astype(np.float32)
    for at, end in (([0, 1000], n), ([-5, 100], 100), ([200, 100, 150], 150)):
        y = be.upload(np.full(n * c, 7, np.float32))
        be.group_norm(be.upload(x), None, None, y, n, c, 4, 1e-5, offsets=be.upload_i32(np.array(at, np.int32)))
        got = be.download(y).reshape(n, c)
        a = max(0, at[-2])
        exp, tol, _ = more.group_norm(x[a:end].astype(np.float64), [0, end - a], None, None, 4, float(np.float32(1e-5)), "none")
        ref.check(got[a:end], exp, tol + ref.stored(exp, sh.F32), "clamped")
        assert np.all(got[end:] == 7) and np.all(got[:a] == 7)


def test_refusals(backends):
    be, n, c = backends[sh.BF16], 8, 64
    x, y, at = be.alloc(n * c), be.alloc(n * c), be.upload_i32(np.array([0, n], np.int32))
    g = np.ones(c, np.float32)

    def refuse(status=sh.INVALID_ARGUMENT, **kw):
        a = dict(x=x, gamma=g, beta=g, y=y, n=n, c=c, groups=8, eps=1e-5, offsets=at)
        a.update(kw)
        with pytest.raises(sh.HipError) as e:
            be.group_norm(**a)
        assert e.value.status == status

    refuse(groups=7)
    refuse(groups=0)
    refuse(groups=-8)
    refuse(n=0)
    refuse(n=n + 1)
    refuse(c=0)
    refuse(eps=0.0)
    refuse(eps=float("nan"))
    refuse(offsets=x)
    refuse(x=at)
    refuse(y=at)
    refuse(x=be.alloc_rows8(n, c))
    refuse(y=be.alloc_rows_int8(n, c))
    refuse(y=be.alloc(n * c - 1))
    L, one = sh.LIB.trellis_sparse_hip_group_norm, ctypes.c_float(1e-5)
    assert L(be.ptr, x.handle, None, 2, None, None, y.handle, n, c, 8, one, 0) == sh.INVALID_ARGUMENT
    assert L(be.ptr, x.handle, at.handle, 2, None, None, y.handle, n, c, 8, one, 0) == sh.INVALID_ARGUMENT
    assert L(be.ptr, x.handle, at.handle, 0, None, None, y.handle, n, c, 8, one, 0) == sh.INVALID_ARGUMENT
    assert L(be.ptr, x.handle, at.handle, 1, None, None, y.handle, n, c, 8, one, 4) == sh.INVALID_ARGUMENT
    assert L(be.ptr, x.handle, at.handle, 1, None, None, y.handle, n, c, 8, one, -1) == sh.INVALID_ARGUMENT
