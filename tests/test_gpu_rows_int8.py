"""8-bit integer rows against float64: codes to the last one (halves too), scales, norms, products with their exact sums, every
block shape, refusals."""
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


def expanded(be, rows, n, c):
    y = be.alloc(n * c)
    be.expand_rows8(rows, y, n, c)
    return be.download(y).reshape(n, c)


def check_rows(be, dtype, rows, v, what, norm=1.0):
    """The values of `rows` are codes of v (float64, times norm a row); a code beside the right one is off by 1 / 127 of the
    largest, which the rounding of a value with the type (2^-8 of it at most) does not hide."""
    codes, scales = more.int8_rows(v)
    exp = codes * scales * norm
    ref.check(expanded(be, rows, *v.shape), exp, 4 * ref.E * np.abs(exp) + ref.stored(exp, dtype), what)
    return codes


WIDTHS = [1, 7, 8, 31, 64, 100, 128, 129, 256, 300, 512, 1000, 1024, 2048, 2052, 4096, 4100, 5001]


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_pack(backends, dtype, c):
    be, rng = backends[dtype], np.random.default_rng(c)
    for n in (1, 3, 130):
        x = sh.storage_round((rng.standard_normal((n, c)) * np.exp(3 * rng.standard_normal((n, 1)))).astype(np.float32), dtype)
        rows = be.alloc_rows_int8(n, c)
        be.pack_rows8(be.upload(x), rows, n, c)
        check_rows(be, dtype, rows, x.astype(np.float64), f"pack {n} {c}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_halves_go_to_even(backends, dtype):
    """Values half way between two codes, of which 16-bit rows have many: half of the largest value is 63.5 codes."""
    be, rng = backends[dtype], np.random.default_rng(1)
    n, c = 400, 128
    top = sh.storage_round((1 + rng.random((n, 1))).astype(np.float32) * 2.0 ** rng.integers(-8, 8, (n, 1)), dtype)
    top[:100] = 127.0 * 2.0 ** rng.integers(-7, 7, (100, 1))  # halves of every code
    x = top * sh.storage_round((rng.integers(-254, 255, (n, c)) / 254).astype(np.float32), dtype)
    x[100:] = top[100:] * rng.choice([-0.5, 0.5, 0.25, 1.0], (n - 100, c))
    x[:100] = top[:100] / 127 * rng.integers(-254, 255, (100, c)) / 2
    x[:, 0] = top[:, 0]
    x = sh.storage_round(x.astype(np.float32), dtype)
    rows = be.alloc_rows_int8(n, c)
    be.pack_rows8(be.upload(x), rows, n, c)
    v = x.astype(np.float64)
    codes = check_rows(be, dtype, rows, v, "halves")
    half = 127 * v / np.abs(v).max(1, keepdims=True)
    assert (np.abs(half - np.floor(half) - 0.5) < 1e-12).sum() > 5000
    assert np.all(codes[half == 63.5] == 64) and np.all(codes[half == 0.5] == 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_rows(backends, dtype):
    """Zeros stay zeros, a row with an infinity or a NaN becomes NaN and no other does; the ends of the type's range."""
    be, n, c = backends[dtype], 9, 72
    rng = np.random.default_rng(2)
    x = rng.standard_normal((n, c)).astype(np.float32)
    x[1] = 0
    x[2, 5], x[3, 71], x[4, 0] = np.nan, np.inf, -np.inf
    big, small = {sh.F32: (3.4e38, 1e-30), sh.F16: (65504.0, 6e-8), sh.BF16: (3.3e38, 1e-30)}[dtype]
    x[5, :] = rng.choice([-big, big, big / 2, 0], c)
    x[6, :] = rng.choice([-small, small, 0], c)
    x = sh.storage_round(x, dtype)
    rows = be.alloc_rows_int8(n, c)
    be.pack_rows8(be.upload(x), rows, n, c)
    got = expanded(be, rows, n, c)
    assert np.isnan(got[2:5]).all() and np.all(got[1] == 0)
    rest = [0, 5, 6, 7, 8]
    codes, scales = more.int8_rows(x[rest].astype(np.float64))
    exp = codes * scales
    ref.check(got[rest], exp, 4 * ref.E * np.abs(exp) + ref.stored(exp, dtype), "special")


@pytest.mark.parametrize("c", [1, 40, 128, 300, 512, 1024, 2048, 4096, 5001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm(backends, dtype, c):
    be, rng, eps = backends[dtype], np.random.default_rng(c), 1e-5
    for n in (1, 77):
        x, r = (sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype) for _ in range(2))
        g = (1 + 0.3 * rng.standard_normal(c)).astype(np.float32)
        for residual, gamma in ((None, None), (r, g)):
            rows, total = be.alloc_rows_int8(n, c), be.alloc(n * c)
            be.rms_norm(be.upload(x), gamma, rows, n, c, eps, residual=None if residual is None else be.upload(residual),
                        total=total)
            s = x.astype(np.float64) + (0 if residual is None else residual.astype(np.float64))
            norm = 1 / np.sqrt((s * s).mean(1, keepdims=True) + float(np.float32(eps)))
            check_rows(be, dtype, rows, s * (1 if gamma is None else gamma.astype(np.float64)), f"norm {n} {c}", norm)
            ref.check(be.download(total).reshape(n, c), s, ref.E * np.abs(s) + ref.stored(s, dtype), "total")


@pytest.mark.parametrize("c", [64, 512, 1000, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_at_the_ends_of_the_range(backends, dtype, c):
    """Values whose squares, or whose products with gamma, leave fp32; rows of zeros, of infinities and of NaN beside them,
    gammas of every size; a gamma that is not finite makes every row NaN."""
    be, rng = backends[dtype], np.random.default_rng(c)
    big, small = {sh.F32: (1e37, 1e-37), sh.F16: (6e4, 1e-7), sh.BF16: (1e37, 1e-37)}[dtype]
    size = np.array([1.0, big, big / 1e3, small, small * 10, 0.0, 1.0, 1.0, 1.0])
    n = len(size)
    x = sh.storage_round((np.clip(rng.standard_normal((n, c)), -3, 3) * size[:, None]).astype(np.float32), dtype)
    x[6, 3], x[7, c - 1] = np.inf, np.nan
    for eps, gamma in ((1e-5, None), (1e-5, np.exp(8 * rng.standard_normal(c)).astype(np.float32)),
                       (1e-30, np.full(c, 1e6, np.float32))):
        rows = be.alloc_rows_int8(n, c)
        be.rms_norm(be.upload(x), gamma, rows, n, c, eps)
        s = x.astype(np.float64)
        fine = np.isfinite(s).all(1)
        with np.errstate(invalid="ignore"):
            norm = 1 / np.sqrt((s * s).mean(1, keepdims=True) + float(np.float32(eps)))
            codes, scales = more.int8_rows(s * (1 if gamma is None else gamma.astype(np.float64)))
            exp = codes * scales * norm
        got = expanded(be, rows, n, c)
        assert np.isnan(got[~fine]).all()
        # What the type cannot hold is an infinity; scales below fp32's normal numbers have fewer digits.
        exp, got = exp[fine], got[fine]
        held = np.abs(exp) < {sh.F32: 3e38, sh.F16: 65000.0, sh.BF16: 3e38}[dtype]
        tol = 4 * ref.E * np.abs(exp) + ref.stored(exp, dtype) + 128 * 2.0 ** -149
        ref.check(np.where(held, got, 0), np.where(held, exp, 0), tol, f"ends {c} {eps}")
    for bad in (np.nan, np.inf):
        g = np.ones(c, np.float32)
        g[c // 2] = bad
        rows = be.alloc_rows_int8(n, c)
        be.rms_norm(be.upload(np.ones((n, c), np.float32)), g, rows, n, c, 1e-5)
        assert np.isnan(expanded(be, rows, n, c)).all()


@pytest.mark.parametrize("c", [64, 512, 1024])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_of_a_row_does_not_see_its_neighbours(backends, dtype, c):
    """Ordinary rows among rows at the ends of the range, infinite, NaN and zero: each as if normed alone, to the last bit."""
    be, rng = backends[dtype], np.random.default_rng(c + 1)
    big, small = {sh.F32: (1e37, 1e-37), sh.F16: (6e4, 1e-7), sh.BF16: (1e37, 1e-37)}[dtype]
    size = rng.permutation(np.repeat(np.array([1.0, 1.0, 1.0, big, small, 0.0, 1.0, 1.0]), 5))
    n = len(size)
    x = np.clip(rng.standard_normal((n, c)), -0.9, 0.9) * size[:, None]
    ones = np.flatnonzero(size == 1.0)
    x[ones[3], 5], x[ones[9], c - 1] = np.inf, np.nan
    x = sh.storage_round(x.astype(np.float32), dtype)
    gamma = np.exp(rng.standard_normal(c)).astype(np.float32)
    rows, one = be.alloc_rows_int8(n, c), be.alloc_rows_int8(1, c)
    be.rms_norm(be.upload(x), gamma, rows, n, c, 1e-5)
    got = expanded(be, rows, n, c)
    for i in range(n):
        be.rms_norm(be.upload(x[i:i + 1]), gamma, one, 1, c, 1e-5)
        assert np.array_equal(got[i:i + 1], expanded(be, one, 1, c), equal_nan=True), (i, size[i])


def run_linear(be, dtype, n, ci, co, act, bias, residual, seed=0, norm=False):
    rng = np.random.default_rng(seed + n + 3 * ci + 5 * co)
    x = sh.storage_round((rng.standard_normal((n, ci)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32), dtype)
    w = (rng.standard_normal((co, ci)) / np.sqrt(ci)).astype(np.float32)
    b = rng.standard_normal(co).astype(np.float32) if bias else None
    r = sh.storage_round(rng.standard_normal((n, co)).astype(np.float32), dtype) if residual else None
    rows, y = be.alloc_rows_int8(n, ci), be.alloc(n * co)
    be.pack_rows8(be.upload(x), rows, n, ci)
    be.linear_act(rows, w, b, y, n, ci, co, act=act, residual=None if r is None else be.upload(r))
    d = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    exp, err = more.int8_linear(*more.int8_rows(d(x)), d(w), d(b), act, d(r), dtype == sh.F32)
    ref.check(be.download(y).reshape(n, co), exp, err + ref.stored(exp, dtype), f"linear {n} {ci} {co} {act}")


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 33, 64, 65, 129, 257, 300, 1000])
@pytest.mark.parametrize("ci,co", [(64, 64), (128, 256), (300, 77), (1024, 512), (40, 1000), (4096, 66)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear(backends, dtype, n, ci, co):
    run_linear(backends[dtype], dtype, n, ci, co, ["none", "silu", "gelu", "gelu_tanh"][n % 4], n % 3 > 0, n % 2 == 0)


@pytest.mark.parametrize("ci,co", [(1, 1), (1, 300), (5, 3), (127, 1), (129, 255), (2000, 257), (70, 4), (5001, 34)])
@pytest.mark.parametrize("n", [1, 70])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_odd(backends, dtype, n, ci, co):
    run_linear(backends[dtype], dtype, n, ci, co, "silu", True, True)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_large(backends, dtype, act):
    """Several tiles a block, and parts of the rows in blocks of other shapes."""
    run_linear(backends[dtype], dtype, 9001, 256, 768, act, True, False)
    run_linear(backends[dtype], dtype, 6000, 1024, 514, act, False, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_long_sums(backends, dtype):
    """All codes 127: sums of 2^31 nearly, exact.  (Scales are whole: a row's largest value is 127.)"""
    be, ci, co = backends[dtype], 131072, 3
    for n in (1, 70):
        x = np.full((n, ci), 127, np.float32)
        w = np.full((co, ci), 127, np.float32)
        w[1, ::2] = -127
        rows, y = be.alloc_rows_int8(n, ci), be.alloc(n * co)
        be.pack_rows8(be.upload(x), rows, n, ci)
        b = np.array([-2114060288.0, 5.0, 0.0], np.float32)  # 127 * 127 * 131,072
        be.linear_act(rows, w, b, y, n, ci, co)
        got = be.download(y).reshape(n, co)
        exp = sh.storage_round(np.array([0.0, 5.0, 2114060288.0 if dtype != sh.F16 else np.inf], np.float32), dtype)
        np.testing.assert_array_equal(got, np.tile(exp, (n, 1)))


@pytest.mark.parametrize("n", [1, 40, 500])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_special(backends, dtype, n):
    """A NaN row gives NaNs in its own outputs alone, a weight that is not finite in its channel's."""
    be, ci, co = backends[dtype], 200, 96
    rng = np.random.default_rng(n)
    x = sh.storage_round(rng.standard_normal((n, ci)).astype(np.float32), dtype)
    w = rng.standard_normal((co, ci)).astype(np.float32)
    w[7, 3] = np.inf
    x[n // 2, 9] = np.nan
    rows, y = be.alloc_rows_int8(n, ci), be.alloc(n * co)
    be.pack_rows8(be.upload(x), rows, n, ci)
    be.linear_act(rows, w, None, y, n, ci, co)
    got = be.download(y).reshape(n, co)
    hit = np.zeros((n, co), bool)
    hit[n // 2], hit[:, 7] = True, True
    assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_into_its_residual(backends, dtype):
    be, n, ci, co = backends[dtype], 333, 128, 64
    rng = np.random.default_rng(5)
    x = be.upload(rng.standard_normal((n, ci)).astype(np.float32))
    w, r = rng.standard_normal((co, ci)).astype(np.float32), rng.standard_normal((n, co)).astype(np.float32)
    rows, y, z = be.alloc_rows_int8(n, ci), be.alloc(n * co), be.upload(r)
    be.pack_rows8(x, rows, n, ci)
    be.linear_act(rows, w, None, y, n, ci, co, residual=z)
    be.linear_act(rows, w, None, z, n, ci, co, residual=z)
    np.testing.assert_array_equal(be.download_raw(y), be.download_raw(z))


@pytest.mark.parametrize("n", [1, 6, 200])
def test_linear_repeats_and_rows_do_not_depend_on_others(backends, n):
    """Whole-number sums are the same in any order: a row's outputs are, bit for bit, those of the row alone."""
    be, ci, co = backends[sh.BF16], 1000, 130
    rng = np.random.default_rng(n)
    x = rng.standard_normal((n, ci)).astype(np.float32)
    w, b = rng.standard_normal((co, ci)).astype(np.float32), rng.standard_normal(co).astype(np.float32)

    def run(v):
        m = len(v)
        rows, y = be.alloc_rows_int8(m, ci), be.alloc(m * co)
        be.pack_rows8(be.upload(v), rows, m, ci)
        be.linear_act(rows, w, b, y, m, ci, co, act="silu")
        return be.download_raw(y).reshape(m, co)

    all_rows = run(x)
    for i in range(0, n, 37):
        np.testing.assert_array_equal(run(x[i:i + 1])[0], all_rows[i])


def test_refusals(backends):
    be, n, c = backends[sh.BF16], 64, 64
    x, y, rows = be.alloc(n * c), be.alloc(n * c), be.alloc_rows_int8(n, c)
    w = np.zeros((c, c), np.float32)

    def refuse(call, *a, **kw):
        with pytest.raises(sh.HipError) as e:
            call(*a, **kw)
        assert e.value.status == sh.INVALID_ARGUMENT

    refuse(be.alloc_rows_int8, 0, 4)
    refuse(be.alloc_rows_int8, 4, 0)
    refuse(be.alloc_rows_int8, 4, 2 ** 31 - 1)
    refuse(be.pack_rows8, x, rows, n, c - 1)
    refuse(be.pack_rows8, x, rows, n - 1, c)
    refuse(be.pack_rows8, rows, rows, n, c)
    refuse(be.expand_rows8, rows, rows, n, c)
    refuse(be.linear_act, rows, w, None, rows, n, c, c)
    refuse(be.linear_act, rows, w, None, y, n, c, c, residual=rows)
    refuse(be.linear_act, rows, w, None, y, n, c // 2, c)
    refuse(be.rms_norm, rows, None, y, n, c, 1e-6)
    refuse(be.rms_norm, x, None, y, n, c, 1e-6, total=rows)
    refuse(be.set_scratch, rows)
    refuse(be.download, rows)
    wide = be.alloc_rows_int8(1, 131073)
    refuse(be.linear_act, wide, np.zeros((1, 131073), np.float32), None, y, 1, 131073, 1)
