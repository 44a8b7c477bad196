"""The row operators of transformer blocks over voxel rows (RMS norm, 8-bit rows, linear with activation and residual,
rotary positions) against float64, at one row and odd widths, at both sides of the kernels' row blocks, with every output
that may be an input.  Bounds: tests/rows64.py."""
import ctypes
import math

import numpy as np
import pytest

import rows64 as ref
import sparse_hip as sh

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in DTYPES}
    yield bes
    for b in bes.values():
        b.destroy()


def make(rng, dtype, *shape):
    return sh.storage_round(rng.standard_normal(shape).astype(np.float32), dtype)


def refused(status, call, *args, **more):
    with pytest.raises(sh.HipError) as e:
        call(*args, **more)
    assert e.value.status == status, e.value


# ---- RMS norm -----------------------------------------------------------------------------------------------------

NORM_SHAPES = [(1, 1), (1, 1024), (3, 7), (5, 64), (257, 100), (130, 128), (33, 256), (1000, 512), (70, 1000), (9, 2048),
               (5, 4096), (3, 4100), (2, 5001), (2500, 64)]


@pytest.mark.parametrize("n,c", NORM_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm(backends, dtype, n, c):
    be, rng = backends[dtype], np.random.default_rng(n * c)
    x, r = make(rng, dtype, n, c), make(rng, dtype, n, c)
    g = (1 + 0.1 * rng.standard_normal(c)).astype(np.float32)
    s = x.astype(np.float64) + r
    for residual, gamma in ((True, g), (False, None)):
        xb, rb, yb, tb = be.upload(x), be.upload(r), be.alloc(n * c), be.alloc(n * c)
        be.rms_norm(xb, gamma, yb, n, c, 1e-6, residual=rb if residual else None, total=tb if residual else None)
        v = s if residual else x.astype(np.float64)
        exp = ref.rms_norm(v, gamma, 1e-6)
        ref.check(be.download(yb).reshape(n, c), exp, ref.rms_slack(c) * np.abs(exp) + ref.stored(exp, dtype), "y")
        if residual:
            ref.check(be.download(tb).reshape(n, c), v, 2 * ref.E * np.abs(v) + ref.stored(v, dtype), "total")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [64, 300, 1000, 4100])
def test_rms_norm_in_place(backends, dtype, c):
    """total over the residual and y over x; then total over x and y over the residual: as with buffers of their own."""
    be, rng, n = backends[dtype], np.random.default_rng(c), 19
    x, r = make(rng, dtype, n, c), make(rng, dtype, n, c)
    g = (1 + 0.1 * rng.standard_normal(c)).astype(np.float32)
    out = []
    for case in range(3):
        xb, rb = be.upload(x), be.upload(r)
        yb, tb = ((be.alloc(n * c), be.alloc(n * c)), (xb, rb), (rb, xb))[case]
        be.rms_norm(xb, g, yb, n, c, 1e-6, residual=rb, total=tb)
        out.append((be.download(yb), be.download(tb)))
    for y, t in out[1:]:
        assert np.array_equal(y, out[0][0]) and np.array_equal(t, out[0][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm_special_rows(backends, dtype):
    """A row of zeros gives zeros, a row with a NaN NaNs, a row with an infinity NaN there and zeros elsewhere; their
    neighbours are untouched."""
    be, n, c = backends[dtype], 5, 128
    x = np.ones((n, c), np.float32)
    x[1], x[2, 3], x[3, 5] = 0, np.nan, np.inf
    xb, yb = be.upload(x), be.alloc(n * c)
    be.rms_norm(xb, None, yb, n, c, 1e-6)
    y = be.download(yb).reshape(n, c)
    assert np.all(np.abs(y[[0, 4]] - 1) <= 2.0 ** -8) and not y[1].any() and np.isnan(y[2]).all()
    assert np.isnan(y[3, 5]) and not np.delete(y[3], 5).any()


# ---- 8-bit rows ---------------------------------------------------------------------------------------------------


def expand(be, rows8, n, c):
    y = be.alloc(n * c)
    be.expand_rows8(rows8, y, n, c)
    return be.download(y).reshape(n, c).astype(np.float64)


@pytest.mark.parametrize("n,c", [(1, 1), (1, 32), (3, 33), (7, 100), (65, 128), (300, 512), (5, 1000), (4, 4100), (2, 8200)])
@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_pack_rows8(backends, dtype, n, c):
    """Values over many powers of two, codes and scales exactly as defined (no tolerance; F16 could not hold all of
    them).  Zero blocks, and maxima at the border where the scale moves on."""
    be, rng = backends[dtype], np.random.default_rng(n + c)
    x = make(rng, dtype, n, c) * np.exp2(rng.integers(-20, 20, (n, 1))).astype(np.float32)
    x[n // 2, :32] = 0
    x[0, 0] = 448.0
    x[-1, -1] = 450.0 if dtype == sh.BF16 else np.nextafter(np.float32(448), np.float32(500))
    q = be.alloc_rows8(n, c)
    be.pack_rows8(be.upload(x), q, n, c)
    assert np.array_equal(expand(be, q, n, c), ref.rows8(x.astype(np.float64)))


def test_pack_rows8_all_codes(backends):
    """Every e4m3 value and the midpoints between neighbours (to even), 448 in each block so that the scale is 1."""
    be = backends[sh.F32]
    codes = np.concatenate([np.arange(8) * 2.0 ** -9] + [2.0 ** e * (1 + np.arange(8) / 8) for e in range(-6, 9)])[:-1]
    assert codes[-1] == 448
    v = np.concatenate([codes, (codes[1:] + codes[:-1]) / 2])
    v = np.concatenate([v, -v]).astype(np.float32)
    v = np.concatenate([v, np.zeros(-len(v) % 31, np.float32)]).reshape(-1, 31)
    x = np.concatenate([v, np.full((len(v), 1), 448, np.float32)], 1)
    q = be.alloc_rows8(len(x), 32)
    be.pack_rows8(be.upload(x), q, len(x), 32)
    assert np.array_equal(expand(be, q, len(x), 32), ref.rows8(x.astype(np.float64)))


def test_pack_rows8_extremes(backends):
    """The largest and the smallest magnitudes, and blocks with an infinity or a NaN, which become NaN as a whole."""
    be = backends[sh.F32]
    x = np.zeros((6, 64), np.float32)
    x[0], x[1, 40], x[2, 0], x[2, 1] = np.finfo(np.float32).max, 2.0 ** -149, 2.0 ** -118, 2.0 ** -130
    x[3, 7], x[4, 33], x[5, :] = np.inf, np.nan, -2.0 ** -126
    q = be.alloc_rows8(6, 64)
    be.pack_rows8(be.upload(x), q, 6, 64)
    y = expand(be, q, 6, 64)
    # fp32's largest, (2 - 2^-23) 2^127, is 255.99... at its scale 2^120, of which e4m3 makes 256: 2^128, which the rows hold
    # and fp32 does not, so that it is an infinity when read back.
    exp = ref.rows8(x.astype(np.float64))
    assert np.all(exp[0] == 2.0 ** 128)
    exp[0] = np.inf
    assert np.isnan(y[3, :32]).all() and not y[3, 32:].any() and np.isnan(y[4, 32:]).all() and not y[4, :32].any()
    assert np.array_equal(y[[0, 1, 2, 5]], exp[[0, 1, 2, 5]])


@pytest.mark.parametrize("n,c", [(1, 64), (3, 7), (65, 300), (130, 1024), (4, 4100)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm_to_rows8(backends, dtype, n, c):
    be, rng = backends[dtype], np.random.default_rng(n * c)
    x, r = make(rng, dtype, n, c), make(rng, dtype, n, c)
    g = (1 + 0.1 * rng.standard_normal(c)).astype(np.float32)
    q, tb = be.alloc_rows8(n, c), be.alloc(n * c)
    be.rms_norm(be.upload(x), g, q, n, c, 1e-6, residual=be.upload(r), total=tb)
    s = x.astype(np.float64) + r
    exp = ref.rms_norm(s, g, 1e-6)
    tol = ref.rows8_slack(exp, ref.rms_slack(c) * np.abs(exp))
    got = expand(be, q, n, c)
    ref.check(got, exp, tol + ref.stored(got, dtype), "rows8")
    # All but values at a border are the very codes.
    assert np.mean(got != sh.storage_round(ref.rows8(exp), dtype)) <= 0.001 + 1 / got.size
    ref.check(be.download(tb).reshape(n, c), s, 2 * ref.E * np.abs(s) + ref.stored(s, dtype), "total")


# ---- linear with activation and residual --------------------------------------------------------------------------

LINEAR_SHAPES = [(1, 1, 1), (1, 1024, 4096), (2, 7, 5), (3, 64, 128), (63, 40, 136), (65, 100, 77), (129, 256, 130),
                 (257, 136, 300), (300, 1000, 200), (17, 4096, 64), (1000, 72, 1000), (5003, 512, 256)]


@pytest.mark.parametrize("dtype", [sh.F16, sh.BF16])
@pytest.mark.parametrize("c", [64, 512, 1000, 1024])
def test_rms_norm_to_rows8_codes(backends, dtype, c):
    """Codes are those of the 64-bit norm.  The sum of squares carries 8 squares' fp32 roundings, 3 E of the sum at most, and
    half of it reaches the inverse: 1.5 E, and the two floats' products 2^-45.  A code differs only where a border lies
    between: of 8 borders an octave (uniform values within it) that is 8 x 2 x 1.5 E / ln 2 of the values at most, twice
    for e4m3's coarser steps near zero; 8 standard deviations of that count beside it.  (x + r is exact in fp32 unless one is
    2^13 times the other, which is rarer.)"""
    be, rng, n = backends[dtype], np.random.default_rng(c), 2_000_000 // c
    x, r, g = make(rng, dtype, n, c), make(rng, dtype, n, c), (1 + 0.1 * rng.standard_normal(c)).astype(np.float32)
    q, y = be.alloc_rows8(n, c), be.alloc(n * c)
    be.rms_norm(be.upload(x), g, q, n, c, 1e-6, residual=be.upload(r))
    be.expand_rows8(q, y, n, c)
    exp = ref.rows8(ref.rms_norm(x.astype(np.float64) + r, g.astype(np.float64), 1e-6))
    if dtype == sh.F16:
        exp = exp.astype(np.float16).astype(np.float64)  # the smallest codes are below fp16's normal numbers
    most = n * c * 2 * 8 * 2 * 1.5 * ref.E / math.log(2)
    assert (be.download(y).reshape(n, c) != exp).sum() <= most + 8 * math.sqrt(most)


def linear_case(be, dtype, n, ci, co, act, bias, residual, from8=False):
    rng = np.random.default_rng(n + 3 * ci + 7 * co)
    x, r = make(rng, dtype, n, ci), make(rng, dtype, n, co)
    w = (rng.standard_normal((co, ci)) / math.sqrt(ci)).astype(np.float32)
    b = (0.5 * rng.standard_normal(co)).astype(np.float32)
    xb, yb = be.upload(x), be.alloc(n * co)
    if from8:
        q = be.alloc_rows8(n, ci)
        be.pack_rows8(xb, q, n, ci)
        xb = q
        xv, wv = ref.rows8(x.astype(np.float64)), ref.rows8(w.astype(np.float64))
    else:
        xv, wv = x.astype(np.float64), sh.storage_round(w, dtype).astype(np.float64)
    be.linear_act(xb, w, b if bias else None, yb, n, ci, co, act=act, residual=be.upload(r) if residual else None)
    got = be.download(yb).reshape(n, co)
    rows = np.unique(np.concatenate([np.arange(min(n, 150)), np.arange(max(0, n - 150), n), rng.integers(0, n, 200)]))
    exp, err = ref.linear_act(xv[rows], wv, b.astype(np.float64) if bias else None, act,
                              r[rows].astype(np.float64) if residual else None, from8)
    ref.check(got[rows], exp, err + ref.stored(exp, dtype), f"linear {n} {ci} {co} {act}")


@pytest.mark.parametrize("n,ci,co", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act(backends, dtype, n, ci, co):
    act = list(sh.ACTS)[(n + ci + co) % 4]
    linear_case(backends[dtype], dtype, n, ci, co, act, True, (n + ci) % 2 == 0)


@pytest.mark.parametrize("n,ci,co", LINEAR_SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_from_rows8(backends, dtype, n, ci, co):
    act = list(sh.ACTS)[(n + ci + co + 1) % 4]
    linear_case(backends[dtype], dtype, n, ci, co, act, True, (n + co) % 2 == 0, from8=True)


@pytest.mark.parametrize("act", list(sh.ACTS))
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_epilogues(backends, dtype, act, bias, residual):
    linear_case(backends[dtype], dtype, 70, 128, 136, act, bias, residual)


@pytest.mark.parametrize("from8", [False, True])
@pytest.mark.parametrize("dtype,n,ci,co", [(sh.BF16, 33000, 256, 512), (sh.F16, 66001, 136, 256), (sh.F32, 20000, 64, 512),
                                           (sh.BF16, 20000, 200, 200), (sh.F16, 5003, 1024, 1032)])
def test_linear_act_large_blocks(backends, dtype, n, ci, co, from8):
    linear_case(backends[dtype], dtype, n, ci, co, "gelu", True, True, from8=from8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_residual_in_place(backends, dtype):
    be, rng, n, c = backends[dtype], np.random.default_rng(5), 300, 136
    x, r, w = make(rng, dtype, n, c), make(rng, dtype, n, c), make(rng, dtype, c, c) / 16
    xb, rb, yb = be.upload(x), be.upload(r), be.alloc(n * c)
    be.linear_act(xb, w, None, yb, n, c, c, act="silu", residual=rb)
    be.linear_act(xb, w, None, rb, n, c, c, act="silu", residual=rb)
    assert np.array_equal(be.download(yb), be.download(rb))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("from8", [False, True])
@pytest.mark.parametrize("ci", [40, 100])
def test_linear_act_rows_stay_apart(backends, dtype, from8, ci):
    """NaN and infinities in one row (what follows a short row's end in memory is the next row) reach that row alone."""
    be, rng, n, co = backends[dtype], np.random.default_rng(ci), 40, 24
    x, w = make(rng, dtype, n, ci), make(rng, dtype, co, ci)
    out = []
    for special in (False, True):
        if special:
            x[7], x[21, 0] = np.nan, np.inf
        xb, yb = be.upload(x), be.alloc(n * co)
        if from8:
            q = be.alloc_rows8(n, ci)
            be.pack_rows8(xb, q, n, ci)
            xb = q
        be.linear_act(xb, w, None, yb, n, ci, co)
        out.append(be.download(yb).reshape(n, co))
    others = np.delete(np.arange(n), [7, 21])
    assert np.array_equal(out[0][others], out[1][others]) and np.isfinite(out[0]).all()
    assert np.isnan(out[1][7]).all() and not np.isfinite(out[1][21]).any()


@pytest.mark.parametrize("act", list(sh.ACTS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations_far_out(backends, dtype, act):
    """Identity weights: the activation itself from -60000 to 60000, with the bounds of linear_act."""
    be = backends[dtype]
    z = sh.storage_round(np.concatenate([np.linspace(-12, 12, 4001), np.linspace(-6e4, 6e4, 95)]).astype(np.float32), dtype)
    n, c = z.size // 16, 16
    x = z.reshape(n, c)
    xb, yb = be.upload(x), be.alloc(n * c)
    be.linear_act(xb, np.eye(c, dtype=np.float32), None, yb, n, c, c, act=act)
    exp, err = ref.linear_act(x.astype(np.float64), np.eye(c), None, act, None)
    ref.check(be.download(yb).reshape(n, c), exp, err + ref.stored(exp, dtype), act)


# ---- rotary positions ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dim,pairs", [(8, (1, 1, 1)), (16, (2, 3, 3)), (40, (6, 6, 6)), (48, (8, 8, 8)), (64, (10, 10, 10)),
                                       (64, (0, 32, 0)), (96, (16, 16, 16)), (128, (21, 21, 22)), (256, (40, 40, 48)),
                                       (24, (0, 0, 0))])
@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary(backends, dtype, dim, pairs, split, norm):
    rng = np.random.default_rng(dim + sum(pairs))
    n, heads = int(rng.integers(1, 70)), int(rng.integers(1, 40 if dim < 100 else 9))
    be = backends[dtype]
    x = make(rng, dtype, n, heads, dim)
    coords = rng.integers(-70000, 70000, (n, 4)).astype(np.int32)
    g = (1 + 0.1 * rng.standard_normal((heads, dim))).astype(np.float32) if norm else None
    xb, yb = be.upload(x), be.alloc(n * heads * dim)
    be.rotary(xb, be.upload_i32(coords), yb, n, heads, dim, pairs, split=split, gamma=g, eps=1e-6 if norm else None)
    exp, err = ref.rotary(x.astype(np.float64), coords, pairs, 10000.0, split, g, 1e-6 if norm else None)
    ref.check(be.download(yb).reshape(n, heads, dim), exp, err + ref.stored(exp, dtype), "rotary")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_strides_and_in_place(backends, dtype):
    """q and k columns of a qkv buffer into a buffer of their own, in place, and into the v columns: the same values, and
    nothing else is written."""
    be, rng = backends[dtype], np.random.default_rng(2)
    n, heads, dim = 37, 3, 32
    w = heads * dim
    qkv = make(rng, dtype, n, 3 * w)
    coords = rng.integers(0, 64, (n, 4)).astype(np.int32)
    dm = be.upload_coords(coords)
    for many, off in ((2 * heads, 0), (heads, w)):
        exp, err = ref.rotary(qkv[:, off:off + many * dim].reshape(n, many, dim).astype(np.float64), coords, (5, 5, 5), 100.0,
                              False)
        exp, err = exp.reshape(n, -1), err.reshape(n, -1)
        tol = err + ref.stored(exp, dtype)
        xb, yb = be.upload(qkv), be.upload(np.full((n, many * dim + 8), 7, np.float32))
        be.rotary(xb, dm, yb, n - 1, many, dim, (5, 5, 5), base=100.0, x_offset=off, x_stride=3 * w, y_offset=8,
                  y_stride=many * dim + 8)
        y = be.download(yb).reshape(n, -1)
        ref.check(y[:-1, 8:], exp[:-1], tol[:-1], "apart")
        assert np.all(y[:, :8] == 7) and np.all(y[-1] == 7)
        be.rotary(xb, dm, xb, n, many, dim, (5, 5, 5), base=100.0, x_offset=off, x_stride=3 * w, y_offset=off, y_stride=3 * w)
        y = be.download(xb).reshape(n, -1)
        ref.check(y[:, off:off + many * dim], exp, tol, "in place")
        assert np.array_equal(np.delete(y, np.s_[off:off + many * dim], 1), np.delete(qkv, np.s_[off:off + many * dim], 1))
    xb = be.upload(qkv)
    be.rotary(xb, dm, xb, n, heads, dim, (5, 5, 5), base=100.0, x_offset=w, x_stride=3 * w, y_offset=2 * w, y_stride=3 * w)
    y = be.download(xb).reshape(n, -1)
    ref.check(y[:, 2 * w:], exp, tol, "other columns")
    assert np.array_equal(y[:, :2 * w], qkv[:, :2 * w])
    be.free_map(dm)


# ---- refusals -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_refusals(backends, dtype):
    be, bad = backends[dtype], sh.INVALID_ARGUMENT
    x, y, i32 = be.alloc(64 * 64), be.alloc(64 * 64), be.upload_i32(np.zeros(4 * 64, np.int32))
    q, w = be.alloc_rows8(64, 64), np.zeros((64, 64), np.float32)
    for n, c in ((0, 64), (-1, 64), (64, 0), (1 << 62, 1 << 20)):
        refused(bad, be.rms_norm, x, None, y, n, c, 1e-6)
        refused(bad, be.linear_act, x, w, None, y, n, 64, c)
        refused(bad, be.pack_rows8, x, q, n, c)
        refused(bad, be.expand_rows8, q, y, n, c)
        refused(bad, be.alloc_rows8, n, c)
    refused(bad, be.rms_norm, x, None, y, 64, 65, 1e-6)          # more than the buffers hold
    refused(bad, be.rms_norm, x, None, y, 64, 64, 0.0)
    refused(bad, be.rms_norm, x, None, y, 64, 64, float("nan"))
    refused(bad, be.rms_norm, i32, None, y, 1, 64, 1e-6)         # not rows of the storage type
    refused(bad, be.rms_norm, q, None, y, 64, 64, 1e-6)          # 8-bit rows as input
    refused(bad, be.rms_norm, x, None, q, 32, 64, 1e-6)          # 8-bit rows of another shape
    refused(bad, be.rms_norm, x, None, y, 64, 64, 1e-6, total=y)  # both outputs in one place
    refused(bad, be.pack_rows8, q, q, 64, 64)
    refused(bad, be.linear_act, q, w, None, y, 64, 32, 64)       # 8-bit rows of another width
    refused(bad, be.linear_act, x, w, None, x, 64, 64, 64)       # y over x
    refused(bad, be.linear_act, x, w, None, y, 64, 1 << 21, 64)
    st = sh.LIB.trellis_sparse_hip_linear_act(be.ptr, x.handle, w.ctypes.data, None, 4, None, y.handle, 64, 64, 64)
    assert st == bad
    st = sh.LIB.trellis_sparse_hip_linear_act(be.ptr, x.handle, None, None, 0, None, y.handle, 64, 64, 64)
    assert st == bad

    def rot(**more):
        args = dict(n=64, heads=2, head_dim=32, pairs=(5, 5, 5))
        args.update({k: more.pop(k) for k in list(more) if k in args})
        be.rotary(more.pop("x", x), more.pop("coords", i32), more.pop("y", y), *args.values(), **more)

    rot()
    refused(bad, rot, n=65)
    refused(bad, rot, n=0)
    refused(bad, rot, heads=0)
    refused(bad, rot, head_dim=264)
    refused(bad, rot, pairs=(6, 6, 6))
    refused(bad, rot, pairs=(-1, 5, 5))
    refused(bad, rot, pairs=(2147483647, 2147483647, 2147483647))
    refused(bad, rot, base=0.0)
    refused(bad, rot, eps=-1.0)
    refused(bad, rot, gamma=np.ones(64, np.float32))             # gamma without a norm
    refused(bad, rot, x_stride=32)
    refused(bad, rot, x_offset=8)
    refused(bad, rot, x_offset=-8)
    refused(bad, rot, coords=x)
    refused(bad, rot, coords=be.upload_i32(np.zeros(4 * 63, np.int32)))
    refused(bad, rot, n=32, y=x, y_offset=8, y_stride=64)        # half over x
    refused(bad, rot, x=q)
    refused(sh.NOT_IMPLEMENTED, rot, n=8, head_dim=20, pairs=(3, 3, 3))
    refused(sh.NOT_IMPLEMENTED, rot, n=8, x_stride=68)
    st = sh.LIB.trellis_sparse_hip_rotary(be.ptr, x.handle, i32.handle, None, y.handle, 64, ctypes.byref(sh.RotaryDesc()))
    assert st == bad
    # The slots do not take 8-bit rows.
    refused(bad, be.add, q, x, y, 64)
    refused(bad, be.silu_inplace, q, 64)
    refused(bad, be.linear, q, w, None, y, 64, 64, 64)
    refused(bad, be.download, q)
    refused(bad, be.download_raw, q)


def test_out_of_memory(backends):
    be = sh.Backend(0, sh.BF16)
    try:
        x, y, w = be.alloc(64 * 64), be.alloc(64 * 64), np.zeros((64, 64), np.float32)
        for call in ((be.alloc_rows8, 4096, 4096), (be.linear_act, x, w, None, y, 64, 64, 64)):
            be.fail_alloc(0)
            try:
                refused(sh.OUT_OF_MEMORY, *call)
            finally:
                be.fail_alloc(-1)
        be.linear_act(x, w, None, y, 64, 64, 64)
    finally:
        be.destroy()
