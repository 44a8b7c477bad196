"""Attention with capped scores at every size of the cap, and few queries, whose weights are not rounded to 16 bits: bounds that
a score's own size gives (tests/scored_tight64.py)."""
import numpy as np
import pytest

import rows64 as ref
import scored_tight64 as tight
import sparse_hip as sh

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]
QUICK = 512.0  # 16 bits: caps up to this one leave 2^-22 of the cap


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in DTYPES}
    yield bes
    for b in bes.values():
        b.destroy()


def rows(rng, dtype, n, heads, dim, size=1.0):
    return sh.storage_round((size * rng.standard_normal((n, heads, dim))).astype(np.float32), dtype)


def run(be, dtype, nq, nk, heads, kv_heads, dim, cap=0.0, bias=None, causal=False, prefix=0, sharp=2.0, scale=0.0, slope=1.0,
        half=None, grid=64):
    rng = np.random.default_rng(nq + 3 * nk + 5 * dim + heads)
    q, k, v = rows(rng, dtype, nq, heads, dim, sharp), rows(rng, dtype, nk, kv_heads, dim), rows(rng, dtype, nk, kv_heads, dim)
    slopes = None if bias is None else (slope * rng.random(heads)).astype(np.float32)
    kw, xyz = {}, [None, None]
    if bias == "voxels":
        xyz = [rng.integers(0, grid, (n, 4)).astype(np.int32) for n in (nq, nk)]
        kw = {"q_coords": be.upload_i32(xyz[0]), "k_coords": be.upload_i32(xyz[1])}
    if prefix:
        kw["prefix"] = be.upload_i32(np.array([prefix], np.int32))
    y = be.alloc(nq * heads * dim)
    be.attention_scored(be.upload(q), be.upload(k), be.upload(v), y, nq, nk, heads, kv_heads, dim, scale=scale, cap=cap,
                        slopes=slopes, causal=causal, **kw)
    d = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    half = (ref.E if dtype == sh.F32 else ref.HALF[dtype]) if half is None else half
    of_cap = 2.0 ** -22 if dtype != sh.F32 and cap <= QUICK else 0.0
    exp, tol = tight.attention(d(q), d(k), d(v), float(np.float32(scale)) or dim ** -0.5, half, float(np.float32(cap)), d(slopes),
                               *xyz, causal, prefix, of_cap)
    if half < ref.HALF[dtype] and dtype == sh.F16:
        tol = tol + 2.0 ** -31 * nk * np.abs(v).max()
    ref.check(be.download(y).reshape(exp.shape), exp, tol + ref.stored(exp, dtype), f"{nq} {nk} {dim} cap {cap} {bias}")


@pytest.mark.parametrize("cap", [512.0, 513.0, 1e4, 1e5, 1e7, 1e30, 1e37, 1.1e38])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 13, 160])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_caps(backends, dtype, dim, cap):
    """Scores of ordinary size under caps so large that they change nothing."""
    run(backends[dtype], dtype, 300, 333, 1, 1, dim, cap)
    run(backends[dtype], dtype, 3, 1000, 2, 1, dim, cap, causal=True)


@pytest.mark.parametrize("cap", [600.0, 1e6, 1e30, 1.1e38])
@pytest.mark.parametrize("bias", ["rows", "voxels"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_caps_with_distances(backends, dtype, bias, cap):
    for dim in (64, 128, 20):
        run(backends[dtype], dtype, 200, 300, 2, 2, dim, cap, bias, slope=0.1)
        run(backends[dtype], dtype, 2, 700, 2, 2, dim, cap, bias, causal=True, slope=0.01)


@pytest.mark.parametrize("scale", [1.0, -1.0])
@pytest.mark.parametrize("cap", [0.01, 5.0, 50.0, 512.0, 600.0, 5000.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_below_and_beyond_the_cap(backends, dtype, cap, scale):
    """Scores from far below the cap to many times it."""
    for size in (0.01, 0.3, 1.0, 8.0):
        run(backends[dtype], dtype, 150, 200, 2, 2, 64, cap, scale=scale, sharp=float(size * cap / 8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("form", [dict(), dict(bias="rows", causal=True, slope=0.05), dict(bias="voxels", slope=0.1),
                                  dict(causal=True, prefix=30), dict(cap=30.0), dict(cap=1e5)])
@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim", [(1, 300, 2, 2, 64), (3, 20000, 4, 1, 64), (20, 700, 6, 2, 32),
                                                      (64, 64, 3, 3, 96), (500, 900, 2, 2, 128), (1500, 1500, 2, 2, 64)])
def test_few_queries_cost_no_precision(backends, dtype, form, nq, nk, heads, kv_heads, dim):
    """Nothing but fp32's errors and the output's one rounding: weights of 16 bits are in two parts, which leave 2 HALF^2 of
    them, and 2^-31 of the largest where fp16 has no finer steps."""
    half = ref.E if dtype == sh.F32 else 2 * ref.HALF[dtype] ** 2
    run(backends[dtype], dtype, nq, nk, heads, kv_heads, dim, half=half, **form)
