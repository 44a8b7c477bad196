"""Attention within sequences of voxel rows against float64: one query and many, one key and many, at both sides of the
kernels' tiles, empty sequences, rows in no sequence, grouped heads, strides.  Bounds: tests/rows64.py."""
import ctypes

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


def offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def run_case(be, dtype, q_len, k_len, heads, kv_heads, dim, scale=0.0, seed=0, whole=False, extra=0, sharp=1.0):
    """Sequences of the given lengths; `extra` more rows behind the last of q and of k."""
    rng = np.random.default_rng(seed + sum(q_len) + 3 * sum(k_len) + 5 * dim)
    nq, nk = sum(q_len) + extra, sum(k_len) + extra
    q = sh.storage_round((sharp * rng.standard_normal((nq, heads, dim))).astype(np.float32), dtype)
    k = sh.storage_round(rng.standard_normal((nk, kv_heads, dim)).astype(np.float32), dtype)
    v = sh.storage_round(rng.standard_normal((nk, kv_heads, dim)).astype(np.float32), dtype)
    if extra:
        k[-extra:], v[-extra:] = np.nan, np.inf
    y = be.upload(np.full(nq * heads * dim, 7, np.float32))
    qa, ka = offsets(q_len), offsets(k_len)
    at = {} if whole else {"q_offsets": be.upload_i32(qa), "kv_offsets": be.upload_i32(ka)}
    be.attention(be.upload(q), be.upload(k) if nk else None, be.upload(v) if nk else None, y, nq, nk, heads, kv_heads, dim,
                 scale=scale, **at)
    got = be.download(y).reshape(nq, heads, dim)
    exp, err, inside = ref.attention(q.astype(np.float64), k.astype(np.float64), v.astype(np.float64),
                                     scale or dim ** -0.5, heads // kv_heads, qa, ka, ref.HALF[dtype])
    assert inside.sum() == sum(q_len) and np.all(got[~inside] == 7)
    ref.check(got[inside], exp[inside], (err + ref.stored(exp, dtype))[inside],
              f"attention {q_len} {k_len} {heads}/{kv_heads} {dim}")


@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 96, 128, 13, 160, 192])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_widths(backends, dtype, dim):
    run_case(backends[dtype], dtype, [70], [131], 2, 2, dim, whole=True)


@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (33, 64), (64, 65), (127, 129), (128, 63),
                                   (129, 128), (257, 200), (1, 4097), (3, 700), (40, 5000), (1000, 17)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths(backends, dtype, nq, nk, dim):
    run_case(backends[dtype], dtype, [nq], [nk], 3, 3, dim, whole=(nq + nk) % 2 == 0)


@pytest.mark.parametrize("q_len,k_len", [([5, 0, 130, 1], [5, 0, 130, 1]), ([3, 64, 2], [0, 200, 0]), ([0, 0, 9], [4, 4, 4]),
                                         ([1] * 70, [3, 0] * 35), ([1, 1, 1, 1], [1000, 0, 65, 2500]), ([0], [3]),
                                         ([40] * 9, [0] * 9), ([2] * 130, [7] * 130)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences(backends, dtype, q_len, k_len):
    """Uneven and empty sequences, more of them than a wavefront has lanes; rows behind the last sequence hold NaN and
    infinities as keys and values, which reach nothing, and stay as they were in the output."""
    run_case(backends[dtype], dtype, q_len, k_len, 2, 2, 64, extra=3)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (6, 2), (16, 4), (17, 17), (40, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_heads(backends, dtype, heads, kv_heads):
    run_case(backends[dtype], dtype, [3, 50], [90, 33], heads, kv_heads, 64)
    run_case(backends[dtype], dtype, [1, 1], [900, 333], heads, kv_heads, 32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,sharp", [(0.01, 1.0), (1.0, 1.0), (0.125, 40.0), (-0.2, 1.0)])
def test_scales(backends, dtype, scale, sharp):
    """Nearly even weights, and nearly one-hot ones whose running maximum moves far from tile to tile."""
    run_case(backends[dtype], dtype, [100], [700], 2, 2, 64, scale=scale, sharp=sharp, whole=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rising_scores(backends, dtype):
    """Keys in ascending order of their score: every tile raises the maximum; and in descending order."""
    be, rng, n, dim = backends[dtype], np.random.default_rng(4), 600, 64
    q = sh.storage_round(np.ones((33, 1, dim), np.float32), dtype)
    for order in (1, -1):
        k = sh.storage_round(np.repeat(np.linspace(-4, 4, n)[::order, None, None], dim, 2).astype(np.float32), dtype)
        v = sh.storage_round(rng.standard_normal((n, 1, dim)).astype(np.float32), dtype)
        y = be.alloc(33 * dim)
        be.attention(be.upload(q), be.upload(k), be.upload(v), y, 33, n, 1, 1, dim, scale=1.0)
        exp, err, _ = ref.attention(q.astype(np.float64), k.astype(np.float64), v.astype(np.float64), 1.0, 1, [0, 33], [0, n],
                                    ref.HALF[dtype])
        ref.check(be.download(y).reshape(33, 1, dim), exp, err + ref.stored(exp, dtype), "rising")


@pytest.mark.parametrize("dtype", DTYPES)
def test_special_values(backends, dtype):
    """A NaN query gives NaNs in its own row and head alone; a key whose scores are all -inf has no weight; where all are,
    the row is zero; an infinity among the values shows where its weight is not zero."""
    be, n, dim = backends[dtype], 70, 64
    rng = np.random.default_rng(6)
    q = sh.storage_round(np.abs(rng.standard_normal((n, 2, dim))).astype(np.float32), dtype)
    k = sh.storage_round(rng.standard_normal((n, 2, dim)).astype(np.float32), dtype)
    v = sh.storage_round(rng.standard_normal((n, 2, dim)).astype(np.float32), dtype)

    def run(q, k, v):
        y = be.alloc(n * 2 * dim)
        be.attention(be.upload(q), be.upload(k), be.upload(v), y, n, n, 2, 2, dim)
        return be.download(y).reshape(n, 2, dim)

    base = run(q, k, v)
    q2 = q.copy()
    q2[5, 1, 3] = np.nan
    got = run(q2, k, v)
    assert np.isnan(got[5, 1]).all()
    got[5, 1] = base[5, 1]
    assert np.array_equal(got, base)
    k2 = k.copy()
    k2[9, 0] = -np.inf
    got = run(q, k2, v)
    kept = np.delete(np.arange(n), 9)
    exp, err, _ = ref.attention(q.astype(np.float64), k[kept].astype(np.float64), v[kept].astype(np.float64), dim ** -0.5, 1,
                                [0, n], [0, n - 1], ref.HALF[dtype])
    ref.check(got[:, 0], exp[:, 0], (err + ref.stored(exp, dtype))[:, 0], "a key of no weight")
    assert np.array_equal(got[:, 1], base[:, 1])
    assert not run(q, np.full_like(k, -np.inf), v).any()
    v2 = v.copy()
    v2[11, 0, 7] = np.inf
    got = run(q, k, v2)
    assert np.all(got[:, 0, 7] == np.inf)
    got[:, 0, 7] = base[:, 0, 7]
    assert np.array_equal(got, base)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 20])
def test_strides_and_query_in_place(backends, dtype, dim):
    """q, k and v as columns of one buffer, y as columns of another, and over the q columns: the same values, nothing else
    written."""
    be, rng, n, heads = backends[dtype], np.random.default_rng(dim), 150, 3
    w = heads * dim
    qkv = sh.storage_round(rng.standard_normal((n, 3 * w)).astype(np.float32), dtype)
    q, k, v = (qkv[:, i * w:(i + 1) * w].reshape(n, heads, dim).astype(np.float64) for i in range(3))
    exp, err, _ = ref.attention(q, k, v, dim ** -0.5, 1, [0, n], [0, n], ref.HALF[dtype])
    exp = exp.reshape(n, w)
    tol = err.reshape(n, w) + ref.stored(exp, dtype)
    b, y = be.upload(qkv), be.upload(np.full((n, 2 * w), 7, np.float32))
    at = dict(q_stride=3 * w, k_offset=w, k_stride=3 * w, v_offset=2 * w, v_stride=3 * w)
    be.attention(b, b, b, y, n, n, heads, heads, dim, y_offset=w, y_stride=2 * w, **at)
    got = be.download(y).reshape(n, 2 * w)
    assert np.all(got[:, :w] == 7)
    ref.check(got[:, w:], exp, tol, "columns")
    be.attention(b, b, b, b, n, n, heads, heads, dim, y_stride=3 * w, **at)
    got2 = be.download(b).reshape(n, 3 * w)
    assert np.array_equal(got2[:, :w], got[:, w:]) and np.array_equal(got2[:, w:], qkv[:, w:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_are_clamped(backends, dtype):
    """Offsets past the rows and falling ones: sequences are cut at the rows that there are, or empty."""
    be, rng, n, dim = backends[dtype], np.random.default_rng(8), 64, 64
    q, k, v = (sh.storage_round(rng.standard_normal((n, 1, dim)).astype(np.float32), dtype) for _ in range(3))
    y = be.upload(np.full(n * dim, 7, np.float32))
    be.attention(be.upload(q), be.upload(k), be.upload(v), y, n, n, 1, 1, dim,
                 q_offsets=be.upload_i32(np.array([-5, 20, 10, 40, 100])),
                 kv_offsets=be.upload_i32(np.array([-9, 30, 50, 44, 2000000000])))
    got = be.download(y).reshape(n, 1, dim)
    # Sequences: rows 0..19 on keys 0..29; 20..9: none; 10..39 on 50..43: no keys; 40..63 on 44..63.
    exp, err, _ = ref.attention(*(a.astype(np.float64) for a in (q, k, v)), dim ** -0.5, 1, [0, 10, 40, 64], [0, 30, 30, 64],
                                ref.HALF[dtype])
    tol = err + ref.stored(exp, dtype)
    ref.check(got[:10], exp[:10], tol[:10], "first")
    exp2, err2, _ = ref.attention(q[40:].astype(np.float64), *(a[44:].astype(np.float64) for a in (k, v)), dim ** -0.5, 1,
                                  [0, 24], [0, 20], ref.HALF[dtype])
    ref.check(got[40:], exp2, err2 + ref.stored(exp2, dtype), "last")
    assert not got[20:40].any()


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_refusals(backends, dtype):
    be, bad = backends[dtype], sh.INVALID_ARGUMENT
    n, dim = 64, 32
    q, k, v, y = (be.alloc(n * 2 * dim) for _ in range(4))
    at = be.upload_i32(np.array([0, 64], np.int32))

    def att(**more):
        args = dict(q=q, k=k, v=v, y=y, nq=n, nkv=n, heads=2, kv_heads=2, head_dim=dim)
        args.update({key: more.pop(key) for key in list(more) if key in args})
        be.attention(*args.values(), **more)

    def refuse(status=bad, **more):
        with pytest.raises(sh.HipError) as e:
            att(**more)
        assert e.value.status == status, (more, e.value)

    att()
    refuse(nq=65)
    refuse(nq=0)
    refuse(nkv=65)
    refuse(nkv=-1)
    refuse(nq=1 << 40)
    refuse(heads=0)
    refuse(heads=3)
    refuse(kv_heads=0)
    refuse(heads=2, kv_heads=4)
    refuse(head_dim=0)
    refuse(sh.NOT_IMPLEMENTED, nq=1, nkv=1, head_dim=193)
    refuse(scale=float("nan"))
    refuse(scale=float("inf"))
    refuse(q_offsets=at)
    refuse(kv_offsets=at)
    refuse(q_offsets=at, kv_offsets=be.upload_i32(np.zeros(1, np.int32)))
    refuse(q_offsets=q, kv_offsets=at)
    refuse(k=None)
    refuse(q_stride=8)
    refuse(k_stride=72)
    refuse(v_offset=8)
    refuse(q_offset=-8)
    refuse(y=k)
    refuse(y=v)
    refuse(nq=32, y=q, y_offset=8, y_stride=64)
    refuse(q=at)
    refuse(k=be.alloc_rows8(n, 2 * dim))
    st = sh.LIB.trellis_sparse_hip_attention(be.ptr, q.handle, k.handle, v.handle, y.handle, n, n, None, None, 1,
                                             ctypes.byref(sh.AttentionDesc()))
    assert st == bad
    st = sh.LIB.trellis_sparse_hip_attention(be.ptr, q.handle, k.handle, v.handle, y.handle, n, n, None, None, 1, None)
    assert st == bad
