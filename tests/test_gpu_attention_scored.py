"""Attention with capped, biased and masked scores against float64: every head width and type, one query and many, both sides
of the kernels' tiles, prefixes, rows that see nothing, what is not seen, grouped heads, strides, refusals.  Bounds:
tests/scored64.py."""
import ctypes

import numpy as np
import pytest

import rows64 as ref
import scored64 as more
import sparse_hip as sh

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]
# cap, distances, causal, prefix
FORMS = {"cap": (5.0, None, False, 0), "rows": (0.0, "rows", False, 0), "voxels": (0.0, "voxels", False, 0),
         "causal": (0.0, None, True, 0), "prefix": (0.0, None, True, 40), "all": (8.0, "voxels", True, 9),
         "cap_rows_causal": (20.0, "rows", True, 0), "none": (0.0, None, False, 0)}


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in DTYPES}
    yield bes
    for b in bes.values():
        b.destroy()


def offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def run_case(be, dtype, q_len, k_len, heads, kv_heads, dim, form, scale=0.0, seed=0, extra=0, whole=False, sharp=2.0, grid=64,
             far=0, prefix=None, slopes=None, poison=False):
    """Sequences of the given lengths; `extra` more rows behind the last of q and of k, which hold NaN; `poison`: so do the
    keys and values that no query sees, and in causal forms without a prefix those that only the last query sees."""
    rng = np.random.default_rng(seed + sum(q_len) + 3 * sum(k_len) + 5 * dim)
    cap, bias, causal, pre = FORMS[form] if isinstance(form, str) else form
    nq, nk = sum(q_len) + extra, sum(k_len) + extra
    q = sh.storage_round((sharp * rng.standard_normal((nq, heads, dim))).astype(np.float32), dtype)
    k = sh.storage_round(rng.standard_normal((nk, kv_heads, dim)).astype(np.float32), dtype)
    v = sh.storage_round(rng.standard_normal((nk, kv_heads, dim)).astype(np.float32), dtype)
    if extra:
        k[-extra:], v[-extra:] = np.nan, np.inf
    qa, ka = offsets(q_len), offsets(k_len)
    kw = {}
    if bias and slopes is None:
        slopes = np.float32(2.0) ** -np.arange(1, heads + 1, dtype=np.float32) if bias == "rows" else \
            (0.5 * rng.random(heads)).astype(np.float32)
    q_xyz = k_xyz = None
    if bias == "voxels":
        k_xyz = (rng.integers(0, grid, (nk, 4)) + far).astype(np.int32)
        q_xyz = (rng.integers(0, grid, (nq, 4)) + far).astype(np.int32)
        kw = {"q_coords": be.upload_i32(q_xyz), "k_coords": be.upload_i32(k_xyz) if nk else None}
    if pre or prefix is not None:
        prefix = np.full(len(q_len), pre, np.int32) if prefix is None else np.asarray(prefix, np.int32)
        kw["prefix"] = be.upload_i32(prefix)
    y = be.upload(np.full(nq * heads * dim, 7, np.float32))
    at = {} if whole else {"q_offsets": be.upload_i32(qa), "kv_offsets": be.upload_i32(ka)}
    be.attention_scored(be.upload(q), be.upload(k) if nk else None, be.upload(v) if nk else None, y, nq, nk, heads, kv_heads,
                        dim, scale=scale, cap=cap, slopes=slopes, causal=causal, **kw, **at)
    got = be.download(y).reshape(nq, heads, dim)
    d = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    exp, err, inside = more.attention(d(q), d(k), d(v), scale or dim ** -0.5, heads // kv_heads, qa, ka, ref.HALF[dtype],
                                      float(np.float32(cap)), d(slopes), q_xyz, k_xyz, causal, prefix)
    assert inside.sum() == sum(q_len) and np.all(got[~inside] == 7)
    ref.check(got[inside], exp[inside], (err + ref.stored(exp, dtype))[inside],
              f"{form} {q_len} {k_len} {heads}/{kv_heads} {dim}")


@pytest.mark.parametrize("dim", [8, 16, 32, 40, 64, 96, 128, 13, 160, 192])
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_widths(backends, dtype, form, dim):
    run_case(backends[dtype], dtype, [70], [131], 2, 2, dim, form, whole=True)


@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 2), (2, 1), (31, 33), (32, 32), (33, 64), (64, 65), (127, 129), (128, 63),
                                   (129, 128), (257, 200), (1, 4097), (3, 700), (40, 5000), (1000, 17), (700, 700)])
@pytest.mark.parametrize("form", ["all", "cap_rows_causal", "voxels", "prefix"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths(backends, dtype, form, nq, nk):
    run_case(backends[dtype], dtype, [nq], [nk], 3, 3, 64, form, whole=(nq + nk) % 2 == 0)
    run_case(backends[dtype], dtype, [nq], [nk], 2, 1, 128, form)


@pytest.mark.parametrize("q_len,k_len", [([5, 0, 130, 1], [5, 0, 130, 1]), ([3, 64, 2], [0, 200, 0]), ([0, 0, 9], [4, 4, 4]),
                                         ([1] * 70, [3, 0] * 35), ([1, 1, 1, 1], [1000, 0, 65, 2500]), ([0], [3]),
                                         ([40] * 9, [0] * 9), ([2] * 130, [7] * 130), ([100, 300], [50, 310])])
@pytest.mark.parametrize("form", ["all", "cap_rows_causal", "prefix", "voxels"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_sequences(backends, dtype, form, q_len, k_len):
    run_case(backends[dtype], dtype, q_len, k_len, 2, 2, 64, form, extra=3)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (6, 2), (16, 4), (17, 17), (40, 8)])
@pytest.mark.parametrize("form", ["all", "cap_rows_causal"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_grouped_heads(backends, dtype, form, heads, kv_heads):
    """Each head has a slope of its own, also where heads share keys."""
    run_case(backends[dtype], dtype, [3, 50], [90, 33], heads, kv_heads, 64, form)
    run_case(backends[dtype], dtype, [1, 1], [900, 333], heads, kv_heads, 32, form)


@pytest.mark.parametrize("prefix", [[0, 0, 0], [5, 64, 1], [1000, 1000, 1000], [63, 65, 200], [-3, 2, -1]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_prefixes(backends, dtype, prefix):
    """None, in a tile, whole tiles, beyond the last key, negative; sequences with more queries than keys."""
    for q_len, k_len in (([150, 70, 130], [150, 200, 40]), ([1, 2, 1], [300, 10, 1])):
        run_case(backends[dtype], dtype, q_len, k_len, 2, 2, 64, (0.0, None, True, 0), prefix=prefix)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale,sharp,cap", [(0.01, 1.0, 1.0), (1.0, 1.0, 30.0), (0.125, 40.0, 50.0), (-0.2, 1.0, 5.0),
                                             (1.0, 40.0, 1000.0), (1.0, 5.0, 0.01)])
def test_scales(backends, dtype, scale, sharp, cap):
    """Caps far above the scores and far below them, negative scales."""
    run_case(backends[dtype], dtype, [100], [700], 2, 2, 64, (cap, None, False, 0), scale=scale, sharp=sharp, whole=True)


@pytest.mark.parametrize("grid,far,slope", [(4, 0, 0.7), (128, 0, 0.05), (1024, 0, 0.01), (1024, 60000, 0.3), (2048, -1024, 0.02),
                                            (32768, 0, 0.001), (4096, 0, 0.1), (65536, 1 << 28, 0.01), (64, 0, -0.05)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_voxel_distances(backends, dtype, grid, far, slope):
    """Grids of every size, away from the origin too; negative slopes."""
    run_case(backends[dtype], dtype, [70, 200], [131, 200], 2, 2, 64, "voxels", grid=grid, far=far,
             slopes=np.array([slope, 0.0], np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
def test_near_voxels_far_from_the_others(backends, dtype):
    """Two clusters a million voxels apart: distances within each are right to the last voxel."""
    be, rng, n, dim = backends[dtype], np.random.default_rng(7), 200, 64
    xyz = rng.integers(0, 4, (n, 4)).astype(np.int32)
    xyz[rng.random(n) < 0.5, 1:] += 1 << 20
    q, k, v = (sh.storage_round(rng.standard_normal((n, 1, dim)).astype(np.float32), dtype) for _ in range(3))
    slopes = np.array([1.5], np.float32)
    y, at = be.alloc(n * dim), be.upload_i32(xyz)
    be.attention_scored(be.upload(q), be.upload(k), be.upload(v), y, n, n, 1, 1, dim, slopes=slopes, q_coords=at, k_coords=at)
    d = lambda a: a.astype(np.float64)  # noqa: E731
    exp, err, _ = more.attention(d(q), d(k), d(v), dim ** -0.5, 1, [0, n], [0, n], ref.HALF[dtype], 0.0, d(slopes), xyz, xyz)
    ref.check(be.download(y).reshape(n, 1, dim), exp, err + ref.stored(exp, dtype), "clusters")


@pytest.mark.parametrize("n", [40, 70, 129, 300])
@pytest.mark.parametrize("dim", [64, 96, 13])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_is_not_seen_reaches_nothing(backends, dtype, n, dim):
    """Keys and values that hold NaN, infinities or the type's lowest value change nothing for the queries before them; the
    queries that see such a value have it, those that see such a key are NaN."""
    be, rng = backends[dtype], np.random.default_rng(n + dim)
    q, k, v = (sh.storage_round(rng.standard_normal((n, 2, dim)).astype(np.float32), dtype) for _ in range(3))

    def run(q, k, v):
        y = be.alloc(n * 2 * dim)
        be.attention_scored(be.upload(q), be.upload(k), be.upload(v), y, n, n, 2, 2, dim, causal=True)
        return be.download(y).reshape(n, 2, dim)

    base, at = run(q, k, v), 2 * n // 3
    for bad in (np.nan, np.inf, -np.inf, {sh.F32: -3.4e38, sh.F16: -65504.0, sh.BF16: -3.38e38}[dtype]):
        v2 = v.copy()
        v2[at, 1, 5] = bad
        got = run(q, k, v2)
        np.testing.assert_array_equal(got[:, 0], base[:, 0])
        np.testing.assert_array_equal(got[:at], base[:at])
        others = np.arange(dim) != 5
        np.testing.assert_array_equal(got[at:, 1][:, others], base[at:, 1][:, others])
        if not np.isfinite(bad):
            assert np.all(np.isnan(got[at:, 1, 5])) if np.isnan(bad) else np.all(got[at:, 1, 5] == bad)
        k2 = k.copy()
        k2[at:, 1] = bad
        got = run(q, k2, v)
        np.testing.assert_array_equal(got[:, 0], base[:, 0])
        np.testing.assert_array_equal(got[:at], base[:at])
        if np.isnan(bad):
            assert np.isnan(got[at:, 1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_changes_as_attention(backends, dtype):
    """No cap, slopes or mask: the scores of attention (to the bounds of both)."""
    run_case(backends[dtype], dtype, [500, 3], [400, 70], 4, 2, 64, "none")


@pytest.mark.parametrize("dim", [64, 128, 20])
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_offsets(backends, dtype, dim):
    """q, k and v as columns of one buffer, y as columns of another with other columns left as they were; y in q's place."""
    be, rng, n, heads = backends[dtype], np.random.default_rng(9), 150, 2
    c = heads * dim
    qkv = sh.storage_round(rng.standard_normal((n, 3 * c + 8)).astype(np.float32), dtype)
    xyz = rng.integers(0, 32, (n, 4)).astype(np.int32)
    slopes = np.array([0.2, 0.05], np.float32)
    d = lambda a: a.astype(np.float64)  # noqa: E731
    q, k, v = (qkv[:, i * c:(i + 1) * c].reshape(n, heads, dim) for i in range(3))
    exp, err, _ = more.attention(d(q), d(k), d(v), dim ** -0.5, 1, [0, n], [0, n], ref.HALF[dtype], 10.0, d(slopes), xyz, xyz,
                                 True)
    at, buf, pitch = be.upload_i32(xyz), be.upload(qkv), 3 * c + 8
    places = dict(q_stride=pitch, k_offset=c, k_stride=pitch, v_offset=2 * c, v_stride=pitch, cap=10.0, slopes=slopes,
                  q_coords=at, k_coords=at, causal=True)
    y = be.upload(np.full(n * (c + 16), 7, np.float32))
    be.attention_scored(buf, buf, buf, y, n, n, heads, heads, dim, y_offset=8, y_stride=c + 16, **places)
    got = be.download(y).reshape(n, c + 16)
    assert np.all(got[:, :8] == 7) and np.all(got[:, 8 + c:] == 7)
    ref.check(got[:, 8:8 + c].reshape(n, heads, dim), exp, err + ref.stored(exp, dtype), "columns")
    be.attention_scored(buf, buf, buf, buf, n, n, heads, heads, dim, y_stride=pitch, **places)
    own = be.download(buf).reshape(n, pitch)
    np.testing.assert_array_equal(own[:, :c], got[:, 8:8 + c])
    np.testing.assert_array_equal(own[:, c:], qkv[:, c:])


def test_refusals(backends):
    be, n, dim = backends[sh.BF16], 16, 32
    q, k, v, y = (be.alloc(n * 2 * dim) for _ in range(4))
    at, pre = be.upload_i32(np.zeros(n * 4, np.int32)), be.upload_i32(np.zeros(1, np.int32))
    one = np.ones(2, np.float32)

    def refuse(status=sh.INVALID_ARGUMENT, **kw):
        a = dict(q=q, k=k, v=v, y=y, nq=n, nkv=n, heads=2, kv_heads=2, head_dim=dim)
        a.update(kw)
        with pytest.raises(sh.HipError) as e:
            be.attention_scored(**a)
        assert e.value.status == status

    refuse(cap=-1.0)
    refuse(cap=float("nan"))
    refuse(cap=float("inf"))
    refuse(cap=3e38)
    refuse(cap=1e-38, scale=1e3)
    refuse(prefix=pre)
    refuse(prefix=q, causal=True)
    refuse(q_coords=at, k_coords=at)
    refuse(slopes=one, q_coords=at)
    refuse(slopes=one, k_coords=at)
    refuse(slopes=one, q_coords=q, k_coords=at)
    refuse(slopes=one, q_coords=pre, k_coords=at)
    refuse(slopes=one, q_coords=at, k_coords=pre)
    refuse(slopes=np.array([1, np.nan], np.float32))
    refuse(slopes=np.array([np.inf, 1], np.float32))
    refuse(slopes=np.array([1, 1e20], np.float32))
    refuse(nq=n + 1)
    refuse(nkv=n + 1)
    refuse(heads=3)
    refuse(y=k)
    refuse(head_dim=200, status=sh.NOT_IMPLEMENTED)
    seqs = be.upload_i32(np.array([0, 3, n], np.int32))
    refuse(q_offsets=seqs, kv_offsets=seqs, causal=True, prefix=pre)
    d, s = sh.AttentionDesc(ctypes.sizeof(sh.AttentionDesc), 2, 2, dim), sh.ScoresDesc(ctypes.sizeof(sh.ScoresDesc))

    def call(desc, scores):
        return sh.LIB.trellis_sparse_hip_attention_scored(be.ptr, q.handle, k.handle, v.handle, y.handle, n, n, None, None, 1,
                                                          desc, scores)
    assert call(None, ctypes.byref(s)) == sh.INVALID_ARGUMENT
    assert call(ctypes.byref(d), None) == sh.INVALID_ARGUMENT
    s.causal = 2
    assert call(ctypes.byref(d), ctypes.byref(s)) == sh.INVALID_ARGUMENT
    s.causal, s.struct_size = 0, 8
    assert call(ctypes.byref(d), ctypes.byref(s)) == sh.INVALID_ARGUMENT
    s.struct_size = ctypes.sizeof(s)
    assert call(ctypes.byref(d), ctypes.byref(s)) == sh.OK
    be.synchronize()
