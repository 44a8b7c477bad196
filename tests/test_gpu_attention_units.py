"""Attention with changed scores where its work is dealt out in uncommon ways: units beyond whole rounds of the CUs split over
their keys while the others are not, splits joined by sixteen wavefronts a query; and keys and values that hold NaN where no
query, or not every one, sees them, in every form."""
import numpy as np
import pytest

import rows64 as ref
import scored_tight64 as tight
import sparse_hip as sh
from test_gpu_attention_caps import run
from test_gpu_attention_scored import offsets, run_case

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]
CUS = 256


@pytest.fixture
def backend(request):
    be = sh.Backend(0, request.param)
    yield request.param, be
    be.destroy()


def scratch_of(units, key_tiles, dim):
    """Bytes of the units that are left over after whole rounds, in as many splits as they get."""
    whole, splits = units // CUS * CUS, min(8, key_tiles // 16)
    assert units > 2 * CUS and 0 < whole < units and splits > 1
    return splits * (units - whole) * 128 * (dim + 2) * 4


@pytest.mark.parametrize("cap,bias", [(8.0, None), (0.0, "voxels"), (8.0, "rows")])
@pytest.mark.parametrize("q_len,k_len,heads,kv_heads,dim", [
    ([33], [9000], 520, 520, 8), ([300], [2111], 180, 180, 64), ([150, 0, 300], [2100, 2500, 3000], 110, 110, 32),
    ([50, 40], [2500, 1700], 360, 180, 96), ([130], [2048], 260, 260, 128)])
@pytest.mark.parametrize("backend", DTYPES, indirect=True)
def test_whole_units_and_split_ones(backend, q_len, k_len, heads, kv_heads, dim, cap, bias):
    """All rows of some heads against float64: the first ones' units are whole, the last one's are split."""
    dtype, be = backend
    rng, nq, nk, group = np.random.default_rng(heads + dim), sum(q_len), sum(k_len), heads // kv_heads
    q, k, v = (sh.storage_round(rng.standard_normal((n, h, dim), np.float32), dtype)
               for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads)))
    slopes = None if bias is None else (0.05 * rng.random(heads)).astype(np.float32)
    kw, xyz = {}, [None, None]
    if bias == "voxels":
        xyz = [rng.integers(0, 64, (n, 4)).astype(np.int32) for n in (nq, nk)]
        kw = {"q_coords": be.upload_i32(xyz[0]), "k_coords": be.upload_i32(xyz[1])}
    qa, ka = offsets(q_len), offsets(k_len)
    if len(q_len) > 1:
        kw.update(q_offsets=be.upload_i32(qa), kv_offsets=be.upload_i32(ka))
    y = be.alloc(nq * heads * dim)
    be.attention_scored(be.upload(q), be.upload(k), be.upload(v), y, nq, nk, heads, kv_heads, dim, cap=cap, slopes=slopes, **kw)
    tiles = nq * group // 128 + len(q_len)
    assert be.scratch_bytes == scratch_of(tiles * kv_heads, (nk // len(k_len) + 63) // 64, dim)
    got, d = be.download(y).reshape(nq, heads, dim), lambda a: None if a is None else a.astype(np.float64)
    half = ref.E if dtype == sh.F32 else ref.HALF[dtype]
    for h in (0, kv_heads // 2, kv_heads - 2, kv_heads - 1):
        own = slice(h * group, (h + 1) * group)
        for s in range(len(q_len)):
            a, b = slice(qa[s], qa[s + 1]), slice(ka[s], ka[s + 1])
            exp, tol = tight.attention(d(q[a, own]), d(k[b, h:h + 1]), d(v[b, h:h + 1]), dim ** -0.5, half, cap,
                                       None if slopes is None else d(slopes[own]), None if xyz[0] is None else xyz[0][a],
                                       None if xyz[1] is None else xyz[1][b], of_cap=0.0 if dtype == sh.F32 else 2.0 ** -22)
            ref.check(got[a, own], exp, tol + ref.stored(exp, dtype), f"head {h} of {kv_heads}, sequence {s}")


@pytest.mark.parametrize("form", [dict(), dict(bias="rows", causal=True, slope=0.001), dict(bias="voxels", slope=0.05),
                                  dict(cap=20.0, causal=True, prefix=100)])
@pytest.mark.parametrize("nq,heads,kv_heads,dim", [(1, 1, 1, 64), (1, 4, 1, 128), (20, 1, 1, 8), (31, 1, 1, 96), (100, 1, 1, 40),
                                                   (40, 2, 2, 32)])
@pytest.mark.parametrize("backend", DTYPES, indirect=True)
def test_many_splits(backend, form, nq, heads, kv_heads, dim):
    """40,000 keys in 156 splits."""
    dtype, be = backend
    half = ref.E if dtype == sh.F32 else 2 * ref.HALF[dtype] ** 2
    run(be, dtype, nq, 40000, heads, kv_heads, dim, half=half, **form)
    queries = nq * heads // kv_heads
    wide = 32 if queries <= 32 else 128
    assert be.scratch_bytes == 156 * (queries // wide + 1) * kv_heads * wide * (dim + 2) * 4


@pytest.mark.parametrize("form", ["voxels", "cap_rows_causal", "all"])
@pytest.mark.parametrize("backend", DTYPES, indirect=True)
def test_many_splits_of_uneven_sequences(backend, form):
    """One long cache, one of five rows and one of none: 143 splits of each."""
    dtype, be = backend
    run_case(be, dtype, [1, 1, 1], [110000, 0, 5], 2, 1, 64, form)
    assert be.scratch_bytes >= 143 * 32 * 66 * 4


@pytest.mark.parametrize("nq,nk,prefix,heads,kv_heads,dim", [(40, 40, 0, 2, 2, 64), (200, 200, 70, 6, 2, 64), (129, 300, 100, 4, 1, 96),
                                                             (300, 129, 5, 3, 3, 128), (70, 70, 64, 2, 1, 13), (3, 20000, 7, 4, 1, 64),
                                                             (2, 500, 0, 2, 2, 32), (1000, 1000, 300, 8, 4, 64)])
@pytest.mark.parametrize("bias", [None, "rows", "voxels"])
@pytest.mark.parametrize("backend", DTYPES, indirect=True)
def test_unseen_keys_hold_anything(backend, bias, nq, nk, prefix, heads, kv_heads, dim):
    """Keys and values behind a query's own place and the prefix hold NaN, infinities or the type's lowest value: the queries
    that do not see them have the bits that they have without."""
    dtype, be = backend
    rng = np.random.default_rng(nq + nk + prefix + dim)
    q, k, v = (sh.storage_round(rng.standard_normal((n, h, dim)).astype(np.float32), dtype)
               for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads)))
    kw = dict(slopes=np.full(heads, 0.02, np.float32)) if bias else {}
    if bias == "voxels":
        kw.update({f"{a}_coords": be.upload_i32(rng.integers(0, 64, (n, 4)).astype(np.int32)) for a, n in (("q", nq), ("k", nk))})
    if prefix:
        kw["prefix"] = be.upload_i32(np.array([prefix], np.int32))

    def call(k, v):
        y = be.alloc(nq * heads * dim)
        be.attention_scored(be.upload(q), be.upload(k), be.upload(v), y, nq, nk, heads, kv_heads, dim, cap=20.0, causal=True, **kw)
        return be.download(y).reshape(nq, heads, dim)

    base, place = call(k, v), np.arange(nq) + nk - nq
    assert np.isfinite(base).all()
    lowest = {sh.F32: -3.4e38, sh.F16: -65504.0, sh.BF16: -3.38e38}[dtype]
    for first in sorted({max(prefix, nk - 1), max(prefix, nk - max(1, nq // 3)), max(prefix, nk - nq + 1)}):
        if first >= nk:
            continue
        blind = place < first
        for bad in (np.nan, np.inf, lowest):
            k2, v2 = k.copy(), v.copy()
            k2[first:], v2[first:] = bad, bad
            np.testing.assert_array_equal(call(k2, v2)[blind], base[blind])
