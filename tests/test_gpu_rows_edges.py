"""The row operators at their edges: rows behind the last stay as they were, sums and keys split through scratch of the
pool's, of the caller's and of none, thousands of short sequences, rows whose alignment leaves the wide kernels.  Bounds:
tests/rows64.py."""
import numpy as np
import pytest

import rows64 as ref
import sparse_hip as sh
from test_gpu_attention import run_case
from test_gpu_rows import make, refused

pytestmark = pytest.mark.gpu
DTYPES = [sh.F32, sh.F16, sh.BF16]
GUARD = 300  # rows, more than any block has


@pytest.fixture(scope="module")
def backends():
    bes = {dt: sh.Backend(0, dt) for dt in DTYPES}
    yield bes
    for b in bes.values():
        b.destroy()


def guarded(be, n, c):
    """Rows for an output, with GUARD more behind them; and what checks those."""
    y = be.upload(np.full((n + GUARD, c), 7, np.float32))

    def rows():
        got = be.download(y).reshape(n + GUARD, c)
        assert np.all(got[n:] == 7)
        return got[:n]
    return y, rows


@pytest.mark.parametrize("from8", [False, True])
@pytest.mark.parametrize("n,ci,co", [(1, 64, 64), (1, 4096, 1024), (5, 300, 77), (33, 2048, 130), (65, 128, 256), (129, 36, 4),
                                     (1000, 1024, 1024), (20000, 256, 512), (20001, 200, 1032)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_ends_at_its_rows(backends, dtype, n, ci, co, from8):
    be, rng = backends[dtype], np.random.default_rng(n + ci + co)
    x, r, w = make(rng, dtype, n, ci), make(rng, dtype, n, co), make(rng, dtype, co, ci) / 16
    xb = be.upload(x)
    if from8:
        q = be.alloc_rows8(n, ci)
        be.pack_rows8(xb, q, n, ci)
        xb = q
    y, rows = guarded(be, n, co)
    plain = be.alloc(n * co)
    be.linear_act(xb, w, None, plain, n, ci, co, act="gelu", residual=be.upload(r))
    be.linear_act(xb, w, None, y, n, ci, co, act="gelu", residual=be.upload(r))
    assert np.array_equal(rows(), be.download(plain).reshape(n, co))


@pytest.mark.parametrize("act", list(sh.ACTS))
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_act_of_the_largest_blocks(backends, dtype, act, residual):
    """51 x 4 tiles of 256 x 256, whose outputs are computed while earlier ones are stored; many tiles a block too."""
    be, rng = backends[dtype], np.random.default_rng(3)
    for n, ci, co in ((13056, 200, 1024), (40000, 96, 1024)):
        x, r, w = make(rng, dtype, n, ci), make(rng, dtype, n, co), (rng.standard_normal((co, ci)) / 14).astype(np.float32)
        b = rng.standard_normal(co).astype(np.float32)
        y = be.alloc(n * co)
        be.linear_act(be.upload(x), w, b, y, n, ci, co, act=act, residual=be.upload(r) if residual else None)
        got = be.download(y).reshape(n, co)
        rows = np.concatenate([np.arange(300), rng.integers(0, n, 300), np.arange(n - 300, n)])
        exp, err = ref.linear_act(x[rows].astype(np.float64), sh.storage_round(w, dtype).astype(np.float64),
                                  b.astype(np.float64), act, r[rows].astype(np.float64) if residual else None)
        ref.check(got[rows], exp, err + ref.stored(exp, dtype), f"{n} {act}")


@pytest.mark.parametrize("n,c", [(1, 64), (33, 100), (7, 512), (130, 1024), (5, 4100)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_and_expansion_end_at_their_rows(backends, dtype, n, c):
    be, rng = backends[dtype], np.random.default_rng(n + c)
    x = make(rng, dtype, n, c)
    xb, plain = be.upload(x), be.alloc(n * c)
    y, rows = guarded(be, n, c)
    t, total = guarded(be, n, c)
    be.rms_norm(xb, None, plain, n, c, 1e-6, residual=xb)
    be.rms_norm(xb, None, y, n, c, 1e-6, residual=xb, total=t)
    assert np.array_equal(rows(), be.download(plain).reshape(n, c))
    total()
    q = be.alloc_rows8(n, c)
    be.pack_rows8(xb, q, n, c)
    y, rows = guarded(be, n, c)
    be.expand_rows8(q, y, n, c)
    be.expand_rows8(q, plain, n, c)
    assert np.array_equal(rows(), be.download(plain).reshape(n, c))


@pytest.mark.parametrize("n,dim", [(1, 64), (15, 48), (17, 128), (100, 256)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_ends_at_its_rows(backends, dtype, n, dim):
    be, rng, heads = backends[dtype], np.random.default_rng(n + dim), 2
    x = be.upload(make(rng, dtype, n, heads * dim))
    coords = be.upload_i32(rng.integers(0, 64, (n, 4)).astype(np.int32))
    y, rows = guarded(be, n, heads * dim)
    be.rotary(x, coords, y, n, heads, dim, (dim // 8,) * 3, 10000.0)
    assert np.isfinite(rows()).all()


def split_calls(be, rng, dtype):
    """Calls that split: {name: (call on an output of so many values)}; their inputs stay alive in them."""
    x, w = be.upload(make(rng, dtype, 3, 4096)), make(rng, dtype, 512, 4096) / 64
    wide, w2 = be.upload(make(rng, dtype, 700, 2048)), make(rng, dtype, 77, 2048) / 64
    q, k = be.upload(make(rng, dtype, 5, 128)), be.upload(make(rng, dtype, 9000, 128))
    v = be.upload(make(rng, dtype, 9000, 128))
    many = be.upload(make(rng, dtype, 200, 128))
    return {"linear": (3 * 512, lambda y: be.linear_act(x, w, None, y, 3, 4096, 512, act="silu")),
            "linear odd": (700 * 77, lambda y: be.linear_act(wide, w2, None, y, 700, 2048, 77)),
            "attention": (5 * 128, lambda y: be.attention(q, k, v, y, 5, 9000, 2, 2, 64)),
            "attention many": (200 * 128, lambda y: be.attention(many, k, v, y, 200, 9000, 1, 1, 128))}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["linear", "linear odd", "attention", "attention many"])
def test_scratch(dtype, what):
    """The caller's scratch gives what the pool's does, bit for bit, and is written no further than a call asks; where it is
    too small the pool's serves; without any the result is within the roundings of another order of the sums."""
    be = sh.Backend(0, dtype)
    try:
        count, call = split_calls(be, np.random.default_rng(11), dtype)[what]
        assert be.scratch_bytes == 0
        y = be.alloc(count)
        call(y)
        need, pooled = be.scratch_bytes, be.download(y)
        assert need > 0 and need % 4 == 0
        words = np.full(need // 4 + 64, 7, np.int32)
        scratch = be.upload_i32(words)
        be.set_scratch(scratch)
        got = be.alloc(count)
        call(got)
        assert np.array_equal(be.download(got), pooled)
        after = be.download_i32(scratch)
        assert np.all(after[need // 4:] == 7) and not np.all(after[:need // 4] == 7)
        small = be.upload_i32(words[:need // 4 - 1])
        be.set_scratch(small)
        call(got)
        assert np.array_equal(be.download(got), pooled) and np.all(be.download_i32(small) == 7)
        be.set_scratch(scratch)
        scratch.free()  # unset with it
        be.trim(sh.TRIM_FREE_BUFFERS)
        be.fail_alloc(0)
        try:
            call(got)
        finally:
            be.fail_alloc(-1)
        # 9,000 terms of fp32 in another order, 8 sqrt(9000) 2^-24 of sums that stay within 4; and two roundings to the type.
        one = be.download(got)
        tol = 8 * np.sqrt(9000) * ref.E * 4 + 2 * ref.HALF[dtype] * np.abs(pooled)
        if what.startswith("attention"):
            tol = tol + 2 * ref.HALF[dtype] * 4 * 9000 ** -0.5 * 8  # each weight rounded twice, 8 deviations
        assert np.all(np.abs(one - pooled) <= tol)
    finally:
        be.destroy()


def test_scratch_refusals():
    be = sh.Backend(0, sh.BF16)
    try:
        rng = np.random.default_rng(2)
        w = make(rng, sh.BF16, 512, 4096)
        big = be.upload(np.zeros(1 << 21, np.float32))
        x, y = be.upload(make(rng, sh.BF16, 1, 4096)), be.alloc(512)
        be.linear_act(x, w, None, y, 1, 4096, 512)
        assert 0 < be.scratch_bytes <= 1 << 22
        refused(sh.INVALID_ARGUMENT, be.set_scratch, be.alloc_rows8(64, 64))
        be.set_scratch(big)
        refused(sh.INVALID_ARGUMENT, be.linear_act, x, w, None, big, 1, 4096, 512)
        refused(sh.INVALID_ARGUMENT, be.linear_act, big, w, None, y, 1, 4096, 512)
        refused(sh.INVALID_ARGUMENT, be.linear_act, x, w, None, y, 1, 4096, 512, residual=big)
        k = be.alloc(9000 * 64)
        refused(sh.INVALID_ARGUMENT, be.attention, big, k, k, y, 1, 9000, 1, 1, 64)
        refused(sh.INVALID_ARGUMENT, be.attention, y, k, big, x, 1, 9000, 1, 1, 64)
        be.set_scratch(None)
        be.linear_act(big, w, None, y, 1, 4096, 512)
        be.linear_act(x, w, None, big, 1, 4096, 512)
    finally:
        be.destroy()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("seqs,most", [(64, 40), (65, 3), (1000, 2), (5000, 3), (300, 200)])
def test_many_sequences(backends, dtype, seqs, most):
    """More sequences than are found in one look, of 0 to `most` rows each."""
    rng = np.random.default_rng(seqs)
    q_len, k_len = (rng.integers(0, most + 1, seqs) for _ in range(2))
    run_case(backends[dtype], dtype, list(q_len), list(k_len), 2, 1, 32, extra=5)


@pytest.mark.parametrize("dim", [4, 12, 36, 68, 100, 124, 128, 132])
def test_fp32_head_widths(backends, dim):
    run_case(backends[sh.F32], sh.F32, [70, 1], [131, 65], 2, 2, dim)
    run_case(backends[sh.F32], sh.F32, [1], [5000], 4, 2, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_attention_of_rows_off_16_bytes(backends, dtype, shift):
    """Rows and strides that no 16-byte load can take: the same values."""
    be, rng, n, heads, dim = backends[dtype], np.random.default_rng(shift), 100, 2, 64
    w = heads * dim
    qkv = make(rng, dtype, n, 3 * w)
    q, k, v = (qkv[:, i * w:(i + 1) * w].reshape(n, heads, dim).astype(np.float64) for i in range(3))
    exp, err, _ = ref.attention(q, k, v, dim ** -0.5, 1, [0, n], [0, n], ref.HALF[dtype])
    pitch = 3 * w + shift
    rows = np.full((n, pitch), 9, np.float32)
    rows[:, shift:] = qkv
    b, y = be.upload(rows), be.upload(np.full((n, w + shift), 7, np.float32))
    be.attention(b, b, b, y, n, n, heads, heads, dim, q_offset=shift, q_stride=pitch, k_offset=w + shift, k_stride=pitch,
                 v_offset=2 * w + shift, v_stride=pitch, y_offset=shift, y_stride=w + shift)
    got = be.download(y).reshape(n, w + shift)
    assert np.all(got[:, :shift] == 7)
    ref.check(got[:, shift:].reshape(n, heads, dim), exp, err + ref.stored(exp, dtype), "shifted")


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_offsets_over_the_output(backends, dtype):
    """Offsets read while rows of y are written: refused."""
    be, n, dim = backends[dtype], 32, 32
    q = be.alloc(n * dim)
    at = be.upload_i32(np.array([0, n] + [0] * n * dim, np.int32))
    refused(sh.INVALID_ARGUMENT, be.attention, q, q, q, at, n, n, 1, 1, dim, q_offsets=at, kv_offsets=at)
