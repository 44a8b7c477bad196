"""Group norm, integer rows and attention with changed scores as they are used together: the attention block of a sparse
U-Net stage by stage against float64, in a torch program (streams, graphs, rows beyond 2^31 elements), with scratch of the
caller's, without memory, and the transformer block with its linears in integers."""
import os
import subprocess
import sys

import numpy as np
import pytest

import int_block
import rows64 as ref
import rows_block
import scored64 as more
import sparse_hip as sh
from test_gpu_rows_together import block_args

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
DTYPES = [sh.F32, sh.F16, sh.BF16]


@pytest.mark.parametrize("n", [1, 50, 3001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_block_stage_by_stage(dtype, n):
    """Each stage against float64 of the rows that it read."""
    be, rng = sh.Backend(0, dtype), np.random.default_rng(n)
    try:
        blk = int_block.IntBlock(dtype)
        c, fp32 = blk.c, dtype == sh.F32
        coords, at = int_block.voxels(n, rng)
        x = sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype)
        b = blk.buffers(be, n)
        blk.run(be, be.upload(x), be.upload_i32(coords), be.upload_i32(at), n, b)
        d = lambda a: a.astype(np.float64)  # noqa: E731
        norm, qkv, att, out = (d(be.download(b[k]).reshape(n, -1)) for k in ("norm", "qkv", "att", "out"))
        e, t, inside = more.group_norm(d(x), at, d(blk.g), d(blk.b), blk.groups, float(np.float32(blk.eps)), "none")
        assert inside.all()
        ref.check(norm, e, t + ref.stored(e, dtype), "group norm")
        e, t = more.int8_linear(*more.int8_rows(norm), d(blk.wqkv), d(blk.bqkv), "none", None, fp32)
        ref.check(qkv, e, t + ref.stored(e, dtype), "qkv")
        q, k, v = (qkv[:, i * c:(i + 1) * c].reshape(n, blk.heads, blk.dim) for i in range(3))
        e, t, _ = more.attention(q, k, v, blk.dim ** -0.5, 1, at, at, ref.HALF[dtype], blk.cap, d(blk.slopes), coords, coords)
        ref.check(att.reshape(n, blk.heads, blk.dim), e, t + ref.stored(e, dtype), "attention")
        e, t = more.int8_linear(*more.int8_rows(att), d(blk.wo), d(blk.bo), "none", d(x), fp32)
        ref.check(out, e, t + ref.stored(e, dtype), "out")
    finally:
        be.destroy()


@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_transformer_block_in_integers(dtype, n):
    """rows8 = 2 is the calls one by one, bit for bit."""
    be, rng = sh.Backend(0, dtype), np.random.default_rng(n)
    try:
        blk = rows_block.Block(dtype)
        c, w, hid = blk.c, 3 * blk.c, blk.hidden
        coords, at = rows_block.voxels(n, rng)
        x = be.upload(sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype))
        cb, ab, out = be.upload_i32(coords), be.upload_i32(at), be.alloc(n * c)
        be.transformer_block(x, cb, out, n, offsets=ab, rows8=2, **block_args(blk))
        rows, rows_h = be.alloc_rows_int8(n, c), be.alloc_rows_int8(n, hid)
        qkv, att, mid, h, y = (be.alloc(n * m) for m in (w, c, c, hid, c))
        be.rms_norm(x, blk.g1, rows, n, c, 1e-6)
        be.linear_act(rows, blk.wqkv, blk.bqkv, qkv, n, c, w)
        be.rotary(qkv, cb, qkv, n, 2 * blk.heads, blk.dim, (5, 5, 5), gamma=blk.gqk, eps=1e-6, x_stride=w, y_stride=w)
        be.attention(qkv, qkv, qkv, att, n, n, blk.heads, blk.heads, blk.dim, q_offsets=ab, kv_offsets=ab, q_stride=w,
                     k_offset=c, k_stride=w, v_offset=2 * c, v_stride=w)
        be.pack_rows8(att, rows, n, c)
        be.linear_act(rows, blk.wo, blk.bo, mid, n, c, c, residual=x)
        be.rms_norm(mid, blk.g2, rows, n, c, 1e-6)
        be.linear_act(rows, blk.w1, blk.b1, h, n, c, hid, act="gelu_tanh")
        be.pack_rows8(h, rows_h, n, hid)
        be.linear_act(rows_h, blk.w2, blk.b2, y, n, hid, c, residual=mid)
        np.testing.assert_array_equal(be.download_raw(out), be.download_raw(y))
        with pytest.raises(sh.HipError) as e:
            be.transformer_block(x, cb, out, n, offsets=ab, rows8=3, **block_args(blk))
        assert e.value.status == sh.INVALID_ARGUMENT
    finally:
        be.destroy()


def test_scratch_of_the_caller():
    """The same bits in scratch of the caller's as in the pool's; rows, offsets, coordinates and prefixes in it are refused,
    and the output is as it was."""
    be, rng, n, dtype = sh.Backend(0, sh.BF16), np.random.default_rng(4), 4000, sh.BF16
    try:
        c, heads, dim = 64, 1, 64
        x = sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype)
        xyz = rng.integers(0, 64, (n, 4)).astype(np.int32)
        at, pre = np.array([0, 1500, n], np.int32), np.array([7, 9], np.int32)
        slopes = np.array([0.1], np.float32)
        xb, y = be.upload(x), be.upload(np.full(n * c, 7, np.float32))

        def norm(y=y, offsets=None, x=xb):
            be.group_norm(x, None, None, y, n, c, 8, 1e-5, offsets=offsets or be.upload_i32(at))

        def attend(y=y, coords=None, prefix=None, offsets=None):
            coords, offsets = coords or be.upload_i32(xyz), offsets or be.upload_i32(at)
            be.attention_scored(xb, xb, xb, y, n, n, heads, heads, dim, q_offsets=offsets, kv_offsets=offsets, slopes=slopes,
                                q_coords=coords, k_coords=coords, causal=True, prefix=prefix or be.upload_i32(pre))

        norm()
        first, need = be.download_raw(y), be.scratch_bytes
        assert need > 0
        attend()
        second = be.download_raw(y)
        assert be.scratch_bytes > need
        need = be.scratch_bytes
        spare = lambda a: be.upload_i32(np.concatenate([a.ravel(), np.zeros(need // 4, np.int32)]))  # noqa: E731
        rows, coords = be.upload(np.concatenate([x.ravel(), np.zeros(need, np.float32)])), spare(xyz)
        prefix = spare(pre)
        y.free()
        for scratch in (be.alloc(need), rows, coords, prefix):
            be.set_scratch(scratch)
            y = be.upload(np.full(n * c, 7, np.float32))
            norm(y)
            np.testing.assert_array_equal(be.download_raw(y), first)
            attend(y)
            np.testing.assert_array_equal(be.download_raw(y), second)
        rows = be.upload(np.concatenate([x.ravel(), np.zeros(need, np.float32)]))
        coords, prefix = spare(xyz), spare(pre)
        y = be.upload(np.full(n * c, 7, np.float32))
        for scratch, call in ((rows, lambda: norm(y, x=rows)), (rows, lambda: norm(rows)), (coords, lambda: attend(y, coords=coords)),
                              (prefix, lambda: attend(y, prefix=prefix)), (rows, lambda: attend(rows))):
            be.set_scratch(scratch)
            with pytest.raises(sh.HipError) as e:
                call()
            assert e.value.status == sh.INVALID_ARGUMENT and "scratch" in str(e.value)
            assert np.all(be.download(y) == 7)
        be.set_scratch(None)
    finally:
        be.destroy()


def test_without_memory():
    """No memory for integer rows is a status; group norm and attention do without scratch, within their bounds."""
    be, rng, n, c = sh.Backend(0, sh.F32), np.random.default_rng(6), 3000, 64
    try:
        x = rng.standard_normal((n, c)).astype(np.float32)
        xb, y, z = be.upload(x), be.alloc(n * c), be.alloc(n * c)
        at, q = be.upload_i32(np.array([0, n], np.int32)), be.upload(x[:2])
        slopes, w = np.array([0.01], np.float32), rng.standard_normal((c, c)).astype(np.float32)

        def attend(y):
            be.attention_scored(q, xb, xb, y, 2, n, 1, 1, c, slopes=slopes, cap=5.0)

        def norm(y):
            be.group_norm(xb, None, None, y, n, c, 8, 1e-5, offsets=at, act="silu")

        norm(y)
        attend(z)
        exp = [be.download(y), be.download(z, 2 * c)]
        be.trim(sh.TRIM_FREE_BUFFERS)
        be.fail_alloc(0, 1 << 40)
        try:
            with pytest.raises(sh.HipError) as e:
                be.alloc_rows_int8(n, c)
            assert e.value.status == sh.OUT_OF_MEMORY
            norm(y)
            attend(z)
        finally:
            be.fail_alloc(-1, 0)
        # fp32 sums and exponentials in another order: a few of the 3,000 keys' roundings.
        np.testing.assert_allclose(be.download(y), exp[0], rtol=2 ** -20, atol=2 ** -20)
        np.testing.assert_allclose(be.download(z, 2 * c), exp[1], rtol=2 ** -16, atol=2 ** -18)
        be.fail_alloc(0, 1 << 40)
        try:
            with pytest.raises(sh.HipError) as e:
                be.group_norm(xb, w[0], None, y, n, c, 8, 1e-5)
            assert e.value.status == sh.OUT_OF_MEMORY
            with pytest.raises(sh.HipError) as e:
                be.attention_scored(q, xb, xb, z, 2, n, 1, 1, c, slopes=w[0, :1].copy())
            assert e.value.status == sh.OUT_OF_MEMORY
        finally:
            be.fail_alloc(-1, 0)
        norm(y)
        np.testing.assert_array_equal(be.download(y), exp[0])
    finally:
        be.destroy()


@pytest.fixture(scope="module")
def torch_program():
    r = subprocess.run([sys.executable, "-u", os.path.join(HERE, "int_block_with_torch.py")], capture_output=True, text=True,
                       timeout=110)
    return r.returncode, r.stdout, r.stderr[-3000:]


@pytest.mark.parametrize("what", ["tensors_and_streams", "graphs", "graphs_without_scratch", "beyond_32_bits",
                                  "two_backends_at_once"])
def test_with_torch(torch_program, what):
    rc, out, err = torch_program
    assert f"{what}: ok" in out.splitlines() and rc == 0, f"exit {rc}\n{out}\n{err}"
