"""Scratch that the caller gives: what may not lie in it, and which buffer it is."""
import ctypes

import numpy as np
import pytest

import rows_block
import sparse_hip as sh
from test_gpu_rows import make, refused
from test_gpu_rows_together import block_args

pytestmark = pytest.mark.gpu


def attention_of_offsets(be, q, k, v, y, nq, nk, q_at, k_at, seqs, heads, dim):
    """The call itself: buffers of offsets may be longer than the sequences need."""
    d = sh.AttentionDesc(ctypes.sizeof(sh.AttentionDesc), heads, heads, dim)
    be._check(sh.LIB.trellis_sparse_hip_attention(be.ptr, q.handle, k.handle, v.handle, y.handle, nq, nk, q_at.handle,
                                                  k_at.handle, seqs, ctypes.byref(d)), "attention")


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_offsets_in_the_scratch(dtype):
    """Offsets are read while other blocks write the scratch: refused where the call takes it, and the output as it was;
    fine where it does not, or lies elsewhere."""
    be, rng, nk = sh.Backend(0, dtype), np.random.default_rng(1), 9000
    try:
        q, k, v = (be.upload(make(rng, dtype, m, 128)) for m in (2, nk, nk))
        at = np.zeros(1 << 20, np.int32)
        at[:3] = 0, 1, 2
        kat = at.copy()
        kat[:3] = 0, 4000, nk
        qo, ko, small_q, small_k = (be.upload_i32(a) for a in (at, kat, at[:3], kat[:3]))
        y = be.alloc(2 * 128)
        attention_of_offsets(be, q, k, v, y, 2, nk, qo, ko, 2, 2, 64)
        exp = be.download(y)
        assert 0 < be.scratch_bytes <= 4 * at.size
        for scratch, a, b in ((qo, qo, small_k), (ko, small_q, ko), (qo, qo, qo)):
            be.set_scratch(scratch)
            y = be.upload(np.full(2 * 128, 7, np.float32))
            refused(sh.INVALID_ARGUMENT, attention_of_offsets, be, q, k, v, y, 2, nk, a, b, 2, 2, 64)
            assert np.all(be.download(y) == 7)
        assert np.array_equal(be.download_i32(qo), at) and np.array_equal(be.download_i32(ko), kat)
        be.set_scratch(small_q)  # too small: the pool's serves
        attention_of_offsets(be, q, k, v, y, 2, nk, small_q, small_k, 2, 2, 64)
        assert np.array_equal(be.download(y), exp)
        be.set_scratch(qo)
        attention_of_offsets(be, q, k, v, y, 2, nk, small_q, small_k, 2, 2, 64)
        assert np.array_equal(be.download(y), exp)
    finally:
        be.destroy()


def wrap_again(be, buf):
    """Another buffer over a buffer's memory, as int32 (a buffer's first field is its address)."""
    h = sh.c_void_p()
    at = ctypes.cast(buf.handle, ctypes.POINTER(ctypes.c_void_p))[0]
    be._check(sh.LIB.trellis_sparse_hip_wrap_i32(be.ptr, at, buf.count, ctypes.byref(h)), "wrap")
    return sh.Buffer(be, h, buf.count)


def test_another_buffer_over_the_scratch():
    """Freeing another buffer over the same memory leaves the scratch set; freeing the buffer that it is unsets it."""
    be, rng = sh.Backend(0, sh.BF16), np.random.default_rng(2)
    try:
        w = make(rng, sh.BF16, 512, 4096)
        x, y = be.upload(make(rng, sh.BF16, 1, 4096)), be.alloc(512)
        be.linear_act(x, w, None, y, 1, 4096, 512)
        exp, need = be.download(y), be.scratch_bytes
        assert need > 0
        words = np.full(need // 4, 7, np.int32)
        memory = be.upload_i32(words)
        scratch, other = wrap_again(be, memory), wrap_again(be, memory)
        be.set_scratch(scratch)
        other.free()
        be.linear_act(x, w, None, y, 1, 4096, 512)
        assert np.array_equal(be.download(y), exp) and not np.array_equal(be.download_i32(memory), words)
        memory = be.upload_i32(words)
        scratch, other = wrap_again(be, memory), wrap_again(be, memory)
        be.set_scratch(scratch)
        scratch.free()
        be.linear_act(x, w, None, y, 1, 4096, 512)
        assert np.array_equal(be.download(y), exp) and np.array_equal(be.download_i32(memory), words)
    finally:
        be.destroy()


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_block_with_rows_in_the_scratch(dtype):
    """The block's first linear writes its partial sums while h, the coordinates and the offsets are still to be read:
    none of the block's buffers may be the scratch, and beside it they give what they give without."""
    be, rng, n = sh.Backend(0, dtype), np.random.default_rng(3), 40
    try:
        blk = rows_block.Block(dtype, heads=16, dim=64, hidden=256)
        coords, at = rows_block.voxels(n, rng)
        x = sh.storage_round(rng.standard_normal((n, blk.c)).astype(np.float32), dtype)
        xb, cb, ab, out = be.upload(x), be.upload_i32(coords), be.upload_i32(at), be.alloc(n * blk.c)

        def block(h=xb, coords=cb, offsets=ab, y=out):
            be.transformer_block(h, coords, y, n, offsets=offsets, **block_args(blk))

        block()
        exp, need = be.download(out), be.scratch_bytes
        assert need > 0
        big = be.alloc(max(need, x.size * 4))
        big_i32 = be.upload_i32(np.pad(coords.ravel(), (0, need // 4)))
        be.set_scratch(big)
        for more in (dict(h=big), dict(y=big), dict(h=big, y=big)):
            refused(sh.INVALID_ARGUMENT, block, **more)
        be.set_scratch(big_i32)
        refused(sh.INVALID_ARGUMENT, block, coords=big_i32)
        assert np.array_equal(be.download_i32(big_i32)[:4 * n], coords.ravel())
        be.set_scratch(ab)
        refused(sh.INVALID_ARGUMENT, block)
        be.set_scratch(cb)
        refused(sh.INVALID_ARGUMENT, block)
        be.set_scratch(big)
        block()
        assert np.array_equal(be.download(out), exp)
    finally:
        be.destroy()
