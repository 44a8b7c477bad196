"""The row operators as a transformer block over voxel rows uses them: stage by stage on the backend's buffers, and on a
torch program's own tensors, streams and graphs.  The latter runs in a process of its own (rows_with_torch.py): a process
that uses both imports torch first, so that both take the HIP runtime that torch brings."""
import os
import subprocess
import sys

import numpy as np
import pytest

import rows64 as ref
import rows_block
import sparse_hip as sh

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
def test_block_stage_by_stage(dtype):
    """Every stage against float64 on what the stage before it left in its buffer, with that stage's own bound."""
    be, rng, n = sh.Backend(0, dtype), np.random.default_rng(1), 333
    try:
        blk = rows_block.Block(dtype)
        coords, at = rows_block.voxels(n, rng)
        x = sh.storage_round(rng.standard_normal((n, blk.c)).astype(np.float32), dtype).astype(np.float64)
        xb, b = be.upload(x), blk.buffers(be, n)
        cb, ab = be.upload_coords(coords), be.upload_i32(at)
        blk.run(be, xb, cb, ab, n, b)

        def got(name, m):
            if name in ("n2", "hid8"):
                y = be.alloc(n * m)
                be.expand_rows8(b[name], y, n, m)
                return be.download(y).reshape(n, m).astype(np.float64)
            return be.download(b[name]).reshape(n, m).astype(np.float64)

        c, hid, heads, dim = blk.c, blk.hidden, blk.heads, blk.dim
        d = lambda a: a.astype(np.float64)  # noqa: E731
        e = ref.rms_norm(x, blk.g1, 1e-6)
        n1 = got("n1", c)
        ref.check(n1, e, ref.rms_slack(c) * np.abs(e) + ref.stored(e, dtype), "norm")
        # The linear's own output was turned in place: v is as it left it, q and k are the rotary of it rounded.
        qkv = got("qkv", 3 * c)
        e, t = ref.linear_act(n1, d(blk.wqkv), d(blk.bqkv), "none", None)
        t = t + ref.stored(e, dtype)
        ref.check(qkv[:, 2 * c:], e[:, 2 * c:], t[:, 2 * c:], "v")
        two = be.alloc(n * 3 * c)
        be.linear_act(b["n1"], blk.wqkv, blk.bqkv, two, n, c, 3 * c)
        z = be.download(two).reshape(n, 3 * c)[:, :2 * c].reshape(n, 2 * heads, dim)
        e, t = ref.rotary(d(z), coords, (5, 5, 5), 10000.0, False, d(blk.gqk), 1e-6)
        ref.check(qkv[:, :2 * c].reshape(e.shape), e, t + ref.stored(e, dtype), "q and k")
        q, k, v = (qkv[:, i * c:(i + 1) * c].reshape(n, heads, dim) for i in range(3))
        e, t, _ = ref.attention(q, k, v, dim ** -0.5, 1, at, at, ref.HALF[dtype])
        att = got("att", c)
        ref.check(att.reshape(e.shape), e, t + ref.stored(e, dtype), "attention")
        e, t = ref.linear_act(att, d(blk.wo), d(blk.bo), "none", x)
        h = got("h", c)
        ref.check(h, e, t + ref.stored(e, dtype), "first half")
        e = ref.rms_norm(h, blk.g2, 1e-6)
        n2 = got("n2", c)
        ref.check(n2, e, ref.rows8_slack(e, ref.rms_slack(c) * np.abs(e)) + ref.stored(n2, dtype), "norm to 8 bits")
        e, t = ref.linear_act(n2, ref.rows8(d(blk.w1)), d(blk.b1), "gelu_tanh", None, from8=True)
        hidden = got("hid", hid)
        ref.check(hidden, e, t + ref.stored(e, dtype), "hidden")
        hid8 = got("hid8", hid)
        assert np.array_equal(hid8, sh.storage_round(ref.rows8(hidden), dtype))
        e, t = ref.linear_act(ref.rows8(hidden), ref.rows8(d(blk.w2)), d(blk.b2), "none", h, from8=True)
        ref.check(got("out", c), e, t + ref.stored(e, dtype), "second half")
        be.free_map(cb)
    finally:
        be.destroy()


def block_args(blk):
    w = dict(norm1_gamma=blk.g1, qkv_w=blk.wqkv, qkv_b=blk.bqkv, qk_gamma=blk.gqk, out_w=blk.wo, out_b=blk.bo,
             norm2_gamma=blk.g2, mlp0_w=blk.w1, mlp0_b=blk.b1, mlp2_w=blk.w2, mlp2_b=blk.b2)
    return dict(heads=blk.heads, head_dim=blk.dim, hidden=blk.hidden, weights=w, pairs=(5, 5, 5), qk_eps=1e-6)


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("rows8", [False, True])
def test_block_in_one_call(dtype, rows8):
    """transformer_block gives the very bits of the calls that it stands for, also over its own input, with one sequence
    and with two, rows that are in none (no attention there), from an int32 buffer of coordinates and from a device map."""
    be, rng, n = sh.Backend(0, dtype), np.random.default_rng(5), 270
    try:
        blk = rows_block.Block(dtype)
        c, w, hid = blk.c, 3 * blk.c, blk.hidden
        coords, at = rows_block.voxels(n, rng)
        x = sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype)
        xb, cb, dm, ab = be.upload(x), be.upload_i32(coords), be.upload_coords(coords), be.upload_i32(at)
        short = be.upload_i32(np.array([0, 100, 230], np.int32))
        for offsets in (None, ab, short):
            rows = be.upload(np.zeros((n, c), np.float32))
            qkv, mid, hidden, out = (be.alloc(n * m) for m in (w, c, hid, c))
            dirt = be.upload(np.full((n, c), np.nan, np.float32))
            dirt.free()  # what an intermediate's block held before shows nowhere
            rows8b, hid8 = be.alloc_rows8(n, c), be.alloc_rows8(n, hid)
            normed = rows8b if rows8 else be.alloc(n * c)
            be.rms_norm(xb, blk.g1, normed, n, c, 1e-6)
            be.linear_act(normed, blk.wqkv, blk.bqkv, qkv, n, c, w)
            be.rotary(qkv, cb, qkv, n, 2 * blk.heads, blk.dim, (5, 5, 5), gamma=blk.gqk, eps=1e-6, x_stride=w, y_stride=w)
            be.attention(qkv, qkv, qkv, rows, n, n, blk.heads, blk.heads, blk.dim, q_offsets=offsets, kv_offsets=offsets,
                         q_stride=w, k_offset=c, k_stride=w, v_offset=2 * c, v_stride=w)
            if rows8:
                be.pack_rows8(rows, rows8b, n, c)
            be.linear_act(rows8b if rows8 else rows, blk.wo, blk.bo, mid, n, c, c, residual=xb)
            be.rms_norm(mid, blk.g2, normed, n, c, 1e-6)
            be.linear_act(normed, blk.w1, blk.b1, hidden, n, c, hid, act="gelu_tanh")
            if rows8:
                be.pack_rows8(hidden, hid8, n, hid)
            be.linear_act(hid8 if rows8 else hidden, blk.w2, blk.b2, out, n, hid, c, residual=mid)
            exp = be.download(out)
            assert np.isfinite(exp).all() and np.abs(exp - x.ravel()).max() > 0.1
            got = be.alloc(n * c)
            be.transformer_block(xb, cb, got, n, rows8=rows8, offsets=offsets, **block_args(blk))
            assert np.array_equal(be.download(got), exp)
            over = be.upload(x)
            be.transformer_block(over, dm, over, n, rows8=rows8, offsets=offsets, **block_args(blk))
            assert np.array_equal(be.download(over), exp)
        be.free_map(dm)
    finally:
        be.destroy()


def test_block_refusals():
    be, n = sh.Backend(0, sh.BF16), 40
    try:
        blk = rows_block.Block(sh.BF16)
        x, out, cb = be.alloc(n * blk.c), be.alloc(n * blk.c), be.upload_i32(np.zeros((n, 4), np.int32))
        args = block_args(blk)

        def refuse(status=sh.INVALID_ARGUMENT, **more):
            a = {**args, **{k: v for k, v in more.items() if k in args}}
            h, co, o, m = (more.get(k, v) for k, v in (("h", x), ("coords", cb), ("out", out), ("n", n)))
            rest = {k: v for k, v in more.items() if k not in args and k not in ("h", "coords", "out", "n")}
            with pytest.raises(sh.HipError) as e:
                be.transformer_block(h, co, o, m, **a, **rest)
            assert e.value.status == status, (more, e.value)

        be.transformer_block(x, cb, out, n, **args)
        refuse(n=0)
        refuse(n=n + 1)
        refuse(heads=0)
        refuse(head_dim=0)
        refuse(hidden=0)
        refuse(eps=0.0)
        refuse(pairs=(9, 9, 9))
        refuse(weights={**args["weights"], "out_w": None})
        refuse(coords=be.upload_i32(np.zeros((n - 1, 4), np.int32)))
        refuse(offsets=x)
        refuse(h=cb)
        refuse(out=cb)
        refuse(sh.NOT_IMPLEMENTED, heads=8, head_dim=12, pairs=(2, 2, 2), weights={**args["weights"], "qk_gamma": None})
        with pytest.raises(TypeError):
            be.transformer_block(x, cb, out, n, **{**args, "weights": {**args["weights"], "qkv": blk.wqkv}})
        st = sh.LIB.trellis_sparse_hip_transformer_block(be.ptr, x.handle, cb.handle, None, None, 1,
                                                         sh.ctypes.byref(sh.BlockDesc()), out.handle, n)
        assert st == sh.INVALID_ARGUMENT
        be.trim(sh.TRIM_FREE_BUFFERS)
        for after in range(3):
            be.fail_alloc(after)
            try:
                refuse(sh.OUT_OF_MEMORY)
            finally:
                be.fail_alloc(-1)
            be.trim(sh.TRIM_FREE_BUFFERS)
        be.transformer_block(x, cb, out, n, **args)
    finally:
        be.destroy()


@pytest.fixture(scope="module")
def torch_program():
    r = subprocess.run([sys.executable, "-u", os.path.join(HERE, "rows_with_torch.py")], capture_output=True, text=True,
                       timeout=110)
    return r.returncode, r.stdout, r.stderr[-3000:]


@pytest.mark.parametrize("what", ["tensors_and_streams", "graphs", "split_graphs", "beyond_32_bits", "two_backends_at_once",
                                  "wrap_refusals"])
def test_with_torch(torch_program, what):
    rc, out, err = torch_program
    assert f"{what}: ok" in out.splitlines() and rc == 0, f"exit {rc}\n{out}\n{err}"
