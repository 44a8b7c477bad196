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


@pytest.fixture(scope="module")
def torch_program():
    r = subprocess.run([sys.executable, "-u", os.path.join(HERE, "rows_with_torch.py")], capture_output=True, text=True,
                       timeout=110)
    return r.returncode, r.stdout, r.stderr[-3000:]


@pytest.mark.parametrize("what", ["tensors_and_streams", "graphs", "two_backends_at_once", "wrap_refusals"])
def test_with_torch(torch_program, what):
    rc, out, err = torch_program
    assert f"{what}: ok" in out.splitlines() and rc == 0, f"exit {rc}\n{out}\n{err}"
