"""The row operators on a torch program's tensors, streams and graphs; run by test_gpu_rows_together.py in a process of its
own.  Prints one line per check that held."""
import os
import sys

import torch  # before sparse_hip: both use the HIP runtime that torch brings

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [os.path.join(ROOT, "tests"), os.path.join(ROOT, "trellis2.c_amd")]

import numpy as np  # noqa: E402
from pytest import raises  # noqa: E402

import rows_block  # noqa: E402
import sparse_hip as sh  # noqa: E402


def program():
    """A backend on torch's stream, a block and its inputs as torch tensors, and what the block gives on buffers."""
    dtype, n = sh.BF16, 200
    rng, blk = np.random.default_rng(3), rows_block.Block(sh.BF16)
    coords, at = rows_block.voxels(n, rng)
    xs = [sh.storage_round(rng.standard_normal((n, blk.c)).astype(np.float32), dtype) for _ in range(3)]
    be = sh.Backend(0, dtype)
    exp = []
    for x in xs:
        b = blk.buffers(be, n)
        blk.run(be, be.upload(x), be.upload_i32(coords), be.upload_i32(at), n, b)
        exp.append(be.download(b["out"]).reshape(n, blk.c))
    dev = torch.device("cuda", 0)
    t = dict(x=[torch.from_numpy(x).to(dev).to(torch.bfloat16) for x in xs], coords=torch.from_numpy(coords).to(dev),
             at=torch.from_numpy(at).to(dev))
    torch.cuda.synchronize()
    return be, blk, n, t, exp


def tensors_and_streams(program):
    """Inputs made and outputs read on torch's streams, the backend queued between them with no wait of the host's, on the
    default stream, on one of its own, and back."""
    be, blk, n, t, exp = program
    out = torch.empty((n, blk.c), dtype=torch.bfloat16, device="cuda")
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.default_stream()):
        be.set_stream(stream.cuda_stream)
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            kept = []
            for x in t["x"]:
                big = torch.randn((2048, 2048), device="cuda")
                big = big @ big  # the stream is busy
                x2 = x + 0 * big[:n, :blk.c].nan_to_num(0.0, 0.0, 0.0).to(torch.bfloat16)
                b = blk.buffers(be, n)
                b["out"] = be.wrap(out)
                blk.run(be, be.wrap(x2), be.wrap(t["coords"]), be.wrap(t["at"]), n, b)
                kept.append(out.float().cpu().numpy())
        for got, e in zip(kept, exp):
            assert np.array_equal(got, e)
        torch.cuda.synchronize()
    be.set_stream(None)
    b = blk.buffers(be, n)
    blk.run(be, be.wrap(t["x"][0]), be.wrap(t["coords"]), be.wrap(t["at"]), n, b)
    assert np.array_equal(be.download(b["out"]).reshape(exp[0].shape), exp[0])


def graphs(program):
    """The block captured twice, into graphs with buffers of their own that share the weights, replayed in turn with other
    inputs and eager calls of the same backend between; calls that would allocate are refused while capturing."""
    be, blk, n, t, exp = program
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    made = []
    for _ in range(2):
        x = t["x"][0].clone()
        out = torch.empty((n, blk.c), dtype=torch.bfloat16, device="cuda")
        b = blk.buffers(be, n)
        b["out"] = be.wrap(out)
        xb, cb, ab = be.wrap(x), be.wrap(t["coords"]), be.wrap(t["at"])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            blk.run(be, xb, cb, ab, n, b)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                blk.run(be, xb, cb, ab, n, b)
                if not made:
                    with raises(sh.HipError) as e:
                        be.alloc_rows8(n, 64)
                    assert e.value.status == sh.ERROR and "captured" in str(e.value)
                    with raises(sh.HipError) as e:
                        be.linear_act(xb, np.zeros((8, blk.c), np.float32), None, b["hid"], n, blk.c, 8)
                    assert e.value.status == sh.ERROR
        made.append((g, x, out, b))
    for step in range(6):
        g, x, out, _ = made[step % 2]
        i = step % 3
        with torch.cuda.stream(stream):
            x.copy_(t["x"][i])
            out.zero_()
            g.replay()
            b = blk.buffers(be, n)
            blk.run(be, be.wrap(t["x"][(i + 1) % 3]), be.wrap(t["coords"]), be.wrap(t["at"]), n, b)
        stream.synchronize()
        assert np.array_equal(out.float().cpu().numpy(), exp[i]), step
        assert np.array_equal(be.download(b["out"]).reshape(exp[0].shape), exp[(i + 1) % 3]), step
    be.set_stream(None)


def two_backends_at_once(program):
    """Two backends on two streams, queued in turn with no wait between: each gives its own results."""
    be, blk, n, t, exp = program
    other = sh.Backend(0, sh.BF16)
    try:
        runs = []
        for i in range(6):
            one = (be, other)[i % 2]
            b = blk.buffers(one, n)
            blk.run(one, one.wrap(t["x"][i % 3]), one.wrap(t["coords"]), one.wrap(t["at"]), n, b)
            runs.append((one, b, i % 3))
        for one, b, i in runs:
            assert np.array_equal(one.download(b["out"]).reshape(exp[0].shape), exp[i])
    finally:
        other.destroy()


def wrap_refusals(program):
    be = program[0]
    x = torch.zeros(1024, dtype=torch.bfloat16, device="cuda")
    for ptr, count in ((0, 16), (x.data_ptr() + 2, 16), (x.data_ptr(), 0), (x.data_ptr(), 1 << 40),
                       (x.cpu().data_ptr() // 16 * 16, 16)):
        out = sh.c_void_p(5)
        st = sh.LIB.trellis_sparse_hip_wrap_f32(be.ptr, ptr, count, sh.ctypes.byref(out))
        assert st == sh.INVALID_ARGUMENT and not out.value
    with raises(TypeError):
        be.wrap(x.float())
    with raises(ValueError):
        be.wrap(x.reshape(32, 32).t())
    # Freed, trimmed and used again: the memory stays the tensor's.
    buf = be.wrap(x)
    buf.free()
    be.trim(sh.TRIM_FREE_BUFFERS)
    x += 1
    assert float(x.float().sum()) == 1024.0
    # The slots take wrapped rows too.
    a, y = be.wrap(x), be.wrap(torch.empty_like(x))
    torch.cuda.synchronize()
    be.add(a, a, y, 1024)
    assert np.all(be.download(y) == 2.0)


if __name__ == "__main__":
    for check in (tensors_and_streams, graphs, two_backends_at_once, wrap_refusals):
        p = program()
        check(p)
        p[0].destroy()
        print(f"{check.__name__}: ok", flush=True)
