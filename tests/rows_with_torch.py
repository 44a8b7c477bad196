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


def split_graphs(program):
    """Calls that split through scratch, captured into two graphs with scratch of their own: every replay is the eager call's
    result, bit for bit, with eager calls through the pool's scratch between; without scratch they are captured unsplit.
    While a stream is captured no other can be set, and stage times are not recorded."""
    be = program[0]
    stream, other = torch.cuda.Stream(), torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    be.profile(True)
    gen = torch.Generator().manual_seed(5)
    rows = lambda *shape: torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()  # noqa: E731
    w = np.random.default_rng(1).standard_normal((512, 4096)).astype(np.float32) / 64
    k, v = rows(20000, 128), rows(20000, 128)
    xs = [(rows(2, 4096), rows(3, 128)) for _ in range(3)]
    kb, vb = be.wrap(k), be.wrap(v)

    def run(x, q, y, o):
        be.linear_act(x, w, None, y, 2, 4096, 512, act="gelu")
        be.attention(q, kb, vb, o, 3, 20000, 2, 2, 64)

    def outputs():
        t = torch.empty((2, 512), dtype=torch.bfloat16, device="cuda"), torch.empty((3, 128), dtype=torch.bfloat16, device="cuda")
        return t, [be.wrap(a) for a in t]

    torch.cuda.synchronize()
    exp = []
    for x, q in xs:
        t, b = outputs()
        run(be.wrap(x), be.wrap(q), *b)
        torch.cuda.synchronize()
        exp.append([a.float().cpu().numpy() for a in t])
    made = []
    for with_scratch in (True, True, False):
        x, q = (a.clone() for a in xs[0])
        t, b = outputs()
        scratch = torch.empty(be.scratch_bytes // 4, dtype=torch.int32, device="cuda")
        xb, qb, sb = be.wrap(x), be.wrap(q), be.wrap(scratch)
        torch.cuda.synchronize()
        be.set_scratch(sb if with_scratch else None)
        with torch.cuda.stream(stream):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                run(xb, qb, *b)
                for back in (other.cuda_stream, 0, None):
                    with raises(sh.HipError) as e:
                        be.set_stream(back)
                    assert e.value.status == sh.ERROR
        be.set_scratch(None)
        made.append((g, x, q, t, (b, scratch, xb, qb, sb)))
    for step in range(9):
        g, x, q, t, _ = made[step % 3]
        i = step // 3
        with torch.cuda.stream(stream):
            x.copy_(xs[i][0])
            q.copy_(xs[i][1])
            for a in t:
                a.zero_()
            g.replay()
            eager, b = outputs()
            run(be.wrap(xs[(i + 1) % 3][0]), be.wrap(xs[(i + 1) % 3][1]), *b)
        stream.synchronize()
        for got, e in zip(t, exp[i]):
            got = got.float().cpu().numpy()
            # Unsplit sums: another order, within a few roundings of bf16.
            assert np.array_equal(got, e) if step % 3 < 2 else np.allclose(got, e, rtol=2 ** -6, atol=2 ** -8), step
        for got, e in zip(eager, exp[(i + 1) % 3]):
            assert np.array_equal(got.float().cpu().numpy(), e), step
    be.profile(False)
    be.set_stream(None)


def beyond_32_bits(program):
    """Rows that lie more than 2^31 elements behind their buffer's start: keys and values far apart (both kernels), a norm,
    8-bit rows, a linear and a rotary over 1.2 M rows of 2,048; the last rows are what the same rows give alone."""
    be, dev = program[0], torch.device("cuda", 0)
    bf = torch.bfloat16
    gen = torch.Generator().manual_seed(9)
    rows = lambda *shape: torch.randn(shape, generator=gen).to(bf).cuda()  # noqa: E731
    for heads, dim, stride, n in ((2, 64, 1 << 22, 700), (1, 24, 1 << 24, 170)):
        w = heads * dim
        far = torch.zeros((n - 1) * stride + 2 * w, dtype=bf, device=dev)
        kv = far.as_strided((n, 2 * w), (stride, 1))
        kv.copy_(rows(n, 2 * w))
        near, q = kv.contiguous(), rows(n, w)
        a, b = torch.empty_like(q), torch.empty_like(q)
        torch.cuda.synchronize()
        fb, nb, qb = be.wrap(far), be.wrap(near), be.wrap(q)
        be.attention(qb, fb, fb, be.wrap(a), n, n, heads, heads, dim, k_stride=stride, v_offset=w, v_stride=stride)
        be.attention(qb, nb, nb, be.wrap(b), n, n, heads, heads, dim, k_stride=2 * w, v_offset=w, v_stride=2 * w)
        out = be.download(be.wrap(a))
        # Strides beyond 2^23 leave the wide kernel: its weights are rounded, 2^-8 of sum p |v| <= 1, and both outputs are.
        tol = 0 if stride <= 1 << 23 else 2 ** -7
        assert np.allclose(out, be.download(be.wrap(b)), rtol=tol, atol=tol) and np.abs(out).max() > 0.1
        del far, kv
    n, c, last = 1_200_000, 2048, 64
    x = torch.zeros((n, c), dtype=bf, device=dev)
    x[-last:] = rows(last, c)
    tail = x[-last:].clone()
    y = torch.zeros_like(x)
    coords = torch.randint(0, 64, (n, 4), dtype=torch.int32, generator=gen).cuda()
    end = coords[-last:].clone()
    weight = np.random.default_rng(4).standard_normal((64, c)).astype(np.float32) / 45
    torch.cuda.synchronize()
    xb, yb, tb, cb, eb = (be.wrap(t) for t in (x, y, tail, coords, end))
    alone = be.alloc(last * c)

    def same(width=c):
        torch.cuda.synchronize()
        got = y.reshape(-1)[:n * width].reshape(n, width)
        assert np.array_equal(got[-last:].float().cpu().numpy(), be.download(alone)[:last * width].reshape(last, width))
        assert not got[:1000].any()

    be.rms_norm(xb, None, yb, n, c, 1e-6, residual=xb)
    be.rms_norm(tb, None, alone, last, c, 1e-6, residual=tb)
    same()
    big8, small8 = be.alloc_rows8(n, c), be.alloc_rows8(last, c)
    be.rms_norm(xb, None, big8, n, c, 1e-6)
    be.rms_norm(tb, None, small8, last, c, 1e-6)
    be.expand_rows8(big8, yb, n, c)
    be.expand_rows8(small8, alone, last, c)
    same()
    be.rotary(xb, cb, yb, n, 16, 128, (21, 21, 21), 10000.0, eps=1e-6)
    be.rotary(tb, eb, alone, last, 16, 128, (21, 21, 21), 10000.0, eps=1e-6)
    same()
    for a, b in ((xb, tb), (big8, small8)):
        be.linear_act(a, weight, None, yb, n, c, 64)
        be.linear_act(b, weight, None, alone, last, c, 64)
        torch.cuda.synchronize()
        got = y.reshape(-1)[:n * 64].reshape(n, 64)[-last:].float().cpu().numpy()
        # Other blocks and splits: sums of 2,048 in another order, 8 sqrt(2048) 2^-24 of 4 at most, and a rounding to bf16.
        assert np.allclose(got, be.download(alone)[:last * 64].reshape(last, 64), rtol=2 ** -7, atol=1e-4)


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
    for check in (tensors_and_streams, graphs, split_graphs, beyond_32_bits, two_backends_at_once,
                  wrap_refusals):
        p = program()
        check(p)
        p[0].destroy()
        print(f"{check.__name__}: ok", flush=True)
