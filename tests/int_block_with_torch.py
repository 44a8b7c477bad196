"""Group norm, integer rows and attention with changed scores on a torch program's tensors, streams and graphs; run by
test_gpu_int_block.py in a process of its own.  Prints one line per check that held."""
import os
import sys

import torch  # before sparse_hip: both use the HIP runtime that torch brings

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [os.path.join(ROOT, "tests"), os.path.join(ROOT, "trellis2.c_amd")]

import numpy as np  # noqa: E402
from pytest import raises  # noqa: E402

import int_block  # noqa: E402
import sparse_hip as sh  # noqa: E402


def program():
    """A backend, a block and its inputs as torch tensors, and what the block gives on the backend's own buffers."""
    dtype, n = sh.BF16, 3000
    rng, blk = np.random.default_rng(3), int_block.IntBlock(sh.BF16)
    coords, at = int_block.voxels(n, rng)
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
    """Inputs made and outputs read on torch's streams, the backend queued between them with no wait of the host's."""
    be, blk, n, t, exp = program
    out = torch.empty((n, blk.c), dtype=torch.bfloat16, device="cuda")
    for stream in (torch.cuda.default_stream(), torch.cuda.Stream(), torch.cuda.default_stream()):
        be.set_stream(stream.cuda_stream)
        stream.wait_stream(torch.cuda.default_stream())
        with torch.cuda.stream(stream):
            kept = []
            for x in t["x"]:
                big = torch.randn((2048, 2048), device="cuda")
                big = big @ big  # the stream is busy
                x2 = x + 0 * big.reshape(-1)[:n * blk.c].reshape(n, blk.c).nan_to_num(0.0, 0.0, 0.0).to(torch.bfloat16)
                b = blk.buffers(be, n)
                b["out"] = be.wrap(out)
                blk.run(be, be.wrap(x2), be.wrap(t["coords"]), be.wrap(t["at"]), n, b)
                kept.append(out.float().cpu().numpy())
        for got, e in zip(kept, exp):
            assert np.array_equal(got, e)
        torch.cuda.synchronize()
    be.set_stream(None)


def graphs(program):
    """The block captured twice, into graphs with buffers and scratch of their own, replayed in turn with other inputs and
    eager calls of the same backend between: every replay is the eager call's result, bit for bit."""
    be, blk, n, t, exp = program
    assert be.scratch_bytes > 0
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    made = []
    for _ in range(2):
        x = t["x"][0].clone()
        out = torch.empty((n, blk.c), dtype=torch.bfloat16, device="cuda")
        b = blk.buffers(be, n)
        b["out"] = be.wrap(out)
        scratch = torch.empty(be.scratch_bytes // 4, dtype=torch.int32, device="cuda")
        xb, cb, ab, sb = be.wrap(x), be.wrap(t["coords"]), be.wrap(t["at"]), be.wrap(scratch)
        torch.cuda.synchronize()
        be.set_scratch(sb)
        with torch.cuda.stream(stream):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                blk.run(be, xb, cb, ab, n, b)
                if not made:
                    with raises(sh.HipError) as e:
                        be.alloc_rows_int8(n, 64)
                    assert e.value.status == sh.ERROR and "captured" in str(e.value)
                    with raises(sh.HipError) as e:  # gammas that are not on the device yet
                        be.group_norm(xb, np.ones(blk.c, np.float32), None, b["norm"], n, blk.c, 8, 1e-5)
                    assert e.value.status == sh.ERROR
        be.set_scratch(None)
        made.append((g, x, out, b, scratch, sb))
    for step in range(6):
        g, x, out = made[step % 2][:3]
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


def graphs_without_scratch(program):
    """Captured without scratch, group norm takes a block per group and attention all keys in one: sums in another order,
    within a few roundings of bf16 of the eager calls, and the same from replay to replay."""
    be, blk, n, t, _ = program
    stream = torch.cuda.Stream()
    be.set_stream(stream.cuda_stream)
    gen = torch.Generator().manual_seed(5)
    rows = lambda *shape: torch.randn(shape, generator=gen).to(torch.bfloat16).cuda()  # noqa: E731
    k, v, at = rows(20000, 128), rows(20000, 128), be.wrap(t["at"])
    kb, vb = be.wrap(k), be.wrap(v)
    slopes, gamma = np.array([0.01, 0.001], np.float32), np.ones(blk.c, np.float32)

    def run(x, q, y, o):
        be.group_norm(x, gamma, None, y, n, blk.c, 8, 1e-5, act="silu", offsets=at)
        be.attention_scored(q, kb, vb, o, 3, 20000, 2, 2, 64, cap=5.0, slopes=slopes, causal=True)

    def outputs():
        a = torch.zeros((n, blk.c), dtype=torch.bfloat16, device="cuda"), torch.zeros((3, 128), dtype=torch.bfloat16, device="cuda")
        return a, [be.wrap(x) for x in a]

    qs = [rows(3, 128) for _ in range(3)]
    torch.cuda.synchronize()
    exp = []
    for x, q in zip(t["x"], qs):
        a, b = outputs()
        run(be.wrap(x), be.wrap(q), *b)
        torch.cuda.synchronize()
        exp.append([o.float().cpu().numpy() for o in a])
    x, q = t["x"][0].clone(), qs[0].clone()
    a, b = outputs()
    xb, qb = be.wrap(x), be.wrap(q)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            run(xb, qb, *b)
    seen = {}
    for step in range(6):
        i = step % 3
        with torch.cuda.stream(stream):
            x.copy_(t["x"][i])
            q.copy_(qs[i])
            for o in a:
                o.zero_()
            g.replay()
            eager, eb = outputs()
            run(be.wrap(t["x"][i]), be.wrap(qs[i]), *eb)
        stream.synchronize()
        got = [o.float().cpu().numpy() for o in a]
        for o, e, other in zip(got, exp[i], eager):
            assert np.allclose(o, e, rtol=2 ** -6, atol=2 ** -8), step
            assert np.array_equal(other.float().cpu().numpy(), e), step
        for o, e in zip(got, seen.setdefault(i, got)):
            assert np.array_equal(o, e), step
    be.set_stream(None)


def beyond_32_bits(program):
    """Rows that lie more than 2^31 elements behind their buffer's start give what the same rows give alone: a group norm's
    last sequence, integer rows and their linear, keys and values of one far cache."""
    be, dev, bf = program[0], torch.device("cuda", 0), torch.bfloat16
    gen = torch.Generator().manual_seed(9)
    rows = lambda *shape: torch.randn(shape, generator=gen).to(bf).cuda()  # noqa: E731
    n, c, last = 1_200_000, 2048, 3000
    x = torch.zeros((n, c), dtype=bf, device=dev)
    x[-last:] = rows(last, c)
    tail = x[-last:].clone()
    y, alone = torch.zeros_like(x), torch.zeros_like(tail)
    at = torch.tensor([0, n - last, n], dtype=torch.int32, device=dev)
    torch.cuda.synchronize()
    xb, yb, tb, ob, ab = (be.wrap(a) for a in (x, y, tail, alone, at))
    be.group_norm(xb, None, None, yb, n, c, 32, 1e-5, act="silu", offsets=ab)
    be.group_norm(tb, None, None, ob, last, c, 32, 1e-5, act="silu")
    torch.cuda.synchronize()
    # Sums of 64 bits in another order: what a rounding of the last bit of fp32 may turn.
    far, near = y[-last:].float(), alone.float()
    assert float((far - near).abs().max()) <= 2 ** -7 * float(near.abs().max()) and float((far != near).float().mean()) < 1e-4
    assert not y[:1000].any()
    big, small = be.alloc_rows_int8(n, c), be.alloc_rows_int8(last, c)
    be.pack_rows8(xb, big, n, c)
    be.pack_rows8(tb, small, last, c)
    be.expand_rows8(big, yb, n, c)
    be.expand_rows8(small, ob, last, c)
    torch.cuda.synchronize()
    assert torch.equal(y[-last:], alone) and not y[:1000].any()
    be.rms_norm(xb, None, big, n, c, 1e-6)
    be.rms_norm(tb, None, small, last, c, 1e-6)
    weight = np.random.default_rng(4).standard_normal((64, c)).astype(np.float32) / 45
    be.linear_act(big, weight, None, yb, n, c, 64)
    be.linear_act(small, weight, None, ob, last, c, 64)
    torch.cuda.synchronize()
    assert torch.equal(y.reshape(-1)[:n * 64].reshape(n, 64)[-last:], alone.reshape(-1)[:last * 64].reshape(last, 64))
    big.free()
    del x, y
    for heads, dim, stride, m in ((2, 64, 1 << 22, 700), (1, 24, 1 << 24, 170)):
        w = heads * dim
        cache = torch.zeros((m - 1) * stride + 2 * w, dtype=bf, device=dev)
        kv = cache.as_strided((m, 2 * w), (stride, 1))
        kv.copy_(rows(m, 2 * w))
        near, q = kv.contiguous(), rows(5, w)
        a, b = torch.empty_like(q), torch.empty_like(q)
        torch.cuda.synchronize()
        fb, nb, qb = be.wrap(cache), be.wrap(near), be.wrap(q)
        more = dict(cap=9.0, causal=True, slopes=np.full(heads, 0.01, np.float32))
        be.attention_scored(qb, fb, fb, be.wrap(a), 5, m, heads, heads, dim, k_stride=stride, v_offset=w, v_stride=stride, **more)
        be.attention_scored(qb, nb, nb, be.wrap(b), 5, m, heads, heads, dim, k_stride=2 * w, v_offset=w, v_stride=2 * w, **more)
        torch.cuda.synchronize()
        # Strides beyond 2^23 leave the wide kernel: weights of few queries are whole in both.
        tol = 0 if stride <= 1 << 23 else 2 ** -7
        assert np.allclose(a.float().cpu(), b.float().cpu(), rtol=tol, atol=tol) and float(a.abs().max()) > 0.1
        del cache, kv


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


if __name__ == "__main__":
    for check in (tensors_and_streams, graphs, graphs_without_scratch, beyond_32_bits, two_backends_at_once):
        p = program()
        check(p)
        p[0].destroy()
        print(f"{check.__name__}: ok", flush=True)
