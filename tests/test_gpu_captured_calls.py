"""The slots and the other calls while the caller's stream is captured into a graph: what allocates nothing is captured, and
what is refused leaves the capture as it was."""
import numpy as np
import pytest

import sparse_hip as sh
from hip_capture import Captured
from test_gpu_rows import make

pytestmark = pytest.mark.gpu


def test_conv_whose_rows_would_be_ordered_next():
    """A rulebook's rows are brought into the order of their masks once its convs' work pays for that, which takes memory: a
    captured conv takes the order that there is, the same bits, and leaves the ordering to the next eager one."""
    be, rng = sh.Backend(0, sh.BF16), np.random.default_rng(1)
    side, c = 34, 256
    coords = np.stack(np.meshgrid([0], *[np.arange(side)] * 3, indexing="ij"), -1).reshape(-1, 4).astype(np.int32)
    n = len(coords)
    assert n * c * c < 4e9 < 2 * n * c * c  # the first conv leaves the rows, the second orders them
    cap = None
    try:
        rb = be.build_rulebook(coords)
        w = (rng.standard_normal((c, 27, c)) / 83).astype(np.float32)
        xs = [be.upload(make(rng, sh.BF16, n, c)) for _ in range(2)]
        x, out, eager = be.alloc(n * c), be.alloc(n * c), be.alloc(n * c)
        zeros = be.upload(np.zeros((n, c), np.float32))
        cap = Captured(be)
        be.add(xs[0], zeros, x, n * c)
        be.conv(rb, x, w, None, out, c, c)
        with cap.capture():
            be.conv(rb, x, w, None, out, c, c)
        for step in range(6):
            be.add(xs[step % 2], zeros, x, n * c)
            be.add(zeros, zeros, out, n * c)
            cap.replay()
            be.conv(rb, x, w, None, eager, c, c)  # (the first of these orders the rows)
            assert np.array_equal(be.download(out), be.download(eager)), step
        assert be.download(out).any()
    finally:
        if cap is not None:
            cap.close()
        be.destroy()


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_calls_that_wait_are_refused(dtype):
    """Downloads and whatever else waits for the stream: ERROR, while the calls around them are captured and replayed."""
    be, rng, n, c = sh.Backend(0, dtype), np.random.default_rng(2), 70, 64
    cap = None
    try:
        coords = np.stack([np.zeros(n), np.arange(n), np.arange(n), np.arange(n)], 1).astype(np.int32)
        rb, dm = be.build_rulebook(coords), be.upload_coords(coords)
        logits = be.upload(np.ones((n, 8), np.float32))
        at, fine, parent, sub = (be.upload_i32(a) for a in (coords, np.zeros((8 * n, 4)), np.zeros(8 * n), np.zeros(8 * n)))
        be.build_c2s_map_into(at, logits, n, fine, parent, sub)  # (its scratch's event is of another stream)
        xs = [make(rng, dtype, n, c) for _ in range(2)]
        x, a, y = (be.upload(xs[0]) for _ in range(3))
        sources = [be.upload(v) for v in xs]
        zeros, g = be.upload(np.zeros((n, c), np.float32)), np.ones(c, np.float32)
        cap = Captured(be)
        be.rms_norm(x, g, a, n, c, 1e-6)
        be.event(0)
        be.pairs(rb)
        be.neighbors(rb)
        waits = [be.synchronize, lambda: be.download(a), lambda: be.download_raw(a), lambda: be.download_i32(at),
                 lambda: be.download_c2s_coords(dm), lambda: be.trim(sh.TRIM_FREE_BUFFERS), lambda: be.trim(sh.TRIM_WEIGHTS),
                 lambda: be.build_c2s_map_into(at, logits, n, fine, parent, sub), lambda: be.rulebook_stats(rb),
                 lambda: be.pairs(rb), lambda: be.neighbors(rb), be.profile_read, lambda: be.event(1), lambda: be.elapsed(0, 0)]
        with cap.capture():
            be.rms_norm(x, g, a, n, c, 1e-6)
            for i, wait in enumerate(waits):
                with pytest.raises(sh.HipError) as e:
                    wait()
                assert e.value.status == sh.ERROR and "captured" in str(e.value), i
            be.add(a, a, y, n * c)
        for step in range(4):
            be.add(sources[step % 2], zeros, x, n * c)
            cap.replay()
            got = be.download(y)
            eager = be.alloc(n * c)
            be.rms_norm(sources[step % 2], g, eager, n, c, 1e-6)
            be.add(eager, eager, eager, n * c)
            assert np.array_equal(got, be.download(eager)) and got.any(), step
        be.build_c2s_map_into(at, logits, n, fine, parent, sub)
        for wait in waits:
            wait()
    finally:
        if cap is not None:
            cap.close()
        be.destroy()
