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
