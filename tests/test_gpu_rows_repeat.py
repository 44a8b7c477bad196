"""Calls that split their sums or keys, walk many tiles or join them give the same bits every time, with other work between."""
import numpy as np
import pytest

import sparse_hip as sh
from test_gpu_rows import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("what", ["attention", "few queries", "linear", "linear split", "linear in 8 bits", "norm to 8 bits"])
def test_same_bits(dtype, what):
    be, rng = sh.Backend(0, dtype), np.random.default_rng(7)
    try:
        if what in ("attention", "few queries"):
            nq, nk, heads, dim = (3000, 3000, 4, 64) if what == "attention" else (3, 20000, 8, 64)
            q, k, v = (be.upload(make(rng, dtype, n, heads * dim)) for n in (nq, nk, nk))
            count, call = nq * heads * dim, lambda y: be.attention(q, k, v, y, nq, nk, heads, heads, dim)
        elif what == "norm to 8 bits":
            n, c = 5003, 1024
            x, g, q8 = be.upload(make(rng, dtype, n, c)), np.ones(c, np.float32), be.alloc_rows8(n, c)

            def call(y):
                be.rms_norm(x, g, q8, n, c, 1e-6)
                be.expand_rows8(q8, y, n, c)
            count = n * c
        else:
            n, ci, co = (5, 4096, 512) if what == "linear split" else (20000, 256, 1024)
            x, w = be.upload(make(rng, dtype, n, ci)), make(rng, dtype, co, ci) / 16
            if what == "linear in 8 bits":
                q8 = be.alloc_rows8(n, ci)
                be.pack_rows8(x, q8, n, ci)
                x = q8
            count, call = n * co, lambda y: be.linear_act(x, w, None, y, n, ci, co, act="gelu")
        y, other = be.alloc(count), be.upload(np.ones(count, np.float32))
        call(y)
        first = be.download_raw(y).tobytes()
        for _ in range(4):
            be.add(other, other, y, count)
            call(y)
            assert be.download_raw(y).tobytes() == first
    finally:
        be.destroy()
