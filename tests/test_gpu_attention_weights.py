"""Attention where its softmax is extreme: many keys whose weights are small beside the largest, and the largest scales."""
import numpy as np
import pytest

import rows64 as ref
import sparse_hip as sh
from test_gpu_rows import refused

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("nq", [1, 40, 3000, 70000])
@pytest.mark.parametrize("below", [17.375, 17.0, 13.0])
@pytest.mark.parametrize("value", [0, 2])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_weights(dtype, nq, below, value, first):
    """One key of score 0 with the value 0 or 2, and 80,000 of -17.375 (weights of 2^-25.07), -17 or -13 with the value 1:
    split over the keys and not (70,000 queries), the largest met first or last.  With S = 80,000 exp(-below) the exact result
    is (value + S) / (1 + S).

    A weight is rounded by half a step relative, or by 2^-32 of the largest where fp16 has no finer steps; all of them
    alike here, so the errors add up: (half a step + 4 E below) S + 80,000 x 2^-32 beside weights that sum to 1 + S.  A sum
    of N terms one after the other takes N roundings, each at most E of the sum, and of equal terms all may be the same way:
    with at least one key at a time N = n for the values' products; a lane adds a quarter of the weights: n / 4.  (The value 0
    shows the small weights alone: weights that fp16 loses leave nothing of S / (1 + S) = 0.0023, of which this is 1 %.)"""
    be, n, dim = sh.Backend(0, dtype), 80001, 32
    try:
        q, k, v = np.zeros((nq, dim), np.float32), np.zeros((n, dim), np.float32), np.ones((n, dim), np.float32)
        q[:, 0], k[:, 0] = 1, -below
        top = 0 if first else n - 1
        k[top, 0], v[top] = 0, value
        y = be.alloc(nq * dim)
        be.attention(be.upload(q), be.upload(k), be.upload(v), y, nq, n, 1, 1, dim, scale=1.0)
        s = (n - 1) * np.exp(-below)
        exp = np.full(nq * dim, (value + s) / (1 + s))
        half = ref.HALF[dtype] if dtype != sh.F32 else 0.0
        err = ((half + 4 * ref.E * below) * s + (80000 * 2.0 ** -32 if dtype == sh.F16 else 0.0)) / (1 + s)
        err = err + 1.25 * n * ref.E * exp
        ref.check(be.download(y), exp, err + ref.stored(exp, dtype), "y")
    finally:
        be.destroy()


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
def test_largest_scales(dtype):
    """The kernels' scale is log2(e) times the caller's: refused where fp32 has no such number (scores of 0 would be NaN),
    one-hot weights just below that."""
    be = sh.Backend(0, dtype)
    try:
        q = be.upload(np.eye(2, 32, dtype=np.float32))
        k, v = be.upload(np.eye(2, 32, dtype=np.float32)), be.upload(np.arange(64, dtype=np.float32).reshape(2, 32))
        y = be.alloc(64)
        for scale in (2.4e38, -2.4e38, float(np.finfo(np.float32).max)):
            refused(sh.INVALID_ARGUMENT, be.attention, q, k, v, y, 2, 2, 1, 1, 32, scale=scale)
        be.attention(q, k, v, y, 2, 2, 1, 1, 32, scale=2.3e38)
        assert np.array_equal(be.download(y), np.arange(64))
    finally:
        be.destroy()


@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("nq,nk,heads,kv_heads,dim", [(1, 300, 2, 2, 64), (3, 20000, 4, 1, 64), (20, 700, 6, 2, 32),
                                                      (64, 64, 3, 3, 96), (500, 900, 2, 2, 128), (1500, 1500, 2, 2, 64)])
def test_few_queries_cost_no_precision(dtype, nq, nk, heads, kv_heads, dim):
    """Nothing but fp32's errors and the output's one rounding: weights of 16 bits are in two parts, the first cut, so that
    up to a step is left, 2 HALF of the weight, and the second rounded by half a step of that: 2 HALF^2 (and 2^-31 of the
    largest at most where fp16 has no finer steps)."""
    be, rng = sh.Backend(0, dtype), np.random.default_rng(nq + nk)
    try:
        q, k, v = (sh.storage_round(rng.standard_normal((n, h, dim)).astype(np.float32), dtype)
                   for n, h in ((nq, heads), (nk, kv_heads), (nk, kv_heads)))
        y = be.alloc(nq * heads * dim)
        be.attention(be.upload(q), be.upload(k), be.upload(v), y, nq, nk, heads, kv_heads, dim)
        half = ref.E if dtype == sh.F32 else 2 * ref.HALF[dtype] ** 2
        exp, err, _ = ref.attention(*(a.astype(np.float64) for a in (q, k, v)), dim ** -0.5, heads // kv_heads, [0, nq],
                                    [0, nk], half)
        if dtype == sh.F16:
            err = err + 2.0 ** -31 * nk * np.abs(v).max()
        ref.check(be.download(y).reshape(exp.shape), exp, err + ref.stored(exp, dtype), "y")
    finally:
        be.destroy()
