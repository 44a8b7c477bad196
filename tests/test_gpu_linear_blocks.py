"""linear_act at sizes that take each of its block shapes, with one tile a block and with many, K in splits and not, and rows
in two parts (whole rounds of large blocks, then the rest in smaller ones, split): every type of rows against float64.  Bounds:
tests/rows64.py."""
import functools

import numpy as np
import pytest

import rows64 as ref
import sparse_hip as sh

pytestmark = pytest.mark.gpu

# What the sizes take on 256 CUs (16 and 8 bits; fp32 where it differs).
CASES = [
    (18216, 4096, 1024),  # 256 x 256 in one round, and 1,832 rows of 128 x 128 in splits
    (79523, 512, 2048),   # 256 x 256, ten tiles a block; fp32: and 5,795 rows of 192 x 256
    (60000, 256, 1536),   # 256 x 256, six tiles a block; 8 bits 128 x 128, eleven; fp32: and 5,472 rows of 64 x 128
    (20000, 256, 512),    # 192 x 256
    (40000, 512, 1002),   # 128 x 128, two channels a lane, five tiles a block; fp32: 192 x 256 and 3,136 rows of these
    (30000, 1024, 1001),  # 128 x 128, one channel a lane, four tiles a block
    (5000, 2048, 1024),   # 64 x 128; fp32 in splits
    (2000, 4096, 514),    # 64 x 128 (8 bits 128 x 128) in splits
    (3000, 4096, 257),    # 64 x 64 in splits, an odd number of channels
    (90000, 64, 33),      # 64 x 64, several tiles a block
    (66000, 256, 256),    # 128 x 128, three tiles a block; fp32: 256 x 256 and 464 rows of 64 x 64 in splits
    (33001, 520, 130),    # a last step that is not whole
]


@functools.lru_cache(maxsize=1)
def values(n, ci, co):
    rng = np.random.default_rng(n + ci + co)
    x = rng.standard_normal((n, ci), dtype=np.float32)
    w = rng.standard_normal((co, ci), dtype=np.float32) / np.float32(np.sqrt(ci))
    return x, w, rng.standard_normal(co, dtype=np.float32), rng.standard_normal((n, co), dtype=np.float32)


@pytest.mark.parametrize("from8", [False, True])
@pytest.mark.parametrize("dtype", [sh.F32, sh.F16, sh.BF16])
@pytest.mark.parametrize("n,ci,co", CASES)
def test_blocks(n, ci, co, dtype, from8):
    """Some rows in all channels, and many rows (the last 2,000 among them) in some channels."""
    x, w, b, r = values(n, ci, co)
    x, r = sh.storage_round(x, dtype), sh.storage_round(r, dtype)
    act = "gelu" if (n + ci) % 2 else "none"
    be = sh.Backend(0, dtype)
    try:
        xb, y = be.upload(x), be.upload(np.full((n, co), 7, np.float32))
        if from8:
            xb, rows = be.alloc_rows8(n, ci), xb
            be.pack_rows8(rows, xb, n, ci)
        be.linear_act(xb, w, b, y, n, ci, co, act=act, residual=be.upload(r))
        got = be.download(y).reshape(n, co)
    finally:
        be.destroy()
    rng = np.random.default_rng(1)
    rows = np.unique(np.concatenate([np.arange(300), rng.integers(0, n, 300), np.arange(n - 300, n)]))
    many = np.unique(np.concatenate([np.arange(600), rng.integers(0, n, 4000), np.arange(n - 2000, n)]))
    some = np.unique(np.concatenate([np.arange(co)[:9], rng.integers(0, co, 64), np.arange(co)[-9:]]))
    wide = (lambda a: ref.rows8(a.astype(np.float64))) if from8 else (lambda a: a.astype(np.float64))
    wv = wide(w if from8 else sh.storage_round(w, dtype))
    for at, channels in ((rows, np.arange(co)), (many, some)):
        exp, err = ref.linear_act(wide(x[at]), wv[channels], b[channels].astype(np.float64), act,
                                  r[np.ix_(at, channels)].astype(np.float64), from8)
        ref.check(got[np.ix_(at, channels)], exp, err + ref.stored(exp, dtype), f"{n} {ci} {co} {act}")
