"""What transformer_block refuses it refuses before it writes: its rows stay as they were, also where they are the output."""
import numpy as np
import pytest

import sparse_hip as sh

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [sh.F32, sh.BF16])
@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("what", ["integer rows too wide", "no such activation"])
def test_refused_before_anything_is_written(monkeypatch, dtype, inplace, what):
    monkeypatch.setitem(sh.ACTS, "none of them", 9)
    wide = what == "integer rows too wide"
    be, rng, n, c, hidden = sh.Backend(0, dtype), np.random.default_rng(1), 5, 8, 131080 if wide else 64
    try:
        w = {k: rng.standard_normal(s).astype(np.float32) for k, s in (("qkv_w", (3 * c, c)), ("out_w", (c, c)),
                                                                       ("mlp0_w", (hidden, c)), ("mlp2_w", (c, hidden)))}
        x = sh.storage_round(rng.standard_normal((n, c)).astype(np.float32), dtype)
        h, at = be.upload(x), be.upload_i32(np.zeros((n, 4), np.int32))
        out = h if inplace else be.upload(np.full(n * c, 7, np.float32))
        with pytest.raises(sh.HipError) as e:
            be.transformer_block(h, at, out, n, 1, c, hidden, w, (1, 1, 1), rows8=2 if wide else 0,
                                 act="gelu_tanh" if wide else "none of them")
        assert e.value.status == sh.INVALID_ARGUMENT
        np.testing.assert_array_equal(be.download(out).reshape(n, c), x if inplace else np.full((n, c), 7))
        np.testing.assert_array_equal(be.download(h).reshape(n, c), x)
        if wide:  # as floating 8-bit rows and as rows of the type it runs
            for rows8 in (0, 1):
                be.transformer_block(h, at, out, n, 1, c, hidden, w, (1, 1, 1), rows8=rows8)
                assert np.isfinite(be.download(out)).all()
    finally:
        be.destroy()
