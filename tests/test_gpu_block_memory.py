"""What transformer_block leaves when it ends early: its intermediates go back to the pool."""
import ctypes
import resource

import numpy as np
import pytest

import rows_block
import sparse_hip as sh
from test_gpu_rows_together import block_args

pytestmark = pytest.mark.gpu


def virtual_bytes():
    with open("/proc/self/statm") as f:
        return int(f.read().split()[0]) * resource.getpagesize()


def test_no_host_memory_for_packed_weights():
    """The packed copy of the first weights (12 GiB) does not fit into the address space that is left (4 GiB more than there
    is): OUT_OF_MEMORY, and the intermediates are in the pool, from which a trim releases them."""
    be, n = sh.Backend(0, sh.F32), 3
    heads, dim, hidden = 256, 128, 64
    c = heads * dim
    try:
        # A call before, so that nothing else is loaded under the limit.
        blk = rows_block.Block(sh.F32)
        x, out = be.alloc(n * blk.c), be.alloc(n * blk.c)
        cb = be.upload_i32(np.zeros((n, 4), np.int32))
        be.transformer_block(x, cb, out, n, **block_args(blk))
        x, out = be.upload(np.ones((n, c), np.float32)), be.alloc(n * c)
        weights = np.zeros(3 * c * c, np.float32)  # pages that nothing touches
        names = [f[0] for f in sh.BlockDesc._fields_ if f[1] is sh.c_void_p]
        at = {k: weights.ctypes.data if k in ("qkv_w", "out_w", "mlp0_w", "mlp2_w") else None for k in names}
        d = sh.BlockDesc(ctypes.sizeof(sh.BlockDesc), heads, dim, hidden, 0, 0, (ctypes.c_int32 * 3)(1, 1, 1), 0, 1e-6, 0.0,
                         10000.0, *(at[k] for k in names))
        be.synchronize()
        be.trim(sh.TRIM_FREE_BUFFERS)
        soft, hard = resource.getrlimit(resource.RLIMIT_AS)
        resource.setrlimit(resource.RLIMIT_AS, (virtual_bytes() + (4 << 30), hard))
        try:
            st = sh.LIB.trellis_sparse_hip_transformer_block(be.ptr, x.handle, cb.handle, None, None, 1, ctypes.byref(d),
                                                             out.handle, n)
        finally:
            resource.setrlimit(resource.RLIMIT_AS, (soft, hard))
        assert st == sh.OUT_OF_MEMORY
        assert be.trim(sh.TRIM_FREE_BUFFERS) >= 4 * n * (c + 3 * c + hidden)
        del weights
        blk_out = be.alloc(n * blk.c)
        be.transformer_block(be.alloc(n * blk.c), cb, blk_out, n, **block_args(blk))
    finally:
        be.destroy()
