"""The attention block of a sparse U-Net over voxel rows with its products in 8-bit integers, as a program runs it."""
import numpy as np

import sparse_hip as sh


class IntBlock:
    """x + Wo attention(Wqkv groupnorm(x)): the norm over each object's rows, rows to 8-bit integers before both products,
    scores capped and lowered by the distance of voxels."""

    def __init__(self, dtype, heads=3, dim=32, groups=8, seed=0):
        rng = np.random.default_rng(seed)
        self.heads, self.dim, self.groups, self.c = heads, dim, groups, heads * dim
        c = self.c
        self.g, self.b = (1 + 0.1 * rng.standard_normal(c)).astype(np.float32), (0.1 * rng.standard_normal(c)).astype(np.float32)
        self.wqkv = (rng.standard_normal((3 * c, c)) / np.sqrt(c)).astype(np.float32)
        self.wo = (rng.standard_normal((c, c)) / np.sqrt(c)).astype(np.float32)
        self.bqkv, self.bo = (0.1 * rng.standard_normal(m).astype(np.float32) for m in (3 * c, c))
        self.slopes = (0.3 * 2.0 ** -np.arange(heads)).astype(np.float32)
        self.cap, self.eps = 8.0, 1e-5

    def buffers(self, be, n):
        b = {k: be.alloc(n * m) for k, m in (("norm", self.c), ("qkv", 3 * self.c), ("att", self.c), ("out", self.c))}
        b["rows"] = be.alloc_rows_int8(n, self.c)
        return b

    def run(self, be, x, coords, at, n, b):
        c, w = self.c, 3 * self.c
        be.group_norm(x, self.g, self.b, b["norm"], n, c, self.groups, self.eps, offsets=at)
        be.pack_rows8(b["norm"], b["rows"], n, c)
        be.linear_act(b["rows"], self.wqkv, self.bqkv, b["qkv"], n, c, w)
        be.attention_scored(b["qkv"], b["qkv"], b["qkv"], b["att"], n, n, self.heads, self.heads, self.dim, q_offsets=at,
                            kv_offsets=at, q_stride=w, k_offset=c, k_stride=w, v_offset=2 * c, v_stride=w, cap=self.cap,
                            slopes=self.slopes, q_coords=coords, k_coords=coords)
        be.pack_rows8(b["att"], b["rows"], n, c)
        be.linear_act(b["rows"], self.wo, self.bo, b["out"], n, c, c, residual=x)


def voxels(n, rng):
    """n voxels of a batch of three, one of them without any, ascending, and the rows of each."""
    cells = np.sort(rng.choice(2 * 32 ** 3, n, replace=False))
    c = np.stack([cells // 32768, cells // 1024 % 32, cells // 32 % 32, cells % 32], 1).astype(np.int32)
    first = int((c[:, 0] == 0).sum())
    return c, np.array([0, first, first, n], np.int32)
