"""A transformer block over voxel rows, as a program runs it with this backend's row operators."""
import numpy as np

import sparse_hip as sh


class Block:
    """x + Wo attention(rotary(Wqkv norm(x))), then + W2 gelu(W1 norm(.)), the last two linears' input in 8 bits where
    `in8`: weights as a program holds them."""

    def __init__(self, dtype, heads=3, dim=32, hidden=320, seed=0):
        rng = np.random.default_rng(seed)
        self.heads, self.dim, self.c, self.hidden = heads, dim, heads * dim, hidden
        c = self.c

        def mat(co, ci):
            return sh.storage_round((rng.standard_normal((co, ci)) / np.sqrt(ci)).astype(np.float32), dtype)

        def vec(n, one=0.0):
            return (one + 0.1 * rng.standard_normal(n)).astype(np.float32)

        self.g1, self.g2, self.gqk = vec(c, 1.0), vec(c, 1.0), vec(2 * c, 1.0).reshape(2 * heads, dim)
        self.wqkv, self.bqkv, self.wo, self.bo = mat(3 * c, c), vec(3 * c), mat(c, c), vec(c)
        self.w1, self.b1, self.w2, self.b2 = mat(hidden, c), vec(hidden), mat(c, hidden), vec(c)

    def buffers(self, be, n):
        b = {k: be.alloc(n * m) for k, m in (("n1", self.c), ("qkv", 3 * self.c), ("att", self.c), ("h", self.c),
                                             ("hid", self.hidden), ("out", self.c))}
        b["n2"], b["hid8"] = be.alloc_rows8(n, self.c), be.alloc_rows8(n, self.hidden)
        return b

    def run(self, be, x, coords, at, n, b):
        c, w = self.c, 3 * self.c
        be.rms_norm(x, self.g1, b["n1"], n, c, 1e-6)
        be.linear_act(b["n1"], self.wqkv, self.bqkv, b["qkv"], n, c, w)
        be.rotary(b["qkv"], coords, b["qkv"], n, 2 * self.heads, self.dim, (5, 5, 5), gamma=self.gqk, eps=1e-6, x_stride=w,
                  y_stride=w)
        be.attention(b["qkv"], b["qkv"], b["qkv"], b["att"], n, n, self.heads, self.heads, self.dim, q_offsets=at,
                     kv_offsets=at, q_stride=w, k_offset=c, k_stride=w, v_offset=2 * c, v_stride=w)
        be.linear_act(b["att"], self.wo, self.bo, b["h"], n, c, c, residual=x)
        be.rms_norm(b["h"], self.g2, b["n2"], n, c, 1e-6)
        be.linear_act(b["n2"], self.w1, self.b1, b["hid"], n, c, self.hidden, act="gelu_tanh")
        be.pack_rows8(b["hid"], b["hid8"], n, self.hidden)
        be.linear_act(b["hid8"], self.w2, self.b2, b["out"], n, self.hidden, c, residual=b["h"])


def voxels(n, rng):
    """n voxels of a batch of two, ascending, and the rows of each."""
    cells = np.sort(rng.choice(2 * 20 ** 3, n, replace=False))
    c = np.stack([cells // 8000, cells // 400 % 20, cells // 20 % 20, cells % 20], 1).astype(np.int32)
    return c, np.array([0, int((c[:, 0] == 0).sum()), n], np.int32)
