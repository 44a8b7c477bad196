"""The operators of transformer blocks over voxel rows, as cases that can be timed and compared.

The structured latents that this backend's decoders turn into voxels come from transformers over the same voxels: rows of
channels with (b, x, y, z) coordinates, one sequence of rows per object.  The cases are the operators of such blocks:

  norm     root-mean-square norm of x + residual; the sum comes out too
  norm8    the same into 8-bit rows (e4m3 codes, one power-of-two scale per 32 channels), read back
  linear   x W^T + bias, activation, residual
  linear8  norm to 8-bit rows and the linear that reads them (weights in the same 8-bit format)
  rotary   RMS norm per head and rotary positions with three axes, on the q and k columns of a fused qkv buffer
  attn     attention within sequences of voxel rows (self), of voxel rows to other rows (cross), of one query per sequence

Widths and voxel counts are those of the sparse U-Net cases beside this file (512 and 1024 channels, 18,216 latent voxels,
79,523 one level up), with heads of 64 and 128 channels.  A program has one set of weights and sends one object after
another through them: the weights belong to the case, rows and coordinates to the seed.  Weights have the values that a
16-bit (or 8-bit) checkpoint gives them; a program holds them as fp32 host arrays, as the backend takes them.
"""
import math
import os
import sys
import zlib

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 10000.0


def listed():
    return [
        # One row: a pooled or conditioning token; nothing but latency.
        {"name": "norm_f32_one", "kind": "norm", "dtype": "f32", "n": 1, "c": 1024, "residual": True},
        # The norm before a block's second half, on the voxel set with the most blocks.
        {"name": "norm_bf16_512", "kind": "norm", "dtype": "bf16", "n": 79523, "c": 512, "residual": True},
        # Norm to 8-bit rows on the latent voxels.
        {"name": "norm8_bf16_1024", "kind": "norm8", "dtype": "bf16", "n": 18216, "c": 1024, "residual": True},
        # One row through the widest weights: the conditioning token's MLP.
        {"name": "linear_f16_one", "kind": "linear", "dtype": "f16", "n": 1, "ci": 1024, "co": 4096, "act": "gelu_tanh",
         "residual": False},
        # Odd widths in fp32, as input and output heads have them.
        {"name": "linear_f32_odd", "kind": "linear", "dtype": "f32", "n": 5003, "ci": 300, "co": 77, "act": "silu",
         "residual": True},
        # The MLP's second linear with the residual on the latent voxels.
        {"name": "linear_bf16_4096to1024", "kind": "linear", "dtype": "bf16", "n": 18216, "ci": 4096, "co": 1024,
         "act": "none", "residual": True},
        # The MLP's first half in 8 bits: norm, linear and GELU.
        {"name": "linear8_bf16_512to2048", "kind": "linear8", "dtype": "bf16", "n": 79523, "ci": 512, "co": 2048,
         "act": "gelu", "residual": False},
        # Positions of a small object in fp32, half-split pairs.
        {"name": "rotary_f32_small", "kind": "rotary", "dtype": "f32", "n": 997, "heads": 6, "dim": 48, "pairs": 8,
         "split": True, "norm": False, "grid": 64},
        # q and k of a fused qkv buffer with their norms.
        {"name": "rotary_bf16_64", "kind": "rotary", "dtype": "bf16", "n": 79523, "heads": 8, "dim": 64, "pairs": 10,
         "split": False, "norm": True, "grid": 128},
        # Self-attention over the latent voxels of one object, q, k and v in one buffer.
        {"name": "attn_bf16_self", "kind": "attn", "dtype": "bf16", "nq": 18216, "nk": 18216, "seqs": 1, "heads": 8,
         "kv_heads": 8, "dim": 64, "fused": True},
        # A batch of objects of uneven sizes, one of them empty, with wider heads.
        {"name": "attn_f16_batch", "kind": "attn", "dtype": "f16", "nq": 20011, "nk": 20011, "seqs": 5, "heads": 8,
         "kv_heads": 8, "dim": 128, "fused": False},
        # One query per object over all of its voxels (pooling), heads in groups.
        {"name": "attn_bf16_pool", "kind": "attn", "dtype": "bf16", "nq": 4, "nk": 79523, "seqs": 4, "heads": 16,
         "kv_heads": 4, "dim": 64, "fused": False},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))

    kind = rng.choice(["norm", "norm8", "linear", "linear", "linear8", "rotary", "attn", "attn", "attn"])
    if kind in ("norm", "norm8"):
        c = rng.choice([64, 128, 256, 512, 1024, 2048, spread(32, 2500)])
        return {"kind": kind, "dtype": rng.choice(list(TORCH)) if kind == "norm" else rng.choice(["f16", "bf16"]),
                "n": spread(1, 40000000 // c), "c": c, "residual": rng.random() < 0.7}
    if kind in ("linear", "linear8"):
        dtype = rng.choice(list(TORCH)) if kind == "linear" else rng.choice(["f16", "bf16"])
        ci, co = rng.choice([(256, 1024), (512, 2048), (1024, 4096), (2048, 512), (4096, 1024), (1024, 1024), (512, 1536),
                             (spread(24, 1500), spread(24, 1500))])
        most = 70000000000 if dtype != "f32" else 20000000000
        return {"kind": kind, "dtype": dtype, "n": spread(1, min(80000, most // (ci * co))), "ci": ci, "co": co,
                "act": rng.choice(["none", "silu", "gelu", "gelu_tanh"]), "residual": rng.random() < 0.5}
    if kind == "rotary":
        dim = rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
        grid = rng.choice([64, 128, 1024, 32768])
        return {"kind": kind, "dtype": rng.choice(list(TORCH)), "n": spread(1, 80000), "heads": rng.randint(1, 12),
                "dim": dim, "pairs": rng.randint(dim // 8, dim // 6), "split": rng.random() < 0.5,
                "norm": rng.random() < 0.6, "grid": grid}
    dim, kv_heads, seqs = rng.choice([32, 64, 64, 96, 128, 128]), rng.choice([1, 2, 4, 8]), rng.randint(1, 6)
    heads = kv_heads * rng.choice([1, 1, 2, 4] if kv_heads < 8 else [1, 1, 2])
    form = rng.choice(["self", "cross", "pool"])
    budget = 18000.0 ** 2 * 8 * 64 / (heads * dim)
    dtype = rng.choice(["f16", "bf16"])
    if form == "self":
        n = spread(1, int(min(20000.0, math.sqrt(budget))))
        return {"kind": kind, "dtype": dtype, "nq": n, "nk": n, "seqs": seqs, "heads": heads, "kv_heads": heads, "dim": dim,
                "fused": rng.random() < 0.5}
    if form == "cross":
        nk = spread(1, 3000)
        return {"kind": kind, "dtype": dtype, "nq": spread(1, int(min(20000.0, budget / nk))), "nk": nk, "seqs": seqs,
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "fused": False}
    return {"kind": kind, "dtype": dtype, "nq": seqs, "nk": spread(200, 80000), "seqs": seqs, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "fused": False}


# ---- the program: its weights, and its backend -------------------------------------------------------------------


def weights(case):
    """A model's weights as fp32 tensors on the GPU."""
    kind, dtype = case["kind"], TORCH[case["dtype"]]
    key = {k: v for k, v in case.items() if k not in ("name", "n", "nq", "nk")}
    gen = torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(sorted(key.items())).encode()))

    def vec(*shape, one=0.0):
        return one + 0.1 * torch.randn(shape, generator=gen, device="cuda")

    if kind in ("norm", "norm8"):
        return {"g": vec(case["c"], one=1.0)}
    if kind in ("linear", "linear8"):
        ci, co = case["ci"], case["co"]
        w = torch.randn((co, ci), generator=gen, device="cuda") / math.sqrt(ci)
        w = in_8_bits(w) if kind == "linear8" else w.to(dtype).float()
        return {"w": w.contiguous(), "b": vec(co), "g": vec(ci, one=1.0)}
    if kind == "rotary" and case["norm"]:
        return {"g": vec(2 * case["heads"], case["dim"], one=1.0)}
    return {}


class Program:
    def __init__(self, case):
        self.w = weights(case)
        self.host = {k: np.ascontiguousarray(v.cpu().numpy()) for k, v in self.w.items()}
        self.dtype = case["dtype"]
        self._be = None

    def be(self):
        """The program's backend, on torch's stream: made with the first call."""
        if self._be is None:
            path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trellis2.c_amd")
            if path not in sys.path:
                sys.path.insert(0, path)
            import sparse_hip as sh

            self.sh = sh
            self._be = sh.Backend(0, {"f32": sh.F32, "f16": sh.F16, "bf16": sh.BF16}[self.dtype])
            self._be.set_stream(torch.cuda.current_stream().cuda_stream)
        return self._be


_program = {"key": None, "it": None}


def program(case):
    """The running program: kept while calls of the same model follow each other."""
    key = repr(sorted((k, v) for k, v in case.items() if k not in ("name", "n", "nq", "nk")))
    if _program["key"] != key:
        _program["it"] = None
        _program["it"] = Program(case)
        _program["key"] = key
    return _program["it"]


# ---- inputs ------------------------------------------------------------------------------------------------------


def lengths(total, seqs, empty):
    """Rows of each sequence, uneven: shares of 1, 2, 3, ..., the third of four or more empty where `empty` says so."""
    share = [0 if empty and seqs >= 4 and i == 2 else i + 1 for i in range(seqs)]
    got = [total * s // sum(share) for s in share]
    got[-1] += total - sum(got)
    return got


def query_lengths(case):
    if case["nq"] == case["seqs"] and case["nk"] != case["nq"]:
        return [1] * case["seqs"]  # one query per sequence
    return lengths(case["nq"], case["seqs"], case["nq"] == case["nk"])


def key_lengths(case):
    return lengths(case["nk"], case["seqs"], True)


def inputs(case, seed):
    """The rows of one call, on the GPU."""
    kind, dtype = case["kind"], TORCH[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + zlib.crc32(kind.encode())) % (1 << 31))

    def rows(n, c, size=1.0):
        return (size * torch.randn((n, c), generator=gen, device="cuda")).to(dtype)

    if kind in ("norm", "norm8", "linear8"):
        n, c = case["n"], case.get("c", case.get("ci"))
        # The residual stream: channels of uneven size, rows too.
        loud = torch.exp(0.7 * torch.randn((1, c), generator=gen, device="cuda"))
        d = {"x": (rows(n, c).float() * loud * torch.exp(0.5 * rows(n, 1).float())).to(dtype)}
        if kind != "linear8" and case["residual"]:
            d["r"] = rows(n, c)
        if kind == "linear8" and case["residual"]:
            d["r"] = rows(n, case["co"])
        return d
    if kind == "linear":
        d = {"x": rows(case["n"], case["ci"])}
        if case["residual"]:
            d["r"] = rows(case["n"], case["co"])
        return d
    if kind == "rotary":
        n, w = case["n"], case["heads"] * case["dim"]
        at = torch.randint(0, case["grid"], (n, 4), generator=gen, device="cuda", dtype=torch.int32)
        at[:, 0] = 0
        return {"x": rows(n, 3 * w), "coords": at}
    h, hk, d_ = case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:
        qkv = rows(case["nq"], 3 * h * d_)
        q, k, v = qkv.split(h * d_, 1)
        d = {"qkv": qkv, "q": q, "k": k, "v": v}
    else:
        d = {"q": rows(case["nq"], h * d_), "k": rows(case["nk"], hk * d_), "v": rows(case["nk"], hk * d_)}
    for name, got in (("q_at", query_lengths(case)), ("k_at", key_lengths(case))):
        d[name] = torch.tensor([0] + got, device="cuda").cumsum(0).to(torch.int32)
    return d


def prepare(case, seed):
    s = {"case": dict(case), "p": program(case), **inputs(case, seed)}
    dtype, kind = TORCH[case["dtype"]], case["kind"]

    def out(name, n, c):
        s[name] = torch.empty((n, c), dtype=dtype, device="cuda")

    if kind in ("norm", "norm8"):
        out("y", case["n"], case["c"])
        if case["residual"]:
            out("total", case["n"], case["c"])
    elif kind in ("linear", "linear8"):
        out("y", case["n"], case["co"])
    elif kind == "rotary":
        out("y", case["n"], 2 * case["heads"] * case["dim"])
    else:
        out("y", case["nq"], case["heads"] * case["dim"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


def in_8_bits(v):
    """The values that 8-bit rows hold of v: per 32 channels a scale 2^e, the least that fits them into +-448, and e4m3."""
    n, c = v.shape
    b = torch.nn.functional.pad(v, (0, -c % 32)).reshape(n, -1, 32)
    most, power = torch.frexp(b.abs().amax(2, keepdim=True))  # most * 2^power, most in [0.5, 1)
    e = (power - torch.where(most <= 0.875, 9, 8)).clamp(-126, 127)
    q = torch.ldexp(b, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(q, e).reshape(n, -1)[:, :c]


def rms(s, g):
    return s / (s.square().mean(-1, keepdim=True) + EPS).sqrt() * g


def activate(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def plain_linear(s, x):
    case, w = s["case"], s["p"].w
    v = activate(x @ w["w"].T + w["b"], case["act"])
    return v + s["r"].float() if case["residual"] else v


def plain_rotary(s):
    case, heads, dim = s["case"], 2 * s["case"]["heads"], s["case"]["dim"]
    x = s["x"][:, :heads * dim].float().reshape(-1, heads, dim)
    if case["norm"]:
        x = rms(x, s["p"].w["g"])
    j = torch.arange(case["pairs"], device="cuda", dtype=torch.float64) / case["pairs"]
    angle = (s["coords"][:, 1:, None].double() * BASE ** -j).reshape(-1, 1, 3 * case["pairs"])
    angle = torch.nn.functional.pad(angle, (0, dim // 2 - 3 * case["pairs"]))
    cos, sin = angle.cos().float(), angle.sin().float()
    if case["split"]:
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], 2)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], 3)
    return y.reshape(-1, heads * dim)


def padded(rows, at, most, heads, dim):
    """[sequence][head][row][channel], and which of those rows there are."""
    i = torch.arange(most, device="cuda")
    there = i[None] < (at[1:] - at[:-1])[:, None]
    row = (at[:-1, None] + i[None]).clamp_max(rows.shape[0] - 1).long()
    return rows[row].float().reshape(row.shape[0], most, heads, dim).transpose(1, 2).contiguous(), there


def plain_attention(s):
    case, dim, heads, group = s["case"], s["case"]["dim"], s["case"]["heads"], s["case"]["heads"] // s["case"]["kv_heads"]
    q, q_there = padded(s["q"], s["q_at"], max(query_lengths(case)), heads, dim)
    k, k_there = padded(s["k"], s["k_at"], max(key_lengths(case)), case["kv_heads"], dim)
    v, _ = padded(s["v"], s["k_at"], max(key_lengths(case)), case["kv_heads"], dim)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    score = q @ k.transpose(2, 3).contiguous() * dim ** -0.5
    if case["seqs"] > 1:
        score = score.masked_fill(~k_there[:, None, None], float("-inf"))
    most = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(most), most, 0.0))
    y = (p @ v) / p.sum(3, keepdim=True).clamp_min(1e-30)
    return y.transpose(1, 2)[q_there].reshape(-1, heads * dim)


def plain(s):
    case, dtype = s["case"], TORCH[s["case"]["dtype"]]
    if case["kind"] in ("norm", "norm8"):
        total = s["x"].float() + s["r"].float() if case["residual"] else s["x"].float()
        y = rms(total, s["p"].w["g"])
        y = (in_8_bits(y) if case["kind"] == "norm8" else y).to(dtype)
        return {"y": y, "total": total.to(dtype)} if case["residual"] else {"y": y}
    if case["kind"] == "linear":
        return plain_linear(s, s["x"].float()).to(dtype)
    if case["kind"] == "linear8":
        return plain_linear(s, in_8_bits(rms(s["x"].float(), s["p"].w["g"]))).to(dtype)
    return (plain_rotary(s) if case["kind"] == "rotary" else plain_attention(s)).to(dtype)


# ---- the framework's ---------------------------------------------------------------------------------------------


def kernels(s):
    case, p = s["case"], s["p"]
    be, w, kind = p.be(), p.host, case["kind"]
    if kind in ("norm", "norm8"):
        n, c = case["n"], case["c"]
        x, y = be.wrap(s["x"]), be.wrap(s["y"])
        more = {"residual": be.wrap(s["r"]), "total": be.wrap(s["total"])} if case["residual"] else {}
        if kind == "norm":
            be.rms_norm(x, w["g"], y, n, c, EPS, **more)
        else:
            rows8 = be.alloc_rows8(n, c)
            be.rms_norm(x, w["g"], rows8, n, c, EPS, **more)
            be.expand_rows8(rows8, y, n, c)
        return {"y": s["y"], "total": s["total"]} if case["residual"] else {"y": s["y"]}
    if kind in ("linear", "linear8"):
        n, ci, co = case["n"], case["ci"], case["co"]
        x, y = be.wrap(s["x"]), be.wrap(s["y"])
        if kind == "linear8":
            rows8 = be.alloc_rows8(n, ci)
            be.rms_norm(x, w["g"], rows8, n, ci, EPS)
            x = rows8
        be.linear_act(x, w["w"], w["b"], y, n, ci, co, act=case["act"], residual=be.wrap(s["r"]) if case["residual"] else None)
        return s["y"]
    if kind == "rotary":
        be.rotary(be.wrap(s["x"]), be.wrap(s["coords"]), be.wrap(s["y"]), case["n"], 2 * case["heads"], case["dim"],
                  [case["pairs"]] * 3, base=BASE, split=case["split"], gamma=w.get("g"), eps=EPS if case["norm"] else None,
                  x_stride=3 * case["heads"] * case["dim"])
        return s["y"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["fused"]:
        q = k = v = be.wrap(s["qkv"])
        places = {"q_stride": 3 * h * d, "k_stride": 3 * h * d, "v_stride": 3 * h * d, "k_offset": h * d, "v_offset": 2 * h * d}
    else:
        q, k, v, places = be.wrap(s["q"]), be.wrap(s["k"]), be.wrap(s["v"]), {}
    be.attention(q, k, v, be.wrap(s["y"]), case["nq"], case["nk"], h, hk, d, q_offsets=be.wrap(s["q_at"]),
                 kv_offsets=be.wrap(s["k_at"]), **places)
    return s["y"]


def run(s):
    return kernels(s) if own else plain(s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    kind, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind in ("norm", "norm8"):
        # In: x and the residual; out: the sum and the norm (of norm8 the values that the 8-bit rows stand for).
        return {"bytes": case["n"] * case["c"] * e * (4 if case["residual"] else 2) + 4 * case["c"],
                "flops": 5.0 * case["n"] * case["c"]}
    if kind in ("linear", "linear8"):
        n, ci, co = case["n"], case["ci"], case["co"]
        return {"bytes": n * ci * e + n * co * e * (2 if case["residual"] else 1) + ci * co * (1 if kind == "linear8" else e),
                "flops": 2.0 * n * ci * co}
    if kind == "rotary":
        m = 2 * case["n"] * case["heads"] * case["dim"]
        return {"bytes": 2 * m * e + 16 * case["n"], "flops": 8.0 * m}
    pairs = sum(a * b for a, b in zip(query_lengths(case), key_lengths(case)))
    return {"bytes": 2 * case["dim"] * (case["nq"] * case["heads"] + case["nk"] * case["kv_heads"]) * e,
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------


def codes64(v):
    """8-bit rows in 64 bits: e4m3 has steps of 2^-3 of its value's power of two, down to 2^-9."""
    out = torch.zeros_like(v)
    for at in range(0, v.shape[1], 32):
        b = v[:, at:at + 32]
        most = b.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(most > 0, most, 1.0) / 448))
        u = b / 2.0 ** e
        step = 2.0 ** (torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))).clamp_min(-6) - 3)
        out[:, at:at + 32] = torch.round(u / step) * step * 2.0 ** e
    return out


def exact(case, seed):
    d, w, kind = inputs(case, seed), {k: v.double() for k, v in weights(case).items()}, case["kind"]
    if kind in ("norm", "norm8", "linear8"):
        x = d["x"].double() + (d["r"].double() if "r" in d and kind != "linear8" else 0)
        y = x * torch.rsqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS) * w["g"]
        y = y if kind == "norm" else codes64(y)
        if kind != "linear8":
            return {"y": y, "total": x} if "r" in d else {"y": y}
    if kind in ("linear", "linear8"):
        z = torch.addmm(w["b"], d["x"].double() if kind == "linear" else y, w["w"].t())
        if case["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["act"] != "none":
            z = torch.nn.functional.gelu(z, approximate="none" if case["act"] == "gelu" else "tanh")
        return z + d["r"].double() if "r" in d else z
    if kind == "rotary":
        h, dim, pairs = 2 * case["heads"], case["dim"], case["pairs"]
        x = d["x"][:, :h * dim].double().view(-1, h, dim)
        if case["norm"]:
            x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * w["g"]
        y = x.clone()
        for axis in range(3):
            for j in range(pairs):
                p = axis * pairs + j
                one, two = (p, p + dim // 2) if case["split"] else (2 * p, 2 * p + 1)
                turn = torch.polar(torch.ones(x.shape[0], dtype=torch.float64, device="cuda"),
                                   d["coords"][:, 1 + axis].double() / BASE ** (j / pairs))
                z = torch.complex(x[:, :, one], x[:, :, two]) * turn[:, None]
                y[:, :, one], y[:, :, two] = z.real, z.imag
        return y.reshape(-1, h * dim)
    h, group, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    y = torch.zeros((case["nq"], h * dim), dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for nq, nk in zip(query_lengths(case), key_lengths(case)):
        for i in range(h if nq and nk else 0):
            j = i // group
            q = d["q"][q0:q0 + nq, i * dim:(i + 1) * dim].double()
            k, v = (d[t][k0:k0 + nk, j * dim:(j + 1) * dim].double() for t in ("k", "v"))
            y[q0:q0 + nq, i * dim:(i + 1) * dim] = torch.softmax(q @ k.t() / math.sqrt(dim), 1) @ v
        q0, k0 = q0 + nq, k0 + nk
    return y
