"""Group norm, products of 8-bit integers and attention with capped, biased or masked scores, as cases that can be timed and
compared.

They are what an attention block of a sparse U-Net over voxel rows consists of when its products run in integers:

  gnorm  group norm over the rows of each object and its groups of channels, with the activation that follows
  int8   rows to 8-bit integers, one scale a row (of an RMS norm, or of the rows as they are), and the linear that reads them,
         weights with one scale an output channel, with bias, activation and residual
  attn   attention whose scores are capped by a tanh, lowered by the distance of voxels or of rows, or masked (causal, with
         a prefix that every query sees)

Widths and voxel counts are those of the cases beside this file (128 to 1024 channels, 18,216 latent voxels, 79,523 and 419,340
on the levels above), heads of 64 and 128 channels, 32 groups.  A program has one set of weights and sends one object after
another through them: the weights belong to the case, rows and coordinates to the seed.  Weights of integer products have the
values that an 8-bit checkpoint gives them; a program holds them as fp32 host arrays, as the backend takes them.
"""
import math
import os
import sys
import zlib

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # The norm of a very small object: nothing but latency.
        {"name": "gnorm_f32_small", "kind": "gnorm", "dtype": "f32", "n": 211, "c": 64, "groups": 32, "seqs": 1, "act": "silu"},
        # Odd channel counts: groups of 30 channels, which no vector load is a whole part of.
        {"name": "gnorm_f32_odd", "kind": "gnorm", "dtype": "f32", "n": 5003, "c": 300, "groups": 10, "seqs": 3, "act": "none"},
        # The norm before a residual block's first conv, on the voxel set with the most blocks.
        {"name": "gnorm_bf16_512", "kind": "gnorm", "dtype": "bf16", "n": 79523, "c": 512, "groups": 32, "seqs": 1,
         "act": "silu"},
        # A batch of objects of uneven sizes, one of them empty, on the level above.
        {"name": "gnorm_f16_batch", "kind": "gnorm", "dtype": "f16", "n": 419340, "c": 128, "groups": 32, "seqs": 5,
         "act": "silu"},
        # One row through the widest weights: a conditioning token.
        {"name": "int8_bf16_one", "kind": "int8", "dtype": "bf16", "n": 1, "ci": 1024, "co": 4096, "norm": True,
         "act": "gelu_tanh", "residual": False},
        # Odd widths, as input and output heads have them.
        {"name": "int8_f32_odd", "kind": "int8", "dtype": "f32", "n": 5003, "ci": 300, "co": 77, "norm": False, "act": "silu",
         "residual": True},
        # The MLP's second linear with the residual on the latent voxels.
        {"name": "int8_f16_4096to1024", "kind": "int8", "dtype": "f16", "n": 18216, "ci": 4096, "co": 1024, "norm": False,
         "act": "none", "residual": True},
        # The MLP's first half on the level above: norm, linear, GELU.
        {"name": "int8_bf16_512to2048", "kind": "int8", "dtype": "bf16", "n": 79523, "ci": 512, "co": 2048, "norm": True,
         "act": "gelu", "residual": False},
        # One new row per object behind a long cache, heads in groups: scores capped and lowered by the rows between.
        {"name": "attn_bf16_decode", "kind": "attn", "dtype": "bf16", "nq": 4, "nk": 79523, "seqs": 4, "heads": 16,
         "kv_heads": 4, "dim": 64, "cap": 30.0, "bias": "rows", "causal": True, "prefix": 0},
        # Rows generated in order behind a prefix of conditioning rows.
        {"name": "attn_f16_prefix", "kind": "attn", "dtype": "f16", "nq": 9001, "nk": 9001, "seqs": 2, "heads": 8,
         "kv_heads": 4, "dim": 128, "cap": 0.0, "bias": "none", "causal": True, "prefix": 1374},
        # Self-attention of a batch of objects with capped scores.
        {"name": "attn_f16_cap_batch", "kind": "attn", "dtype": "f16", "nq": 20011, "nk": 20011, "seqs": 5, "heads": 8,
         "kv_heads": 8, "dim": 128, "cap": 50.0, "bias": "none", "causal": False, "prefix": 0},
        # Self-attention over the latent voxels of one object, near voxels first.
        {"name": "attn_bf16_voxels", "kind": "attn", "dtype": "bf16", "nq": 18216, "nk": 18216, "seqs": 1, "heads": 8,
         "kv_heads": 8, "dim": 64, "cap": 0.0, "bias": "voxels", "causal": False, "prefix": 0},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999))))

    kind = rng.choice(["gnorm", "gnorm", "int8", "int8", "attn", "attn", "attn"])
    if kind == "gnorm":
        groups = rng.choice([1, 8, 16, 32, 32, 32])
        c = groups * rng.choice([1, 2, 4, 8, 16, 32, spread(1, 40)])
        c = c if c >= 16 else 32 * c
        return {"kind": kind, "dtype": rng.choice(list(TORCH)), "n": spread(1, min(500000, 40000000 // c)), "c": c,
                "groups": groups, "seqs": rng.choice([1, 1, 2, 4, rng.randint(1, 40)]), "act": rng.choice(["silu", "silu", "none", "gelu"])}
    if kind == "int8":
        ci, co = rng.choice([(256, 1024), (512, 2048), (1024, 4096), (2048, 512), (4096, 1024), (1024, 1024), (512, 1536),
                             (spread(24, 1500), spread(24, 1500))])
        return {"kind": kind, "dtype": rng.choice(["f32", "f16", "bf16", "bf16"]),
                "n": spread(1, min(80000, 70000000000 // (ci * co))), "ci": ci, "co": co, "norm": rng.random() < 0.5,
                "act": rng.choice(["none", "silu", "gelu", "gelu_tanh"]), "residual": rng.random() < 0.5}
    dim, kv_heads, seqs = rng.choice([32, 64, 64, 80, 96, 128, 128]), rng.choice([1, 2, 4, 8]), rng.randint(1, 6)
    heads = kv_heads * rng.choice([1, 1, 2, 4] if kv_heads < 8 else [1, 1, 2])
    form = rng.choice(["self", "cross", "decode"])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    budget = 18000.0 ** 2 * 8 * 64 / (heads * dim) / (8 if dtype == "f32" else 1)
    if form == "self":
        nq = nk = spread(seqs, int(min(20000.0, math.sqrt(budget))))
    elif form == "cross":
        nk = spread(1, 3000)
        nq = spread(1, int(min(20000.0, budget / nk)))
    else:
        nq, nk = seqs, spread(200, 80000)
    causal = form != "cross" and rng.random() < 0.5
    return {"kind": kind, "dtype": dtype, "nq": nq, "nk": nk, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "cap": rng.choice([0.0, 0.0, 20.0, 30.0, 50.0]), "bias": rng.choice(["none", "rows", "voxels", "voxels"]),
            "causal": causal, "prefix": rng.choice([0, spread(1, 1500)]) if causal else 0}


# ---- the program: its weights, and its backend -------------------------------------------------------------------


def model_of(case):
    return sorted((k, v) for k, v in case.items() if k not in ("name", "n", "nq", "nk", "seqs"))


def weights(case):
    """A model's weights as fp32 tensors on the GPU."""
    gen = torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(model_of(case)).encode()))

    def vec(*shape, one=0.0):
        return one + 0.1 * torch.randn(shape, generator=gen, device="cuda")

    if case["kind"] == "gnorm":
        return {"g": vec(case["c"], one=1.0), "b": vec(case["c"])}
    if case["kind"] == "int8":
        ci, co = case["ci"], case["co"]
        w = torch.randn((co, ci), generator=gen, device="cuda") / math.sqrt(ci)
        codes, scale = in_int8(w.double())
        return {"codes": codes, "scale": scale, "w": codes * scale, "b": vec(co), "g": vec(ci, one=1.0)}
    if case["bias"] != "none":
        # Each head looks a little less far than the one before it.
        h = case["heads"]
        return {"slopes": 2.0 ** (-8.0 * (torch.arange(h, device="cuda") + 1) / h)}
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
    key = repr(model_of(case))
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


def starts(got):
    return torch.tensor([0] + got, device="cuda").cumsum(0).to(torch.int32)


def surface(n, gen):
    """n voxels on the surfaces of an object in a grid of 128, in the order of their places."""
    p = torch.randn((n, 3), generator=gen, device="cuda")
    p = p / p.square().sum(1, keepdim=True).sqrt().clamp_min(1e-6)
    r = 40 + 20 * torch.rand((n, 1), generator=gen, device="cuda").round()
    p = (64 + r * p).round().to(torch.int64)
    order = ((p[:, 0] * 128 + p[:, 1]) * 128 + p[:, 2]).argsort()
    return torch.cat([torch.zeros_like(p[:, :1]), p], 1)[order].to(torch.int32).contiguous()


def inputs(case, seed):
    """The rows of one call, on the GPU."""
    kind, dtype = case["kind"], TORCH[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + zlib.crc32(kind.encode())) % (1 << 31))

    def rows(n, c, size=1.0):
        return (size * torch.randn((n, c), generator=gen, device="cuda")).to(dtype)

    def stream(n, c):
        """Channels of uneven size, rows too."""
        loud = torch.exp(0.7 * torch.randn((1, c), generator=gen, device="cuda"))
        return (rows(n, c).float() * loud * torch.exp(0.5 * rows(n, 1).float())).to(dtype)

    if kind == "gnorm":
        # A conv's outputs: channels with means of their own.
        off = torch.randn((1, case["c"]), generator=gen, device="cuda")
        return {"x": (stream(case["n"], case["c"]).float() + off).to(dtype),
                "at": starts(lengths(case["n"], case["seqs"], True))}
    if kind == "int8":
        d = {"x": stream(case["n"], case["ci"])}
        if case["residual"]:
            d["r"] = rows(case["n"], case["co"])
        return d
    h, hk, d_ = case["heads"], case["kv_heads"], case["dim"]
    d = {"q": rows(case["nq"], h * d_, 2.0), "k": rows(case["nk"], hk * d_), "v": rows(case["nk"], hk * d_),
         "q_at": starts(query_lengths(case)), "k_at": starts(key_lengths(case))}
    if case["bias"] == "voxels":
        d["k_xyz"] = surface(case["nk"], gen)
        d["q_xyz"] = d["k_xyz"] if case["nq"] == case["nk"] else surface(case["nq"], gen)
    if case["prefix"]:
        d["prefix"] = torch.full((case["seqs"],), case["prefix"], device="cuda", dtype=torch.int32)
    return d


def prepare(case, seed):
    s = {"case": dict(case), "p": program(case), **inputs(case, seed)}
    n, c = {"gnorm": lambda: (case["n"], case["c"]), "int8": lambda: (case["n"], case["co"]),
            "attn": lambda: (case["nq"], case["heads"] * case["dim"])}[case["kind"]]()
    s["y"] = torch.empty((n, c), dtype=TORCH[case["dtype"]], device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------


def in_int8(v):
    """Codes and scales of rows in 64 bits (a code's border is where 32 lose it)."""
    most = v.abs().amax(1, keepdim=True)
    codes = torch.round(v * 127 / torch.where(most > 0, most, 1.0))
    return codes.float(), (most / 127).float()


def activate(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def padded(rows, at, most, heads):
    """[sequence][head][row][channel], which of those rows there are, and which rows they are."""
    i = torch.arange(most, device="cuda")
    there = i[None] < (at[1:] - at[:-1])[:, None]
    row = (at[:-1, None] + i[None]).clamp_max(rows.shape[0] - 1).long()
    return rows[row].float().reshape(row.shape[0], most, heads, -1).transpose(1, 2).contiguous(), there, row


def plain_gnorm(s):
    case, w, groups = s["case"], s["p"].w, s["case"]["groups"]
    x, there, _ = padded(s["x"], s["at"], max(lengths(case["n"], case["seqs"], True)), groups)
    x = x.masked_fill(~there[:, None, :, None], 0.0)
    count = there.sum(1).clamp_min(1)[:, None, None, None] * x.shape[3]
    x = (x - x.sum((2, 3), keepdim=True, dtype=torch.float64) / count).float().masked_fill(~there[:, None, :, None], 0.0)
    var = x.square().sum((2, 3), keepdim=True, dtype=torch.float64) / count
    x = (x * (1 / (var + EPS).sqrt()).float()).transpose(1, 2)[there].reshape(case["n"], case["c"])
    return activate(x * w["g"] + w["b"], case["act"])


def plain_int8(s):
    case, w, x = s["case"], s["p"].w, s["x"].double()
    if case["norm"]:
        x = x / (x.square().mean(1, keepdim=True) + EPS).sqrt() * w["g"]
    codes, scale = in_int8(x)
    v = activate((codes @ w["codes"].T) * scale * w["scale"].T + w["b"], case["act"])
    return v + s["r"].float() if case["residual"] else v


def plain_attention(s):
    case, dim, heads, group = s["case"], s["case"]["dim"], s["case"]["heads"], s["case"]["heads"] // s["case"]["kv_heads"]
    q, q_there, q_row = padded(s["q"], s["q_at"], max(query_lengths(case)), heads)
    k, k_there, k_row = padded(s["k"], s["k_at"], max(key_lengths(case)), case["kv_heads"])
    v, _, _ = padded(s["v"], s["k_at"], max(key_lengths(case)), case["kv_heads"])
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    score = q @ k.transpose(2, 3).contiguous() * dim ** -0.5
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    # Where a query stands among its sequence's keys: the last one at the last.
    i, j = torch.arange(q.shape[2], device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")
    ahead = i + (s["k_at"][1:] - s["k_at"][:-1] - s["q_at"][1:] + s["q_at"][:-1])[:, None, None] - j
    if case["bias"] == "rows":
        score = score - s["p"].w["slopes"][:, None, None] * ahead.abs().float()[:, None]
    if case["bias"] == "voxels":
        off = s["q_xyz"][q_row][:, :, None, 1:] - s["k_xyz"][k_row][:, None, :, 1:]
        score = score - s["p"].w["slopes"][:, None, None] * off.float().square().sum(3).sqrt()[:, None]
    seen = k_there[:, None]
    if case["causal"]:
        seen = seen & ((ahead >= 0) | (j < s["prefix"][:, None, None] if case["prefix"] else False))
    score = score.masked_fill(~seen[:, None], float("-inf"))
    most = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(most), most, 0.0))
    y = (p @ v) / p.sum(3, keepdim=True).clamp_min(1e-30)
    return y.transpose(1, 2)[q_there].reshape(-1, heads * dim)


def plain(s):
    form = {"gnorm": plain_gnorm, "int8": plain_int8, "attn": plain_attention}[s["case"]["kind"]]
    return form(s).to(TORCH[s["case"]["dtype"]])


# ---- the framework's ---------------------------------------------------------------------------------------------


def kernels(s):
    case, p = s["case"], s["p"]
    be, w, kind = p.be(), p.host, case["kind"]
    if kind == "gnorm":
        be.group_norm(be.wrap(s["x"]), w["g"], w["b"], be.wrap(s["y"]), case["n"], case["c"], case["groups"], EPS,
                      act=case["act"], offsets=be.wrap(s["at"]))
    elif kind == "int8":
        n, ci, co = case["n"], case["ci"], case["co"]
        rows = be.alloc_rows_int8(n, ci)
        if case["norm"]:
            be.rms_norm(be.wrap(s["x"]), w["g"], rows, n, ci, EPS)
        else:
            be.pack_rows8(be.wrap(s["x"]), rows, n, ci)
        be.linear_act(rows, w["w"], w["b"], be.wrap(s["y"]), n, ci, co, act=case["act"],
                      residual=be.wrap(s["r"]) if case["residual"] else None)
    else:
        q_xyz = be.wrap(s["q_xyz"]) if case["bias"] == "voxels" else None
        k_xyz = be.wrap(s["k_xyz"]) if case["bias"] == "voxels" else None
        be.attention_scored(be.wrap(s["q"]), be.wrap(s["k"]), be.wrap(s["v"]), be.wrap(s["y"]), case["nq"], case["nk"],
                            case["heads"], case["kv_heads"], case["dim"], q_offsets=be.wrap(s["q_at"]),
                            kv_offsets=be.wrap(s["k_at"]), cap=case["cap"], slopes=w.get("slopes"), q_coords=q_xyz,
                            k_coords=k_xyz, causal=case["causal"], prefix=be.wrap(s["prefix"]) if case["prefix"] else None)
    return s["y"]


def run(s):
    return kernels(s) if own else plain(s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------


def work(case):
    kind, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "gnorm":
        return {"bytes": 2 * case["n"] * case["c"] * e + 8 * case["c"], "flops": 8.0 * case["n"] * case["c"]}
    if kind == "int8":
        n, ci, co = case["n"], case["ci"], case["co"]
        return {"bytes": n * ci * e + n * co * e * (2 if case["residual"] else 1) + ci * co, "flops": 2.0 * n * ci * co}
    pairs = sum(pairs_of(case, a, b) for a, b in zip(query_lengths(case), key_lengths(case)))
    rows = case["nq"] * case["heads"] + case["nk"] * case["kv_heads"]
    return {"bytes": 2 * case["dim"] * rows * e + (16 * (case["nq"] + case["nk"]) if case["bias"] == "voxels" else 0),
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


def pairs_of(case, nq, nk):
    """Queries and keys of a sequence that see each other."""
    if not case["causal"]:
        return nq * nk
    i = np.arange(nq, dtype=np.int64) + nk - nq + 1
    return int(np.clip(i, min(nk, case["prefix"]), nk).sum())


# ---- the same in 64 bits, from the definitions -------------------------------------------------------------------


def act64(z, act):
    if act == "silu":
        return z * torch.sigmoid(z)
    return z if act == "none" else torch.nn.functional.gelu(z, approximate="none" if act == "gelu" else "tanh")


def codes64(v):
    step = v.abs().max(1, keepdim=True).values / 127
    return torch.round(v / step.clamp_min(1e-300)), step


def exact(case, seed):
    d, w, kind = inputs(case, seed), {k: v.double() for k, v in weights(case).items()}, case["kind"]
    if kind == "gnorm":
        y, a = torch.zeros(d["x"].shape, dtype=torch.float64, device="cuda"), 0
        size = case["c"] // case["groups"]
        for m in lengths(case["n"], case["seqs"], True):
            for g in range(case["groups"] if m else 0):
                ch = slice(g * size, (g + 1) * size)
                x = d["x"][a:a + m, ch].double()
                var, mean = torch.var_mean(x, correction=0)
                y[a:a + m, ch] = act64((x - mean) * torch.rsqrt(var + EPS) * w["g"][ch] + w["b"][ch], case["act"])
            a += m
        return y
    if kind == "int8":
        x = d["x"].double()
        if case["norm"]:
            x = x * torch.rsqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPS) * w["g"]
        a, step = codes64(x)
        z = act64((a @ w["codes"].t()) * step * w["scale"].t() + w["b"], case["act"])
        return z + d["r"].double() if "r" in d else z
    h, group, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    y = torch.zeros((case["nq"], h * dim), dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for nq, nk in zip(query_lengths(case), key_lengths(case)):
        at = torch.arange(nk - nq, nk, device="cuda")[:, None]  # the queries' places among the keys
        key = torch.arange(nk, device="cuda")[None]
        hidden = (key > at) & (key >= case["prefix"]) if case["causal"] else None
        far = (at - key).abs().double() if case["bias"] == "rows" else None
        if case["bias"] == "voxels":
            p, r = d["q_xyz"][q0:q0 + nq, 1:].double(), d["k_xyz"][k0:k0 + nk, 1:].double()
            far = torch.sqrt(sum((p[:, a, None] - r[None, :, a]) ** 2 for a in range(3)))
        for i in range(h if nq and nk else 0):
            j = i // group
            q = d["q"][q0:q0 + nq, i * dim:(i + 1) * dim].double()
            k, v = (d[t][k0:k0 + nk, j * dim:(j + 1) * dim].double() for t in ("k", "v"))
            z = q @ k.t() / math.sqrt(dim)
            z = torch.tanh(z / case["cap"]) * case["cap"] if case["cap"] else z
            z = z if far is None else z - w["slopes"][i] * far
            z = z if hidden is None else z.masked_fill(hidden, -math.inf)
            y[q0:q0 + nq, i * dim:(i + 1) * dim] = torch.nan_to_num(torch.softmax(z, 1), nan=0.0) @ v
        q0, k0 = q0 + nq, k0 + nk
    return y
