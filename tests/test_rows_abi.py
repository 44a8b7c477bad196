"""The row operators' entry points without a device: null arguments, and the layout of their descriptors."""
import ctypes
import os
import re

import sparse_hip as sh

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_null_arguments():
    out = ctypes.c_void_p(7)
    L, bad = sh.LIB, sh.INVALID_ARGUMENT
    assert L.trellis_sparse_hip_wrap_f32(None, 16, 1, ctypes.byref(out)) == bad
    assert L.trellis_sparse_hip_wrap_i32(None, 16, 1, ctypes.byref(out)) == bad
    assert L.trellis_sparse_hip_set_stream(None, None) == bad
    assert L.trellis_sparse_hip_own_stream(None) == bad
    assert L.trellis_sparse_hip_set_scratch(None, None) == bad
    assert L.trellis_sparse_hip_scratch_bytes(None) == 0
    assert L.trellis_sparse_hip_alloc_rows8(None, 1, 1, ctypes.byref(out)) == bad
    assert L.trellis_sparse_hip_pack_rows8(None, None, None, 1, 1) == bad
    assert L.trellis_sparse_hip_expand_rows8(None, None, None, 1, 1) == bad
    assert L.trellis_sparse_hip_rms_norm(None, None, None, None, None, None, 1, 1, 1e-6) == bad
    assert L.trellis_sparse_hip_linear_act(None, None, None, None, 0, None, None, 1, 1, 1) == bad
    assert L.trellis_sparse_hip_rotary(None, None, None, None, None, 1, ctypes.byref(sh.RotaryDesc())) == bad
    assert L.trellis_sparse_hip_attention(None, None, None, None, None, 1, 1, None, None, 1,
                                          ctypes.byref(sh.AttentionDesc())) == bad
    assert L.trellis_sparse_hip_transformer_block(None, None, None, None, None, 1, ctypes.byref(sh.BlockDesc()), None, 1) == bad


def test_descriptors_match_the_header():
    text = open(os.path.join(ROOT, "include", "trellis_sparse_hip.h")).read()
    for cls, name, size in ((sh.RotaryDesc, "trellis_sparse_hip_rotary_desc", 80),
                            (sh.AttentionDesc, "trellis_sparse_hip_attention_desc", 88),
                            (sh.BlockDesc, "trellis_sparse_hip_block_desc", 144)):
        body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
        body = re.sub(r"/\*.*?\*/", "", body.split("{", 1)[1], flags=re.S)
        fields = [re.sub(r"[\s*]|\[.*\]", "", f) for line in body.split(";") if line.strip()
                  for f in re.sub(r"^\s*(const\s+)?\w+\s+", "", line).split(",")]
        assert fields == [f[0] for f in cls._fields_]
        assert ctypes.sizeof(cls) == size
    for i, name in enumerate(("NONE", "SILU", "GELU", "GELU_TANH")):
        assert re.search(rf"TRELLIS_SPARSE_HIP_ACT_{name} = {i}\b", text) and sh.ACTS[name.lower()] == i
