"""Group norm, integer rows and attention with changed scores without a device: null arguments, and the descriptor's layout."""
import ctypes
import os
import re

import sparse_hip as sh

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_null_arguments():
    out = ctypes.c_void_p(7)
    L, bad = sh.LIB, sh.INVALID_ARGUMENT
    assert L.trellis_sparse_hip_alloc_rows_int8(None, 1, 1, ctypes.byref(out)) == bad
    assert L.trellis_sparse_hip_group_norm(None, None, None, 1, None, None, None, 1, 1, 1, 1e-5, 0) == bad
    d, s = sh.AttentionDesc(), sh.ScoresDesc()
    assert L.trellis_sparse_hip_attention_scored(None, None, None, None, None, 1, 1, None, None, 1, ctypes.byref(d),
                                                 ctypes.byref(s)) == bad
    assert L.trellis_sparse_hip_attention_scored(None, None, None, None, None, 1, 1, None, None, 1, ctypes.byref(d), None) == bad


def test_descriptor_matches_the_header():
    text = open(os.path.join(ROOT, "include", "trellis_sparse_hip.h")).read()
    name = "trellis_sparse_hip_scores_desc"
    body = text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body.split("{", 1)[1], flags=re.S)
    fields = [re.sub(r"[\s*]", "", re.sub(r"^\s*(const\s+)?\w+\s+", "", line)) for line in body.split(";") if line.strip()]
    assert fields == [f[0] for f in sh.ScoresDesc._fields_]
    assert ctypes.sizeof(sh.ScoresDesc) == 48
