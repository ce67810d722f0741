"""Checks of include/spiky_lm_tokens.h and its binding that need no device."""
import ctypes
import os
import re

import pytest
import torch

from spiky_amd import _native, beam_select, embed_tokens, reorder_states

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TEXT = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "spiky_lm_tokens.h")).read(), flags=re.S)


def test_library_exports_every_declared_symbol():
    names = set(re.findall(r"\b(spiky_lm_[a-z0-9_]+)\s*\(", TEXT))
    assert len(names) == 6
    assert all(hasattr(_native.lib(), n) for n in names) and names <= set(_native.exported_symbols())


@pytest.mark.parametrize("struct,name", [(_native.LmEmbedArgs, "spiky_lm_embed_args"), (_native.LmBeamsArgs, "spiky_lm_beams_args"),
                                         (_native.LmState, "spiky_lm_state")])
def test_structures_are_the_headers(struct, name):
    body = next(b for b, n in re.findall(r"typedef struct \{([^}]*)\}\s*(\w+);", TEXT) if n == name)
    kinds = {"uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64, "int": ctypes.c_int, "double": ctypes.c_double}
    fields = []
    for line in filter(None, (s.strip().replace("const ", "") for s in body.split(";"))):
        kind, rest = line.split(None, 1)
        for field in (f.strip() for f in rest.split(",")):
            fields.append((field.lstrip("* "), ctypes.c_void_p if field.startswith("*") or kind == "void" else kinds[kind]))
    assert fields == list(struct._fields_)


def refuse(status, message):
    with pytest.raises(ValueError, match=message):
        _native.check_lm(status)


def embed_args(**kw):
    a = _native.LmEmbedArgs(n=3, vocab=5, cols=8, tokens_i64=1, weight_dtype=1, out_dtype=0, tokens=16, weight=16,
                            weight_stride=8, scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(weight_dtype=3), "unknown element type"),
    (dict(out_dtype=-1), "unknown element type"),
    (dict(out_dtype=2), "one type, or one of them fp32"),
    (dict(n=1 << 31), "too many"),
    (dict(vocab=1 << 31), "too many"),
    (dict(cols=(1 << 26) + 1), "too many"),
    (dict(tokens=None), "null pointer"),
    (dict(weight=None), "null pointer"),
    (dict(scale=float("inf")), "must be finite"),
    (dict(scale=1e39), "must be finite"),
])
def test_embed_entry_refuses(change, message):
    refuse(_native.lib().spiky_lm_embed(embed_args(**change), 16, None), message)


def test_embed_backward_entry_refuses():
    L = _native.lib()
    refuse(L.spiky_lm_embed(None, 16, None), "null pointer")
    refuse(L.spiky_lm_embed(embed_args(), None, None), "null pointer")
    need = L.spiky_lm_embed_workspace(embed_args())
    assert need >= 4 * (5 + 1 + 3) and L.spiky_lm_embed_workspace(embed_args(vocab=0)) == 0
    refuse(L.spiky_lm_embed_backward(embed_args(), 16, 8, 16, 16, need - 1, None), "workspace too small")
    refuse(L.spiky_lm_embed_backward(embed_args(), 16, 8, 16, None, need, None), "workspace too small")
    refuse(L.spiky_lm_embed_backward(embed_args(), 16, 8, None, 16, need, None), "null pointer")
    refuse(L.spiky_lm_embed_backward(embed_args(), None, 8, 16, 16, need, None), "null pointer")
    refuse(L.spiky_lm_embed_backward(embed_args(n=1 << 40), 16, 8, 16, 16, need, None), "too many")
    assert L.spiky_lm_embed(embed_args(n=0, tokens=None), None, None) == 0
    assert L.spiky_lm_embed_backward(embed_args(cols=0), None, 8, None, None, 0, None) == 0


def beams_args(**kw):
    a = _native.LmBeamsArgs(searches=2, beams=3, vocab=10, n=4, dtype=1, logits=16, search_stride=30, beam_stride=10,
                            scores=16, out_scores=16, out_parents=16, out_tokens=16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(dtype=4), "unknown element type"),
    (dict(beams=0), "1 to 64"),
    (dict(beams=65), "1 to 64"),
    (dict(n=0), "1 to 64"),
    (dict(n=65), "1 to 64"),
    (dict(vocab=1 << 31), "too many"),
    (dict(searches=1 << 24), "too many"),
    (dict(length_penalty=8.5), "-8 to 8"),
    (dict(length_penalty=float("nan")), "-8 to 8"),
    (dict(logits=None), "null pointer"),
    (dict(scores=None), "null pointer"),
    (dict(out_tokens=None), "null pointer"),
])
def test_beam_select_entry_refuses(change, message):
    refuse(_native.lib().spiky_lm_beam_select(beams_args(**change), 16, 1 << 40, None), message)


def test_beam_select_workspace():
    L = _native.lib()
    need = L.spiky_lm_beam_select_workspace(beams_args())
    assert need > 0 and need % 8 == 0
    refuse(L.spiky_lm_beam_select(beams_args(), 16, need - 1, None), "workspace too small")
    refuse(L.spiky_lm_beam_select(beams_args(), None, need, None), "workspace too small")
    assert L.spiky_lm_beam_select(beams_args(searches=0), None, 0, None) == 0


def test_reorder_entry_refuses():
    L, S = _native.lib(), _native.LmState

    def call(searches=2, beams=3, n=3, parents=16, **kw):
        s = S(**{"in": 16, "out": 32, "runs": 1, "run_bytes": 8, **kw})
        return L.spiky_lm_reorder(s, 1, parents, 1, searches, beams, n, None)

    refuse(L.spiky_lm_reorder(None, 1, 16, 1, 2, 3, 3, None), "null pointer")
    refuse(call(parents=None), "null pointer")
    refuse(call(**{"in": None}), "null pointer")
    refuse(call(out=None), "null pointer")
    refuse(call(run_bytes=1 << 35), "too long a run")
    refuse(call(runs=1 << 50, run_bytes=1 << 20), "too large a state")
    refuse(call(out=16, n=2), "in place")
    refuse(call(out=16, n=65, beams=65), "in place")
    refuse(call(n=4097), "too many")
    refuse(call(searches=1 << 31), "too many")
    assert call(searches=0) == 0 and call(n=0) == 0 and L.spiky_lm_reorder(None, 0, 16, 1, 2, 3, 3, None) == 0


def test_cpu_tensors_are_refused():
    x, i = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: embed_tokens(i, x[0]), lambda: beam_select(x, x[..., 0]), lambda: reorder_states(x, i)):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call()
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        embed_tokens(i, [1.0])
