"""The language-model operators' checks of arguments, all before any device work, and the C ABI's."""
import ctypes
import os
import re

import pytest
import torch

from spiky_amd import CounterDropout, ResidualNorm, _native, counter_dropout, process_logits, residual_norm
import lm_plain

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(ROOT, "include", "spiky_lm.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"\b(spiky_lm_[a-z0-9_]+)\s*\(", text))
    assert len(names) == 6
    assert all(hasattr(_native.lib(), n) for n in names) and names <= set(_native.exported_symbols())


@pytest.mark.parametrize("struct,name", [(_native.LmResidualArgs, "spiky_lm_residual_args"),
                                         (_native.LmResidualGrads, "spiky_lm_residual_grads"),
                                         (_native.LmLogitsArgs, "spiky_lm_logits_args")])
def test_structures_are_the_headers(struct, name):
    """The ctypes structures have the header's fields, in its order and types."""
    text = open(os.path.join(ROOT, "include", "spiky_lm.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    body = re.findall(r"typedef struct \{([^}]*)\}\s*(\w+);", text)
    body = next(b for b, n in body if n == name)
    kinds = {"uint64_t": ctypes.c_uint64, "int64_t": ctypes.c_int64, "int": ctypes.c_int, "float": ctypes.c_float,
             "double": ctypes.c_double}
    fields = []
    for line in filter(None, (s.strip() for s in body.split(";"))):
        line = line.replace("const ", "")
        kind, rest = line.split(None, 1)
        for field in rest.split(","):
            field = field.strip()
            fields.append((field.lstrip("* "), ctypes.c_void_p if field.startswith("*") or kind == "void" else kinds[kind]))
    assert fields == list(struct._fields_)


def test_philox_rounds_are_the_vector_forms():
    want = lm_plain.philox7(3, 5, 7, 1, 0x89ABCDEF, 0x01234567)
    keep = [w >= 1 << 31 for w in want]
    got = lm_plain.kept(1, 16, 0.5, 0x0123456789ABCDEF, (1 << 32) | 7, row0=5)[0, 12:]
    assert got.tolist() == keep


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4)
    for call in (lambda: counter_dropout(x, 0.5, 1), lambda: residual_norm(x, x), lambda: process_logits(x)):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call()
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        process_logits([1.0])


def test_modules_check_their_arguments():
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="between 0 and 1"):
            CounterDropout(p)
        with pytest.raises(ValueError, match="between 0 and 1"):
            ResidualNorm(8, dropout_p=p)
    with pytest.raises(ValueError, match="'rms' or 'layer'"):
        ResidualNorm(8, post_norm="batch")


def test_gate_rows():
    shape = torch.Size((2, 3, 5, 4))

    def _gate_rows(gate, shape):
        return _native.lm().rows_of_gate(gate, torch.zeros(shape))

    assert _gate_rows(torch.zeros(4), shape)[1] == 30
    assert _gate_rows(torch.zeros(2, 1, 1, 4), shape)[1] == 15
    assert _gate_rows(torch.zeros(2, 3, 1, 4), shape)[1] == 5
    assert _gate_rows(torch.zeros(2, 3, 5, 4), shape)[1] == 1
    for other in ((3, 5, 4), (5, 4), (1,), (2, 1, 1, 1), (2, 1, 5, 4)):
        g, n = _gate_rows(torch.zeros(other), shape)
        assert g.shape == shape and n == 1
    for bad in ((3,), (2, 4), (1, 2, 3, 5, 4)):
        with pytest.raises(ValueError, match="does not broadcast"):
            _gate_rows(torch.zeros(bad), shape)


def test_rows_of_a_tensor():
    base = torch.arange(4 * 6 * 8).reshape(4, 6, 8)
    for t, step in ((base, 8), (base[:, 1], 48), (base[:, 2:4], None), (base[::2, :1], 96), (base[..., 1:3], 8),
                    (base[..., ::2], None), (base.transpose(0, 1), None), (base[0, 0].expand(5, 8), 0), (base[:1, :1], 8)):
        rows, stride = _native.lm().rows_of_tensor(t)
        flat = rows.as_strided((t.numel() // t.shape[-1], t.shape[-1]), (stride, 1))
        assert torch.equal(flat, t.reshape(-1, t.shape[-1]))
        if step is not None:
            assert rows is t and stride == step
    assert _native.lm().rows_of_tensor(torch.tensor(3.0))[1] == 1


def refuse(status, message):
    with pytest.raises(ValueError, match=message):
        _native.check_lm(status)


def test_dropout_entry_refuses():
    L, p = _native.lib(), 16
    refuse(L.spiky_lm_dropout(p, 4, p, 1, 4, 3, 0.5, 0, 0, None, None), "unknown element type")
    refuse(L.spiky_lm_dropout(p, 4, p, 1, 4, 0, 1.5, 0, 0, None, None), "between 0 and 1")
    refuse(L.spiky_lm_dropout(p, 4, p, 1, 4, 0, float("nan"), 0, 0, None, None), "between 0 and 1")
    refuse(L.spiky_lm_dropout(p, 4, p, 1 << 32, 4, 0, 0.5, 0, 0, None, None), "too many rows")
    refuse(L.spiky_lm_dropout(None, 4, p, 1, 4, 0, 0.5, 0, 0, None, None), "null pointer")
    assert L.spiky_lm_dropout(None, 4, None, 0, 4, 0, 0.5, 0, 0, None, None) == 0
    assert L.spiky_lm_last_error() == b""


def residual_args(**kw):
    a = _native.LmResidualArgs(rows=4, cols=8, res_dtype=0, act_dtype=1, pre_norm=1, residual=16, branch=16,
                               residual_stride=8, branch_stride=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(act_dtype=5), "unknown element type"),
    (dict(res_dtype=2), "must be fp32 or have the branch's type"),
    (dict(rows=1 << 32), "too many rows"),
    (dict(pre_norm=3), "unknown norm"),
    (dict(post_weight=16), "parameters of a norm"),
    (dict(pre_norm=0, pre_bias=16), "parameters of a norm"),
    (dict(pre_norm=0, branch=None), "neither a branch nor a norm"),
    (dict(branch=None, gate=16, gate_rows=1), "of no branch"),
    (dict(gate=16, gate_rows=3), "divide the rows"),
    (dict(gate=16, gate_rows=0), "divide the rows"),
    (dict(residual=None), "null pointer"),
    (dict(dropout_p=2.0), "between 0 and 1"),
])
def test_residual_entry_refuses(change, message):
    refuse(_native.lib().spiky_lm_residual_norm(residual_args(**change), 16, 16, None), message)


def test_residual_backward_entry_refuses():
    L = _native.lib()
    G = _native.LmResidualGrads
    refuse(L.spiky_lm_residual_norm(residual_args(), 16, None, None), "null pointer")
    refuse(L.spiky_lm_residual_norm_backward(residual_args(), None, None), "null pointer")
    refuse(L.spiky_lm_residual_norm_backward(residual_args(), G(d_out=16), None), "forward's stats")
    refuse(L.spiky_lm_residual_norm_backward(residual_args(pre_norm=0), G(d_normed=16), None), "of no output")
    refuse(L.spiky_lm_residual_norm_backward(residual_args(branch=None), G(d_branch=16), None), "of no input")
    refuse(L.spiky_lm_residual_norm_backward(residual_args(), G(d_gate=16), None), "of no input")
    args = residual_args(stats=16, pre_weight=16)
    grads = G(d_out=16, d_normed=16, d_pre_weight=16, workspace=16)
    need = L.spiky_lm_residual_norm_workspace(args, grads)
    assert need > 0
    grads.workspace_bytes = need - 1
    refuse(L.spiky_lm_residual_norm_backward(args, grads, None), "workspace too small")
    assert L.spiky_lm_residual_norm(residual_args(rows=0, residual=None), None, None, None) == 0


@pytest.mark.parametrize("change,message", [
    (dict(dtype=7), "unknown element type"),
    (dict(out_dtype=2), "must be fp32 or have the logits' type"),
    (dict(bias=16, bias_dtype=9), "unknown element type"),
    (dict(vocab=1 << 31), "too many entries"),
    (dict(history=1 << 30), "too long a history"),
    (dict(tokens=16, repetition=0.0), "must be positive"),
    (dict(bias_ids=16), "without values"),
    (dict(logits=None), "null pointer"),
])
def test_logits_entry_refuses(change, message):
    a = _native.LmLogitsArgs(rows=2, vocab=8, logits=16, out=16, logits_stride=8, out_stride=8, dtype=1, out_dtype=1,
                             repetition=1.0, temperature=1.0)
    for k, v in change.items():
        setattr(a, k, v)
    refuse(_native.lib().spiky_lm_process_logits(a, None), message)


def test_rows_that_overlap():
    """Rows of two views of one memory, against the elements that they share."""
    base = torch.arange(240)
    views = {f"{at}:{n}x{width}/{step}": base.as_strided((n, width), (step, 1), at)
             for at in (0, 1, 7, 8, 20, 60) for n, width, step in ((1, 8, 8), (3, 8, 8), (4, 5, 12), (2, 10, 24), (5, 6, 0),
                                                                    (3, 0, 9), (6, 7, 5))}
    halves = torch.zeros(480, dtype=torch.int32)
    assert not _native.lm().rows_overlap(base[:24].reshape(3, 8), halves[:24].reshape(3, 8))
    for a in views.values():
        for b in views.values():
            assert _native.lm().rows_overlap(a, b) == bool(set(a.flatten().tolist()) & set(b.flatten().tolist())), (a, b)
    # of other types: the bytes count
    bytes_ = base.view(torch.int8)
    assert _native.lm().rows_overlap(base[4:8].reshape(1, 4), bytes_[63:64].reshape(1, 1))
    assert not _native.lm().rows_overlap(base[4:8].reshape(1, 4), bytes_[64:70].reshape(1, 6))
    assert not _native.lm().rows_overlap(base[4:8].reshape(1, 4), bytes_[20:32].reshape(1, 12))
    assert _native.lm().rows_overlap(base[4:8].reshape(1, 4), bytes_[20:33].reshape(1, 13))
