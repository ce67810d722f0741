"""Loader of libspiky_lut.so, the HIP kernels behind the C ABI in include/spiky_lut.h
and include/spiky_lm.h and include/spiky_lm_tokens.h.

The library is built in-tree (``python -m spiky_amd.build``).  There is no
fallback: if the library is missing or fails to load, every device entry point
raises, so a GPU run can never silently compute somewhere else.
"""
import ctypes
import os
import threading

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libspiky_lut.so")

SPIKY_OK = 0
SPIKY_VALUE_ERROR = 1
SPIKY_RUNTIME_ERROR = 2

_lock = threading.Lock()
_lib = None
_lm = None

_u32 = ctypes.c_uint32
_u64 = ctypes.c_uint64
_i32 = ctypes.c_int
_i64 = ctypes.c_int64
_f32 = ctypes.c_float
_f64 = ctypes.c_double
_vp = ctypes.c_void_p
_pp = ctypes.POINTER(ctypes.c_void_p)

_SIGNATURES = {
    "spiky_lut_last_error": ([], ctypes.c_char_p),
    "spiky_lut_version": ([], ctypes.c_char_p),
    "spiky_lut_create": ([_u32, _u32, _u32, _u32, _u32, _u32, _u64, _u32, _u32, _i32, _f64, _pp], _i32),
    "spiky_lut_destroy": ([_vp], None),
    "spiky_lut_set_ordered_sums": ([_vp, _i32], _i32),
    "spiky_lut_register_synapse_meta": ([_vp, _f32, _f32, _f32, _f32, _f32, ctypes.POINTER(_u32)], _i32),
    "spiky_lut_initialize_neurons": ([_vp, _i32], _i32),
    "spiky_lut_n_lookup_neurons": ([_vp], _u64),
    "spiky_lut_weights_dimension": ([_vp], _u64),
    "spiky_lut_max_forward_groups_per_neuron": ([_vp], _u32),
    "spiky_lut_n_synapses": ([_vp], _u64),
    "spiky_lut_forward_step": ([_vp, _vp, _u32, _vp, _vp, _vp, _vp, _f32, _vp, _vp, _vp], _i32),
    "spiky_lut_forward_step_noalloc": ([_vp, _vp, _u32, _vp, _vp, _vp, _vp, _f32, _vp, _vp, _vp], _i32),
    "spiky_lut_forward_step_i8": ([_vp, _vp, _vp, _u32, _vp, _vp, _vp, _vp, _f32, _vp, _vp, _vp], _i32),
    "spiky_lut_backward_backprop": ([_vp, _vp, _u32, _vp, _vp, _vp, _vp, _vp, _vp, _f64, _vp, _i32, _vp], _i32),
    "spiky_lut_set_sparse_connectivity": ([_vp, _vp, _vp, _u64], _i32),
    "spiky_lut_decode_anchors_compact": ([_vp, _u32, _u32, _u32, _vp, _vp, _vp], _i32),
    "spiky_lut_profiling_stats": ([_vp, ctypes.c_char_p, _u64], _i32),
    "spiky_lut_reset_profiler": ([_vp], None),
    "spiky_lut_set_kernel_timing": ([_vp, _i32], _i32),
    "spiky_lut_kernel_times": ([_vp, ctypes.c_char_p, _u64, _i32], _i32),
    "spiky_lut_scratch_plan": ([_vp, _i32, _u32, _u32, _u32, _u32, _i32, _u64, _vp], _i32),
    "spiky_grow_cuboid": ([_u32, _vp, _vp, _u32, _vp, _vp, _vp, _f32, _u64, _u32, _vp, _vp, _u64,
                           ctypes.POINTER(_u64)], _i32),
    "spiky_densify32_workspace_bytes": ([_u64], _u64),
    "spiky_count_nonzero32": ([_vp, _u64, _vp, _u64, _vp, _vp], _i32),
    "spiky_dense_to_sparse32": ([_vp, _u64, _vp, _vp, _u64, _vp, _u64, _vp, _i32, _i32, _vp], _i32),
}

# Sequence-mode entry points are bound when the library exports them.
_OPTIONAL_SIGNATURES = {
    "spiky_lut_forward_step_concat": (
        [_vp, _vp, _u32, _vp, _vp, _vp, _vp, _f32, _vp, _vp, _vp, _vp, _vp, _vp, _vp], _i32),
    "spiky_lut_backward_backprop_concat": (
        [_vp, _vp, _u32, _vp, _vp, _vp, _vp, _vp, _vp, _f64, _vp, _vp, _vp, _vp, _vp, _i32, _vp], _i32),
    "spiky_lut_forward_step_product": (
        [_vp, _vp, _u32, _u32, _vp, _vp, _vp, _vp, _u32, _u32, _i32, _f32, _vp, _vp], _i32),
    "spiky_lut_backward_backprop_product": (
        [_vp, _vp, _u32, _u32, _vp, _vp, _vp, _vp, _vp, _vp, _f64, _u32, _u32, _i32, _f32, _vp, _vp,
         _vp, _vp], _i32),
}


# include/spiky_lm.h
F32, BF16, F16 = 0, 1, 2
NORM_NONE, NORM_RMS, NORM_LAYER = 0, 1, 2


class LmResidualArgs(ctypes.Structure):
    """spiky_lm_residual_args"""
    _fields_ = [("rows", _u64), ("cols", _u64), ("res_dtype", _i32), ("act_dtype", _i32), ("post_norm", _i32),
                ("pre_norm", _i32), ("par_f32", _i32), ("gate_f32", _i32), ("residual", _vp), ("branch", _vp),
                ("residual_stride", _i64), ("branch_stride", _i64), ("post_weight", _vp), ("post_bias", _vp),
                ("pre_weight", _vp), ("pre_bias", _vp), ("gate", _vp), ("gate_rows", _u64), ("post_eps", _f64),
                ("pre_eps", _f64), ("residual_scale", _f64), ("branch_scale", _f64), ("dropout_p", _f64),
                ("seed", _u64), ("offset", _u64), ("rng", _vp), ("stats", _vp)]


class LmResidualGrads(ctypes.Structure):
    """spiky_lm_residual_grads"""
    _fields_ = [("d_out", _vp), ("d_normed", _vp), ("d_out_stride", _i64), ("d_normed_stride", _i64),
                ("d_residual", _vp), ("d_branch", _vp), ("d_post_weight", _vp), ("d_post_bias", _vp),
                ("d_pre_weight", _vp), ("d_pre_bias", _vp), ("d_gate", _vp), ("workspace", _vp),
                ("workspace_bytes", _u64)]


class LmLogitsArgs(ctypes.Structure):
    """spiky_lm_logits_args"""
    _fields_ = [("rows", _u64), ("vocab", _u64), ("logits", _vp), ("out", _vp), ("logits_stride", _i64),
                ("out_stride", _i64), ("dtype", _i32), ("out_dtype", _i32), ("tokens", _vp), ("tokens_stride", _i64),
                ("history", _u64), ("tokens_i64", _i32), ("lengths_i64", _i32), ("lengths", _vp),
                ("prompt_lengths", _vp), ("repetition", _f32), ("presence", _f32), ("frequency", _f32),
                ("temperature", _f32), ("repetition_rows", _vp), ("presence_rows", _vp), ("frequency_rows", _vp),
                ("temperature_rows", _vp), ("bias", _vp), ("bias_stride", _i64), ("bias_dtype", _i32),
                ("bias_ids", _vp), ("bias_values", _vp), ("bias_ids_stride", _i64), ("bias_values_stride", _i64),
                ("n_bias", _u64), ("bias_ids_i64", _i32), ("mask", _vp), ("mask_stride", _i64), ("mask_bits", _i32)]


# include/spiky_lm_tokens.h
class LmEmbedArgs(ctypes.Structure):
    """spiky_lm_embed_args"""
    _fields_ = [("n", _u64), ("vocab", _u64), ("cols", _u64), ("tokens_i64", _i32), ("weight_dtype", _i32),
                ("out_dtype", _i32), ("tokens", _vp), ("weight", _vp), ("weight_stride", _i64), ("scale", _f64)]


class LmBeamsArgs(ctypes.Structure):
    """spiky_lm_beams_args"""
    _fields_ = [("searches", _u64), ("beams", _u64), ("vocab", _u64), ("n", _u64), ("dtype", _i32),
                ("lengths_i64", _i32), ("logits", _vp), ("search_stride", _i64), ("beam_stride", _i64),
                ("scores", _vp), ("finished", _vp), ("lengths", _vp), ("length_penalty", _f64), ("pad", _i64),
                ("out_scores", _vp), ("out_parents", _vp), ("out_tokens", _vp)]


class LmState(ctypes.Structure):
    """spiky_lm_state"""
    _fields_ = [("in", _vp), ("out", _vp), ("runs", _u64), ("run_bytes", _u64), ("in_search", _i64),
                ("in_beam", _i64), ("in_run", _i64), ("out_search", _i64), ("out_beam", _i64), ("out_run", _i64)]


_LM_SIGNATURES = {
    "spiky_lm_last_error": ([], ctypes.c_char_p),
    "spiky_lm_dropout": ([_vp, _i64, _vp, _u64, _u64, _i32, _f64, _u64, _u64, _vp, _vp], _i32),
    "spiky_lm_residual_norm": ([ctypes.POINTER(LmResidualArgs), _vp, _vp, _vp], _i32),
    "spiky_lm_residual_norm_workspace": ([ctypes.POINTER(LmResidualArgs), ctypes.POINTER(LmResidualGrads)], _u64),
    "spiky_lm_residual_norm_backward": (
        [ctypes.POINTER(LmResidualArgs), ctypes.POINTER(LmResidualGrads), _vp], _i32),
    "spiky_lm_process_logits": ([ctypes.POINTER(LmLogitsArgs), _vp], _i32),
    "spiky_lm_embed": ([ctypes.POINTER(LmEmbedArgs), _vp, _vp], _i32),
    "spiky_lm_embed_workspace": ([ctypes.POINTER(LmEmbedArgs)], _u64),
    "spiky_lm_embed_backward": ([ctypes.POINTER(LmEmbedArgs), _vp, _i64, _vp, _vp, _u64, _vp], _i32),
    "spiky_lm_beam_select_workspace": ([ctypes.POINTER(LmBeamsArgs)], _u64),
    "spiky_lm_beam_select": ([ctypes.POINTER(LmBeamsArgs), _vp, _u64, _vp], _i32),
    "spiky_lm_reorder": ([ctypes.POINTER(LmState), _u64, _vp, _i32, _u64, _u64, _u64, _vp], _i32),
}


def exported_symbols():
    """Names of every C-ABI entry point this module binds."""
    return list(_SIGNATURES) + list(_OPTIONAL_SIGNATURES) + list(_LM_SIGNATURES)


def lib():
    """Load (once) and return the ctypes handle; raises if the library is absent."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"spiky_amd native library not found at {LIB_PATH}; build it with "
                "`python -m spiky_amd.build` (hipcc, gfx950)")
        L = ctypes.CDLL(LIB_PATH)
        for name, (args, res) in [*_SIGNATURES.items(), *_LM_SIGNATURES.items()]:
            fn = getattr(L, name)
            fn.argtypes = args
            fn.restype = res
        for name, (args, res) in _OPTIONAL_SIGNATURES.items():
            fn = getattr(L, name, None)
            if fn is not None:
                fn.argtypes = args
                fn.restype = res
        _lib = L
    return _lib


def lm():
    """The torch binding of include/spiky_lm.h and include/spiky_lm_tokens.h (csrc/lm/lm_torch.cpp,
    csrc/lm/lm_tokens_torch.cpp); raises if it is absent."""
    global _lm
    if _lm is None:
        lib()
        import torch  # noqa: F401  (its libraries are the binding's)
        try:
            from . import _lm_torch
        except ImportError as e:
            raise RuntimeError("spiky_amd's torch binding _lm_torch.so is missing or does not load; build it with "
                               f"`python -m spiky_amd.build`: {e}") from e
        _lm = _lm_torch
    return _lm


def check(status):
    """Map a C-ABI status to the reference's Python exception types."""
    if status == SPIKY_OK:
        return
    msg = lib().spiky_lut_last_error().decode("utf-8", "replace")
    if status == SPIKY_VALUE_ERROR:
        raise ValueError(msg)
    raise RuntimeError(msg)


def check_lm(status):
    """check() for the entry points of include/spiky_lm.h, which keep their own last error."""
    if status == SPIKY_OK:
        return
    msg = lib().spiky_lm_last_error().decode("utf-8", "replace")
    if status == SPIKY_VALUE_ERROR:
        raise ValueError(msg)
    raise RuntimeError(msg)
