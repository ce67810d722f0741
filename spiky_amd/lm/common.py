"""What the operators' Python sides share: checks of tensors, rows, streams."""
import contextlib

import torch

from .. import _native

DTYPES = {torch.float32: _native.F32, torch.bfloat16: _native.BF16, torch.float16: _native.F16}
_MASK64 = (1 << 64) - 1
_no_guard = contextlib.nullcontext()


def dtype_code(t, name):
    code = DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"tensor {name} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def require_device(t, name, device=None):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"tensor {name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise RuntimeError(f"tensor {name} must be on CUDA")
    if device is not None and t.device != device:
        raise RuntimeError(f"tensor {name} must be on {device}, got {t.device}")


def on_device(device):
    """A guard for launches on `device`, which costs nothing where it is the current one."""
    return _no_guard if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream_of(device):
    return torch.cuda.current_stream(device).cuda_stream


def as_rows(t):
    """(tensor, elements from row to row): the tensor seen as rows of its last dimension.  Rows
    at one distance with contiguous columns stay where they are; others are copied."""
    if t.is_contiguous():
        return t, (t.shape[-1] if t.dim() else 1)
    if t.dim() and t.stride(-1) == 1 and t.numel():
        step = None  # the distance of rows, from the innermost dimension of more than one
        for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if step is None:
                step, reach = stride, stride * size
            elif stride == reach:
                reach = stride * size
            else:
                break
        else:
            return t, (step if step is not None else t.shape[-1])
    return t.contiguous(), t.shape[-1]


def generator_state(seed, offset, device):
    """(seed, offset, rng): two numbers of 64 bits, or a device tensor that holds them."""
    if isinstance(seed, torch.Tensor):
        require_device(seed, "seed", device)
        if seed.dtype != torch.int64 or seed.numel() != 2 or not seed.is_contiguous():
            raise RuntimeError("tensor seed must be a contiguous int64 tensor of [seed, offset]")
        if offset:
            raise ValueError("offset is the second element of a seed tensor")
        return 0, 0, seed
    return int(seed) & _MASK64, int(offset) & _MASK64, None


def check_probability(p):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability must be between 0 and 1, got {p}")
