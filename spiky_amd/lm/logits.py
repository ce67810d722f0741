"""What happens to logits before a token is chosen: penalties, biases, temperature, masks."""
import torch

from .. import _native
from .common import DTYPES, dtype_code, on_device, require_device, stream_of


def _ids(t, name, device, rows):
    """(tensor, stride of rows, is int64) of whole numbers [rows, n], or [n] for every row."""
    require_device(t, name, device)
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"tensor {name} must have dtype int32 or int64, got {t.dtype}")
    t, stride = _by_row(t, name, rows)
    return t, stride, t.dtype == torch.int64


def _by_row(t, name, rows):
    if t.dim() == 2 and t.shape[0] != rows or t.dim() not in (1, 2):
        raise ValueError(f"{name} must be [n] or [{rows}, n], got {tuple(t.shape)}")
    if t.dim() == 1:
        return t.contiguous(), 0
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _setting(v, name, rows, device):
    """(number, tensor): one value for all rows, or a float32 tensor of one for each."""
    if not isinstance(v, torch.Tensor):
        return float(v), None
    require_device(v, name, device)
    if v.shape != (rows,):
        raise ValueError(f"{name} must be a number or have shape ({rows},), got {tuple(v.shape)}")
    if not v.is_floating_point():
        raise RuntimeError(f"tensor {name} must be floating point, got {v.dtype}")
    return 1.0, v.to(torch.float32).contiguous()


def _lengths(t, name, rows, device):
    require_device(t, name, device)
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"tensor {name} must have dtype int32 or int64, got {t.dtype}")
    if t.shape != (rows,):
        raise ValueError(f"{name} must have shape ({rows},), got {tuple(t.shape)}")
    return t.contiguous()


def process_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition_penalty=1.0,
                   presence_penalty=0.0, frequency_penalty=0.0, bias=None, bias_ids=None, bias_values=None,
                   temperature=1.0, mask=None, out=None, dtype=None):
    """Logits [B, V] made ready for the choice of each row's next token.  In this order:

        x = logits + bias + the sum of a row's bias_values at its bias_ids
        x = x / repetition_penalty where x > 0, else x * repetition_penalty,
            for entries among the row's tokens
        x = x - frequency_penalty * n - presence_penalty
            for entries that n > 0 of the row's tokens after the prompt are
        x = x / temperature              (rows of temperature 0 or less stay as they are)
        x = -inf where the mask leaves an entry out, whatever it holds; a row whose mask leaves
            nothing is all -inf

    logits: float32, bfloat16 or float16, columns contiguous, rows at any distance (the last
    positions of a [B, S, V] tensor need no copy).  tokens: int32 or int64 [B, L], of which a
    row's first `lengths` count (all, without) and of those the first `prompt_lengths` are its
    prompt (none, without); lengths beyond 0..L are taken as the nearest of these.  Tokens and
    bias ids outside 0..V-1 count nowhere.  Penalties and temperature: a number, or [B] for each
    row.  bias: [V] or [B, V], any of the three types.  bias_ids: [K] or [B, K] with float32
    bias_values of that shape; ids that repeat add up, in their order.  mask: bool [V] or [B, V],
    True where allowed, or int32 [ceil(V / 32)] or [B, ceil(V / 32)] with entry v in bit v % 32 of
    word v // 32.

    Returns a tensor of the logits' type, or of `dtype` float32, or `out`, which may be `logits`.
    There is no gradient."""
    require_device(logits, "logits")
    code, device = dtype_code(logits, "logits"), logits.device
    if logits.dim() != 2:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1:
        if out is logits:
            raise ValueError("logits that are written in place need contiguous columns")
        logits = logits.contiguous()
    if out is None:
        dtype = logits.dtype if dtype is None else dtype
        if dtype not in (logits.dtype, torch.float32):
            raise ValueError(f"dtype must be {logits.dtype} or float32, got {dtype}")
        out = torch.empty((rows, vocab), dtype=dtype, device=device)
    else:
        require_device(out, "out", device)
        if out.shape != logits.shape or out.dtype not in (logits.dtype, torch.float32) or \
                (dtype is not None and dtype != out.dtype):
            raise ValueError(f"out must be {tuple(logits.shape)} of {dtype or f'{logits.dtype} or float32'}")
        if vocab > 1 and out.stride(1) != 1:
            raise ValueError("out must have contiguous columns")
        if out.data_ptr() == logits.data_ptr() and (out.dtype != logits.dtype or out.stride(0) != logits.stride(0)):
            raise ValueError("out may be logits, but not another view of them")
    a = _native.LmLogitsArgs()
    a.rows, a.vocab = rows, vocab
    a.logits, a.logits_stride, a.dtype = logits.data_ptr(), logits.stride(0), code
    a.out, a.out_stride, a.out_dtype = out.data_ptr(), out.stride(0), DTYPES[out.dtype]
    keep = []
    if tokens is not None:
        if tokens.dim() != 2:
            raise ValueError(f"tokens must be [{rows}, L], got {tuple(tokens.shape)}")
        tokens, a.tokens_stride, a.tokens_i64 = _ids(tokens, "tokens", device, rows)
        a.history = tokens.shape[1]
        a.tokens = tokens.data_ptr() if a.history else None
        if lengths is not None:
            lengths = _lengths(lengths, "lengths", rows, device)
            a.lengths, a.lengths_i64 = lengths.data_ptr(), lengths.dtype == torch.int64
        if prompt_lengths is not None:
            prompt_lengths = _lengths(prompt_lengths, "prompt_lengths", rows, device)
            if lengths is not None and prompt_lengths.dtype != lengths.dtype:
                prompt_lengths = prompt_lengths.to(lengths.dtype)
            a.prompt_lengths, a.lengths_i64 = prompt_lengths.data_ptr(), prompt_lengths.dtype == torch.int64
        keep += [tokens, lengths, prompt_lengths]
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths need tokens")
    a.repetition, t = _setting(repetition_penalty, "repetition_penalty", rows, device)
    if t is not None:
        a.repetition_rows = t.data_ptr()
        keep.append(t)
    elif a.repetition <= 0.0:
        raise ValueError(f"repetition_penalty must be positive, got {repetition_penalty}")
    a.presence, t = _setting(presence_penalty, "presence_penalty", rows, device)
    if t is not None:
        a.presence_rows = t.data_ptr()
        keep.append(t)
    a.frequency, t = _setting(frequency_penalty, "frequency_penalty", rows, device)
    if t is not None:
        a.frequency_rows = t.data_ptr()
        keep.append(t)
    a.temperature, t = _setting(temperature, "temperature", rows, device)
    if t is not None:
        a.temperature_rows = t.data_ptr()
        keep.append(t)
    if bias is not None:
        require_device(bias, "bias", device)
        a.bias_dtype = dtype_code(bias, "bias")
        bias, a.bias_stride = _by_row(bias, "bias", rows)
        if bias.shape[-1] != vocab:
            raise ValueError(f"bias must be [{vocab}] or [{rows}, {vocab}], got {tuple(bias.shape)}")
        a.bias = bias.data_ptr()
        keep.append(bias)
    if (bias_ids is None) != (bias_values is None):
        raise ValueError("bias_ids and bias_values go together")
    if bias_ids is not None:
        bias_ids, a.bias_ids_stride, a.bias_ids_i64 = _ids(bias_ids, "bias_ids", device, rows)
        require_device(bias_values, "bias_values", device)
        if bias_values.shape != bias_ids.shape:
            raise ValueError(f"bias_values must have the shape of bias_ids, {tuple(bias_ids.shape)}")
        if bias_values.dtype != torch.float32:
            raise RuntimeError(f"tensor bias_values must be float32, got {bias_values.dtype}")
        bias_values, a.bias_values_stride = _by_row(bias_values, "bias_values", rows)
        a.n_bias = bias_ids.shape[-1]
        if a.n_bias:
            a.bias_ids, a.bias_values = bias_ids.data_ptr(), bias_values.data_ptr()
        keep += [bias_ids, bias_values]
    if mask is not None:
        require_device(mask, "mask", device)
        if mask.dtype not in (torch.bool, torch.int32):
            raise RuntimeError(f"tensor mask must have dtype bool or int32, got {mask.dtype}")
        a.mask_bits = mask.dtype == torch.int32
        mask, a.mask_stride = _by_row(mask, "mask", rows)
        need = (vocab + 31) // 32 if a.mask_bits else vocab
        if mask.shape[-1] != need:
            raise ValueError(f"mask must be [{need}] or [{rows}, {need}], got {tuple(mask.shape)}")
        a.mask = mask.data_ptr()
        keep.append(mask)
    with on_device(device):
        _native.check_lm(_native.lib().spiky_lm_process_logits(a, stream_of(device)))
    return out
