"""The residual join of a block: the norm after it, dropout, gate and scales, the sum, and the
norm before the next block, in one pass over the rows."""
import torch

from .. import _native
from .common import as_rows, check_probability, dtype_code, generator_state, on_device, require_device, stream_of

_NORMS = {None: _native.NORM_NONE, "rms": _native.NORM_RMS, "layer": _native.NORM_LAYER}


def _ptr(t):
    return None if t is None else t.data_ptr()


class _How:
    """What a call has beside its tensors."""
    __slots__ = ("post", "pre", "post_eps", "pre_eps", "alpha", "beta", "p", "seed", "offset", "gate_rows", "dtype")


def _args(how, res, branch, post_weight, post_bias, gate, pre_weight, pre_bias, rng, stats):
    """The C arguments, and the tensors that must outlive the call."""
    cols = res.shape[-1]
    rows = res.numel() // cols if cols else 0
    res, res_stride = as_rows(res)
    act = how.dtype
    branch_stride = 0
    if branch is not None:
        branch, branch_stride = as_rows(branch)
    par = next((t for t in (post_weight, post_bias, pre_weight, pre_bias) if t is not None), None)
    keep = (res, branch)
    return _native.LmResidualArgs(
        rows, cols, dtype_code(res, "residual"), act, how.post, how.pre,
        par is not None and par.dtype == torch.float32, gate is not None and gate.dtype == torch.float32,
        res.data_ptr(), _ptr(branch), res_stride, branch_stride, _ptr(post_weight), _ptr(post_bias),
        _ptr(pre_weight), _ptr(pre_bias), _ptr(gate), how.gate_rows, how.post_eps, how.pre_eps, how.alpha, how.beta,
        how.p, how.seed, how.offset, _ptr(rng), _ptr(stats)), keep


_TORCH = {_native.F32: torch.float32, _native.BF16: torch.bfloat16, _native.F16: torch.float16}


def _forward(how, res, branch, post_weight, post_bias, gate, pre_weight, pre_bias, rng, stats):
    args, keep = _args(how, res, branch, post_weight, post_bias, gate, pre_weight, pre_bias, rng, stats)
    out = None if branch is None else torch.empty(res.shape, dtype=res.dtype, device=res.device)
    normed = None
    if how.pre:
        normed = torch.empty(res.shape, dtype=_TORCH[how.dtype], device=res.device)
    with on_device(res.device):
        _native.check_lm(_native.lib().spiky_lm_residual_norm(args, _ptr(out), _ptr(normed), stream_of(res.device)))
    return out, normed


class _ResidualNormFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, how, rng, res, branch, post_weight, post_bias, gate, pre_weight, pre_bias):
        cols = res.shape[-1]
        stats = torch.empty((res.numel() // cols if cols else 0, 4), dtype=torch.float32, device=res.device)
        out, normed = _forward(how, res, branch, post_weight, post_bias, gate, pre_weight, pre_bias, rng, stats)
        ctx.how = how
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(rng, stats, res, branch, post_weight, post_bias, gate, pre_weight, pre_bias)
        return out, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out, d_normed):
        rng, stats, res, *tensors = ctx.saved_tensors
        branch, post_weight, post_bias, gate, pre_weight, pre_bias = tensors
        if d_out is None and d_normed is None:
            return (None,) * 9
        args, keep = _args(ctx.how, res, *tensors, rng, stats)

        def like(t, i, zero=False):
            if t is None or not ctx.needs_input_grad[i]:
                return None
            # parameters of a pre norm whose output has no gradient get none written
            make = torch.zeros if zero or not args.rows else torch.empty
            return make(t.shape, dtype=t.dtype, device=t.device)

        idle = d_normed is None
        d_res, d_branch = like(res, 2), like(branch, 3)
        d_post_weight, d_post_bias, d_gate = like(post_weight, 4), like(post_bias, 5), like(gate, 6)
        d_pre_weight, d_pre_bias = like(pre_weight, 7, idle), like(pre_bias, 8, idle)
        out_stride = normed_stride = 0
        if d_out is not None:
            d_out, out_stride = as_rows(d_out)
        if d_normed is not None:
            d_normed, normed_stride = as_rows(d_normed)
        grads = _native.LmResidualGrads(
            _ptr(d_out), _ptr(d_normed), out_stride, normed_stride, _ptr(d_res), _ptr(d_branch),
            _ptr(d_post_weight), _ptr(d_post_bias), None if idle else _ptr(d_pre_weight),
            None if idle else _ptr(d_pre_bias), _ptr(d_gate), None, 0)
        lib = _native.lib()
        grads.workspace_bytes = lib.spiky_lm_residual_norm_workspace(args, grads)
        workspace = torch.empty(max(grads.workspace_bytes, 1), dtype=torch.uint8, device=res.device)
        grads.workspace = workspace.data_ptr()
        with on_device(res.device):
            _native.check_lm(lib.spiky_lm_residual_norm_backward(args, grads, stream_of(res.device)))
        return None, None, d_res, d_branch, d_post_weight, d_post_bias, d_gate, d_pre_weight, d_pre_bias


def _norm_kind(norm, weight, bias, name):
    if norm not in _NORMS:
        raise ValueError(f"{name}_norm must be None, 'rms' or 'layer', got {norm!r}")
    if norm is None and (weight is not None or bias is not None):
        raise ValueError(f"{name}_weight and {name}_bias need a {name}_norm")
    return _NORMS[norm]


def _gate_rows(gate, shape):
    """(gate, consecutive rows that share one of its rows).  Gates that are one row, one row for
    each index of some leading dimensions, or of the full shape are read as they are; others that
    broadcast to the shape are expanded to it."""
    lead = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape)
    if len(lead) != len(shape) or any(g not in (1, s) for g, s in zip(lead, shape)):
        raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
    k = len(shape) - 1
    while k > 0 and lead[k - 1] == 1:
        k -= 1
    if lead[-1] != shape[-1] or lead[:k] != tuple(shape[:k]):
        return gate.expand(shape).contiguous(), 1
    share = 1
    for s in shape[k:-1]:
        share *= s
    return gate.contiguous(), share


def residual_norm(residual, branch=None, *, post_norm=None, post_weight=None, post_bias=None, post_eps=1e-5,
                  gate=None, residual_scale=1.0, branch_scale=1.0, dropout_p=0.0, seed=0, offset=0,
                  pre_norm=None, pre_weight=None, pre_bias=None, pre_eps=1e-5, dtype=None):
    """(stream, normed) of a block's residual join:

        v      = post_norm(branch) * post_weight + post_bias
        stream = residual_scale * residual + branch_scale * gate * dropout(v)
        normed = pre_norm(stream) * pre_weight + pre_bias

    over the last dimension.  Norms are None, "rms" (x / sqrt(mean(x^2) + eps)) or "layer"
    ((x - mean) / sqrt(var + eps)); parameters and the gate may be None.  `normed` is of the sum
    before it is rounded to the residual's type, and None without a pre_norm.  Without a branch,
    `stream` is `residual` itself and only the norm is computed.

    residual, branch: one shape [..., D] on a HIP device.  The branch is float32, bfloat16 or
    float16 and the residual has its type or float32; `normed` has the branch's type (without a
    branch: `dtype`, else the residual's).  Norm parameters [D] are all float32 or all of the
    branch's type; so is the gate, of any shape that broadcasts to the branch's: [D], [B, 1, D]
    and full gates are read as they are.  dropout_p, seed and offset are counter_dropout's, over
    the branch.  All sums and intermediate values are 32-bit; gradients, of every tensor, do not
    depend on the order in which workgroups run."""
    require_device(residual, "residual")
    res_code = dtype_code(residual, "residual")
    if residual.dim() == 0:
        raise ValueError("residual must have at least one dimension")
    device, shape = residual.device, residual.shape
    how = _How()
    how.post = _norm_kind(post_norm, post_weight, post_bias, "post")
    how.pre = _norm_kind(pre_norm, pre_weight, pre_bias, "pre")
    if branch is None:
        if post_norm is not None or gate is not None or dropout_p or residual_scale != 1.0:
            raise ValueError("a post_norm, gate, dropout or scale needs a branch")
        if pre_norm is None:
            raise ValueError("neither a branch nor a pre_norm")
        dtype = residual.dtype if dtype is None else dtype
    else:
        require_device(branch, "branch", device)
        dtype_code(branch, "branch")
        if branch.shape != shape:
            raise ValueError(f"branch of shape {tuple(branch.shape)} for a residual of {tuple(shape)}")
        if dtype is not None and dtype != branch.dtype:
            raise ValueError("dtype is the branch's where there is one")
        dtype = branch.dtype
    how.dtype = _native.F32 if dtype is torch.float32 else _native.BF16 if dtype is torch.bfloat16 else \
        _native.F16 if dtype is torch.float16 else None
    if how.dtype is None or res_code not in (how.dtype, _native.F32):
        raise RuntimeError(f"a residual of {residual.dtype} does not go with a branch of {dtype}")
    check_probability(dropout_p)
    parameters = [post_weight, post_bias, pre_weight, pre_bias]
    first = None
    for i, (t, name) in enumerate(zip(parameters, ("post_weight", "post_bias", "pre_weight", "pre_bias"))):
        if t is None:
            continue
        require_device(t, name, device)
        if t.shape != shape[-1:]:
            raise ValueError(f"{name} must have shape ({shape[-1]},), got {tuple(t.shape)}")
        if t.dtype not in (torch.float32, dtype):
            raise RuntimeError(f"tensor {name} must be float32 or {dtype}, got {t.dtype}")
        if first is None:
            first = t.dtype
        elif t.dtype != first:
            raise RuntimeError("the norms' parameters must have one type")
        parameters[i] = t.contiguous()
    post_weight, post_bias, pre_weight, pre_bias = parameters
    how.gate_rows = 1
    if gate is not None:
        require_device(gate, "gate", device)
        if gate.dtype not in (torch.float32, dtype):
            raise RuntimeError(f"tensor gate must be float32 or {dtype}, got {gate.dtype}")
        gate, how.gate_rows = _gate_rows(gate, shape)
    how.post_eps, how.pre_eps = float(post_eps), float(pre_eps)
    how.alpha, how.beta, how.p = float(residual_scale), float(branch_scale), float(dropout_p)
    how.seed, how.offset, rng = generator_state(seed, offset, device) if how.p else (0, 0, None)
    tensors = (residual, branch, post_weight, post_bias, gate, pre_weight, pre_bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        out, normed = _ResidualNormFN.apply(how, rng, *tensors)
    else:
        out, normed = _forward(how, *tensors, rng, None)
    return (residual if branch is None else out), normed


class ResidualNorm(torch.nn.Module):
    """The residual join of one block, with its parameters.

    post_norm, pre_norm: None, "rms" or "layer" over `dim` features, each with a weight (from 1)
    and, with `bias`, a bias (from 0).  gate: the initial value of a learned gate of `dim`
    features, or None.  dropout_p: dropout of the branch in training, call number n with
    offset n, as in CounterDropout."""

    def __init__(self, dim, post_norm=None, pre_norm=None, bias=False, gate=None, residual_scale=1.0,
                 branch_scale=1.0, dropout_p=0.0, seed=0, eps=1e-5, device=None, dtype=None):
        super().__init__()
        check_probability(dropout_p)
        for norm in (post_norm, pre_norm):
            if norm not in _NORMS:
                raise ValueError(f"a norm must be None, 'rms' or 'layer', got {norm!r}")
        self.dim, self.post_norm, self.pre_norm = dim, post_norm, pre_norm
        self.residual_scale, self.branch_scale, self.eps = residual_scale, branch_scale, eps
        self.dropout_p, self.seed, self.calls = float(dropout_p), int(seed), 0

        def parameter(there, value):
            if not there:
                return None
            return torch.nn.Parameter(torch.full((dim,), float(value), device=device, dtype=dtype))

        self.post_weight = parameter(post_norm, 1.0)
        self.post_bias = parameter(post_norm and bias, 0.0)
        self.gate = parameter(gate is not None, gate or 0.0)
        self.pre_weight = parameter(pre_norm, 1.0)
        self.pre_bias = parameter(pre_norm and bias, 0.0)

    def get_extra_state(self):
        return {"seed": self.seed, "calls": self.calls}

    def set_extra_state(self, state):
        self.seed, self.calls = int(state["seed"]), int(state["calls"])

    def forward(self, residual, branch):
        p = self.dropout_p if self.training else 0.0
        if p:
            self.calls += 1
        return residual_norm(residual, branch, post_norm=self.post_norm, post_weight=self.post_weight,
                             post_bias=self.post_bias, post_eps=self.eps, gate=self.gate,
                             residual_scale=self.residual_scale, branch_scale=self.branch_scale, dropout_p=p,
                             seed=self.seed, offset=self.calls, pre_norm=self.pre_norm,
                             pre_weight=self.pre_weight, pre_bias=self.pre_bias, pre_eps=self.eps)

    def extra_repr(self):
        return f"{self.dim}, post_norm={self.post_norm!r}, pre_norm={self.pre_norm!r}, dropout_p={self.dropout_p}"
