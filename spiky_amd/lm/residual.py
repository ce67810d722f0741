"""The residual join of a block: the norm after it, dropout, gate and scales, the sum, and the
norm before the next block, in one pass over the rows."""
import torch

from .. import _native
from .common import CountedMasks, check_probability

_NORMS = (None, "rms", "layer")


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
    depend on the order in which workgroups run.  Tensors with forward-mode tangents are refused."""
    return _native.lm().residual_norm(residual, branch, post_norm, post_weight, post_bias, post_eps, gate, residual_scale,
                                      branch_scale, dropout_p, seed, offset, pre_norm, pre_weight, pre_bias, pre_eps,
                                      dtype)


class ResidualNorm(CountedMasks, torch.nn.Module):
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
        self.dropout_p = float(dropout_p)
        self.count_masks(seed)

        def parameter(there, value):
            if not there:
                return None
            return torch.nn.Parameter(torch.full((dim,), float(value), device=device, dtype=dtype))

        self.post_weight = parameter(post_norm, 1.0)
        self.post_bias = parameter(post_norm and bias, 0.0)
        self.gate = parameter(gate is not None, gate or 0.0)
        self.pre_weight = parameter(pre_norm, 1.0)
        self.pre_bias = parameter(pre_norm and bias, 0.0)

    def forward(self, residual, branch):
        p = self.dropout_p if self.training else 0.0
        seed, offset = self.next_mask(residual) if p else (0, 0)
        return residual_norm(residual, branch, post_norm=self.post_norm, post_weight=self.post_weight,
                             post_bias=self.post_bias, post_eps=self.eps, gate=self.gate,
                             residual_scale=self.residual_scale, branch_scale=self.branch_scale, dropout_p=p,
                             seed=seed, offset=offset, pre_norm=self.pre_norm,
                             pre_weight=self.pre_weight, pre_bias=self.pre_bias, pre_eps=self.eps)

    def extra_repr(self):
        return f"{self.dim}, post_norm={self.post_norm!r}, pre_norm={self.pre_norm!r}, dropout_p={self.dropout_p}"
