"""What the language-model operators say of derivatives that they do not have; checked before the device is."""
import pytest
import torch
from torch.autograd import forward_ad

from spiky_amd import counter_dropout, process_logits, residual_norm


def test_tangents_are_refused():
    """Forward-mode derivatives: a result without a tangent would count as constant."""
    x, w = torch.randn(4, 8), torch.ones(8)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: counter_dropout(dual(x), 0.5, 1), lambda: residual_norm(dual(x), pre_norm="rms")]
        calls += [lambda n=n: residual_norm(x, **{**dict(branch=x, post_norm="rms", pre_norm="rms"), n: dual(x if n == "branch" else w)})
                  for n in ("branch", "post_weight", "post_bias", "gate", "pre_weight", "pre_bias")]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        counter_dropout(forward_ad.unpack_dual(x).primal, 0.5, 1)


def test_traces_are_refused():
    """torch.jit.trace would keep the results of its example inputs as constants."""
    x = torch.randn(4, 8)
    for call in (lambda x: counter_dropout(x, 0.5, 1), lambda x: residual_norm(x, x, pre_norm="rms")[1],
                 lambda x: process_logits(x, temperature=2.0)):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, x)
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call(x)
