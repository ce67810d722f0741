"""Gradients of gradients raise also where they are asked of what the output's gradient depends on."""
import pytest
import torch

from spiky_amd import counter_dropout, embed_tokens, residual_norm

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("unused", [False, True])
def test_gradients_of_the_outputs_gradient(cuda_device, unused):
    x = torch.randn(6, 16, device=cuda_device, requires_grad=True)
    tokens = torch.tensor([1, 5, 1], device=cuda_device)
    calls = (lambda: counter_dropout(x, 0.5, 3), lambda: residual_norm(x, pre_norm="rms")[1], lambda: embed_tokens(tokens, x))
    for call in calls:
        y = call()
        c = torch.randn_like(y, requires_grad=True)
        (dx,) = torch.autograd.grad((y * c).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
            torch.autograd.grad(dx.sum(), c, allow_unused=unused)
        # without a graph of the gradient there is nothing to raise
        (dx,) = torch.autograd.grad((call() * c).sum(), x)
        assert not dx.requires_grad
