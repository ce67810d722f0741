"""Tensors whose sign torch keeps beside their memory: imaginary parts of conjugates."""
import pytest
import torch

from spiky_amd import counter_dropout, process_logits, residual_norm

pytestmark = pytest.mark.gpu


def turned(x):
    """-x in x's memory, a view whose sign is not in it."""
    y = torch._neg_view(x)
    assert y.is_neg() and y.data_ptr() == x.data_ptr()
    return y


def test_one_imaginary_part(cuda_device):
    z = torch.full((1, 1), 2.0 + 3.0j, device=cuda_device).conj()
    assert float(counter_dropout(z.imag, 0.0, 1)) == -3.0
    assert float(residual_norm(z.imag, z.real)[0]) == -1.0
    assert float(process_logits(z.imag)) == -3.0


def test_values_gradients_and_parameters_have_their_signs(cuda_device):
    gen = torch.Generator(cuda_device).manual_seed(1)
    r, a, dz, dh = (torch.randn(6, 64, generator=gen, device=cuda_device) for _ in range(4))
    w, b, g = (torch.randn(64, generator=gen, device=cuda_device) for _ in range(3))

    def step(r, a, w, b, g, dz, dh, turn):
        leaves = [t.clone().requires_grad_() for t in (r, a, w, b, g)]
        v = [turn(t) for t in leaves]
        z, h = residual_norm(v[0], v[1], post_norm="rms", post_weight=v[2], gate=v[4], pre_norm="layer", pre_bias=v[3])
        return [z.detach(), h.detach(), *torch.autograd.grad([z, h], leaves, [turn(dz), turn(dh)])]

    for x, y in zip(step(r, a, w, b, g, dz, dh, turned), step(r, a, w, b, g, dz, dh, torch.neg)):
        assert torch.equal(x, y)
    x = r.clone().requires_grad_()
    y = counter_dropout(turned(x), 0.5, 1)
    assert torch.equal(y, counter_dropout(-r, 0.5, 1))
    assert torch.equal(torch.autograd.grad(y, x, turned(dz))[0], -counter_dropout(-dz, 0.5, 1))


def test_logits_biases_and_results(cuda_device):
    x, bias = torch.randn(3, 50, device=cuda_device), torch.randn(50, device=cuda_device)
    heat = torch.full((3,), -0.5, device=cuda_device)
    want = process_logits(-x, bias=-bias, temperature=-heat)
    assert torch.equal(process_logits(turned(x), bias=turned(bias), temperature=turned(heat)), want)
    out = turned(torch.zeros(3, 50, device=cuda_device))
    with pytest.raises(ValueError, match="signs"):
        process_logits(x, out=out)
    with pytest.raises(ValueError, match="signs"):
        process_logits(out, out=out)
