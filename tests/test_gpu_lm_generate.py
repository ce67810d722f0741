"""Continuations on the GPU whose rows differ in temperature, or that have nothing to choose."""
import pytest
import torch

from test_gpu_lm_model import small

pytestmark = pytest.mark.gpu


def test_each_row_has_its_own_temperature(cuda_device):
    m = small(cuda_device, residual_join=dict(pre_norm="rms"))
    prompts = torch.randint(0, 50, (4, 5), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    largest = m.generate(prompts, 12, temperature=0.0)
    mixed = m.generate(prompts, 12, generator=torch.Generator(cuda_device).manual_seed(1),
                       temperature=torch.tensor([0.0, 5.0, -1.0, 5.0], device=cuda_device))
    assert torch.equal(mixed[[0, 2]], largest[[0, 2]])
    assert not torch.equal(mixed[1], largest[1]) and not torch.equal(mixed[3], largest[3])


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_a_row_without_a_token_to_choose_raises(cuda_device, temperature):
    m = small(cuda_device, residual_join=dict(pre_norm="rms"))
    prompts = torch.randint(0, 50, (3, 5), device=cuda_device)
    mask = torch.ones(3, 50, dtype=torch.bool, device=cuda_device)
    mask[1] = False
    with pytest.raises(ValueError, match="no token"):
        m.generate(prompts, 3, temperature=temperature, mask=mask)
    mask[1, 9] = True
    assert m.generate(prompts, 3, temperature=temperature, mask=mask)[1, 5:].tolist() == [9, 9, 9]
