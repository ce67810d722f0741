"""beam_select on the GPU: numbers past 64 bits, more searches than one side of a grid, values with an offset."""
import pytest
import torch

from spiky_amd import beam_select
import lm_tokens_plain as plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", [dict(n=(1 << 64) + 2), dict(n=-(1 << 64) + 2), dict(pad=1 << 63), dict(pad=-(1 << 63) - 1),
                                 dict(pad=(1 << 64) + 3)])
def test_whole_numbers_past_64_bits_are_refused(cuda_device, how):
    x, scores = torch.zeros(2, 3, 9, device=cuda_device), torch.zeros(2, 3, device=cuda_device)
    with pytest.raises(ValueError, match="must fit 64 bits"):
        beam_select(x, scores, **how)


@pytest.mark.parametrize("pad", [-1, (1 << 63) - 1, -(1 << 63)])
def test_pads_of_64_bits(cuda_device, pad):
    x, scores = torch.zeros(1, 1, 2, device=cuda_device), torch.zeros(1, 1, device=cuda_device)
    got = beam_select(x, scores, 3, finished=torch.ones(1, 1, dtype=torch.bool, device=cuda_device), pad=pad)
    assert got[2].tolist() == [[pad] * 3]


@pytest.mark.parametrize("searches", [(1 << 20) + 1, (1 << 23) + 5])
def test_many_searches(cuda_device, searches):
    """More searches than one side of a grid takes."""
    gen = torch.Generator(cuda_device).manual_seed(3)
    x = torch.randn(searches, 1, 3, generator=gen, device=cuda_device)
    scores = -torch.rand(searches, 1, generator=gen, device=cuda_device)
    got = beam_select(x, scores, 2)
    s, tokens = torch.sort((torch.log_softmax(x.double(), -1) + scores.double()[..., None])[:, 0], descending=True, stable=True)
    assert torch.equal(got[2], tokens[:, :2]) and not bool(got[1].any())
    # three exponentials and their sum, each off by a few half steps, then the score's own rounding
    assert float((got[0].double() - s[:, :2]).abs().max()) <= (48 + 3 * 2 + 16) * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0.0, -2.0, 1000.0, -60000.0])
def test_values_with_an_offset(cuda_device, dtype, offset):
    """Scores of a long search, and logits that are all large: the choice is by differences."""
    gen = torch.Generator().manual_seed(8)
    x = (torch.randn(2, 5, 20003, generator=gen) * 4 + offset).to(dtype)
    for at in (0.0, -1.5e3, -3e4, 1e7):
        scores = at - 3 * torch.rand(2, 5, generator=gen)
        finished, lengths = torch.rand(2, 5, generator=gen) < 0.3, torch.randint(1, 2000, (2, 5), generator=gen)
        for n, alpha in ((16, 0.0), (64, 0.0), (16, 0.7)):
            how = dict(finished=finished, lengths=lengths, length_penalty=alpha)
            got = beam_select(x.to(cuda_device), scores.to(cuda_device), n, **{
                k: v.to(cuda_device) if isinstance(v, torch.Tensor) else v for k, v in how.items()})
            plain.check_select(got, x, scores, n, **how)
