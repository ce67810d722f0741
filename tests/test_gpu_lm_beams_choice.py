"""beam_select on the GPU, each chosen (beam, token) held to its own score, rank and order."""
import math

import pytest
import torch

from spiky_amd import beam_select
from lm_beams_choice import check_choice

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16


def run(device, x, scores, n, **how):
    to = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in how.items()}
    check_choice(beam_select(x.to(device), scores.to(device), n, **to), x, scores, n, **how)


@pytest.mark.parametrize("dtype", [F, B, H])
@pytest.mark.parametrize("searches,beams,vocab,n", [
    (1, 1, 1, 5), (2, 3, 2, 6), (3, 2, 7, 4), (2, 4, 255, 8), (70, 1, 130, 1), (1, 64, 300, 64), (5, 3, 4097, 5), (2, 5, 8193, 10),
    (3, 2, 20001, 64), (1, 33, 9000, 40), (2, 8, 50001, 16), (1, 2, 262147, 64), (9, 16, 8192, 32)])
@pytest.mark.parametrize("offset", [0.0, -2000.0])
def test_each_place(cuda_device, dtype, searches, beams, vocab, n, offset):
    gen = torch.Generator().manual_seed(21)
    x = (torch.randn(searches, beams, vocab, generator=gen) * 4).to(dtype)
    scores = offset - 10 * torch.rand(searches, beams, generator=gen)
    run(cuda_device, x, scores, n)
    finished, lengths = torch.rand(searches, beams, generator=gen) < 0.4, torch.randint(0, 30, (searches, beams), generator=gen)
    for alpha in (0.8, 8.0, -1.0):
        run(cuda_device, x, scores, n, finished=finished, pad=vocab // 2, lengths=lengths, length_penalty=alpha)
    run(cuda_device, x.masked_fill(torch.rand(vocab, generator=gen) < 0.7, -math.inf), scores, n)


def test_few_candidates_unknown_and_dead_beams(cuda_device):
    gen = torch.Generator().manual_seed(22)
    x, scores = torch.randn(4, 3, 9001, generator=gen), -torch.rand(4, 3, generator=gen)
    x[0, 1, 77], x[1, 0, 9000], x[2, :, 5:] = math.nan, math.inf, -math.inf
    scores[0, 0] = scores[3, 1] = -math.inf
    scores[3, 2] = math.nan
    run(cuda_device, x, scores, 20)
    run(cuda_device, x, scores, 20, finished=torch.tensor([[1, 0, 1], [0, 1, 1], [1, 1, 0], [0, 0, 1]], dtype=torch.bool), pad=-1)


def test_a_few_values_everywhere(cuda_device):
    for vocab in (40, 9000, 40000):
        x = ((torch.arange(vocab) * 7 % 5).float() - 2).expand(2, 4, vocab).contiguous()
        for dtype in (F, B):
            run(cuda_device, x.to(dtype), torch.tensor([[0.0, -1.0, -1.0, -2.0], [-5.0] * 4]), 64)
