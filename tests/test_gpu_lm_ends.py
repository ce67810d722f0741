"""Quotients of process_logits by temperatures and penalties near the ends of float32."""
import pytest
import torch

from spiky_amd import process_logits
from test_gpu_lm_logits import STEPS
import lm_plain

pytestmark = pytest.mark.gpu


def divisors(sign=1.0):
    """Numbers of every size, subnormal ones among them, each with a fraction of many bits."""
    gen = torch.Generator().manual_seed(3)
    e = torch.arange(-149, 128, dtype=torch.float64)
    v = sign * torch.exp2(e) * (1.0 + 0.999 * torch.rand(e.shape, generator=gen, dtype=torch.float64))
    v = v.float()
    return v[torch.isfinite(v) & (v != 0)]


def logits(d):
    """For each divisor values whose quotients are near 1, and values of every size."""
    gen = torch.Generator().manual_seed(4)
    near = (d.double().abs()[:, None] * torch.exp2(torch.rand(len(d), 24, generator=gen, dtype=torch.float64) * 8 - 4)).float()
    far = torch.exp2(torch.rand(len(d), 40, generator=gen) * 250 - 125) * (torch.rand(len(d), 40, generator=gen).round() * 2 - 1)
    return torch.cat([near, -near, far], 1).clamp(-3.0e38, 3.0e38)


def check(got, want, size):
    """STEPS half steps of each quotient, which overflow where the quotient does."""
    want = want.float().double()  # past the largest: infinite
    finite = torch.isfinite(want)
    assert torch.equal(got.cpu().double()[~finite], want[~finite])
    lm_plain.near(got.cpu()[finite], want[finite], size[finite], STEPS)


def test_temperatures_of_every_size(cuda_device):
    d = divisors()
    x = logits(d)
    want, size = lm_plain.logits(x, temperature=d)
    check(process_logits(x.to(cuda_device), temperature=d.to(cuda_device)), want, size)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_penalties_of_every_size(cuda_device, sign):
    d = divisors(sign)
    x = logits(d)
    tokens = torch.arange(x.shape[1]).repeat(len(d), 1)
    r, v = d.double()[:, None], x.double()
    want = torch.where(v > 0, v / r, v * r)
    got = process_logits(x.to(cuda_device), tokens=tokens.to(cuda_device), repetition_penalty=d.to(cuda_device))
    check(got, want, want.abs())
