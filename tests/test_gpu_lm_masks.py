"""The masks of the modules' dropout on the GPU in recomputed steps."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from spiky_amd import CounterDropout, ResidualNorm, mask_counters
from test_gpu_lm_model import small

pytestmark = pytest.mark.gpu


class Net(torch.nn.Module):
    def __init__(self, device):
        super().__init__()
        self.drop = CounterDropout(0.5, seed=3)
        self.join = ResidualNorm(96, post_norm="rms", pre_norm="layer", bias=True, gate=0.5, dropout_p=0.25,
                                 seed=(1 << 63) + 9, device=device)

    def forward(self, x):
        z, h = self.join(x, self.drop(x * 2.0))
        return z + h.square()


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_recomputed_step_is_the_whole_one(cuda_device, reentrant):
    x, whole, net = torch.randn(40, 96, device=cuda_device), Net(cuda_device), Net(cuda_device)
    counters = mask_counters(net, cuda_device)
    for _ in range(3):
        results = []
        for m in (whole, net):
            v = x.clone().requires_grad_()
            y = m(v) if m is whole else checkpoint(m, v, use_reentrant=reentrant)
            m.zero_grad()
            y.sum().backward()
            results.append([y.detach(), v.grad, *(p.grad.clone() for p in m.parameters())])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        counters[:, 1] += 1
    assert net.state_dict()["join._extra_state"]["calls"] == whole.join.calls == 3


@pytest.mark.parametrize("reentrant", [True, False])
def test_a_counted_recomputation_raises(cuda_device, reentrant):
    x, net = torch.randn(4, 96, device=cuda_device, requires_grad=True), Net(cuda_device)
    y = checkpoint(net, x, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="mask_counters"):
        y.sum().backward()


def test_a_recomputed_model_is_the_whole_one(cuda_device):
    tokens = torch.randint(0, 50, (4, 8), device=cuda_device)
    join = dict(post_norm="rms", pre_norm="rms", gate=0.5)
    results = []
    for recomputed in (False, True):
        m = small(cuda_device, dropout=0.2, residual_join=join)
        if recomputed:
            mask_counters(m, cuda_device)
        y = checkpoint(m, tokens, use_reentrant=False) if recomputed else m(tokens)
        y.square().sum().backward()
        results.append([y.detach(), *(p.grad for n, p in m.named_parameters() if "_join" in n)])
    assert len(results[0]) == 13 and all(torch.equal(a, b) for a, b in zip(*results))
