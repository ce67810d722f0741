"""The masks of CounterDropout and ResidualNorm in recomputed and captured steps, on the CPU: plain operators in the
place of the library's."""
import copy
import sys

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import spiky_amd
from spiky_amd import CounterDropout, ResidualNorm
import lm_plain


def plain_dropout(x, p, seed, offset=0):
    if isinstance(seed, torch.Tensor):
        assert seed.dtype == torch.int64 and seed.shape == (2,) and seed.is_contiguous() and offset == 0
        seed, offset = seed.tolist()
    keep = lm_plain.kept(x.numel() // x.shape[-1], x.shape[-1], p, seed % (1 << 64), offset).reshape(x.shape)
    return torch.where(keep, x / (1 - p), 0.0)


def plain_residual(residual, branch, *, dropout_p, seed, offset, **how):
    stream = residual + (plain_dropout(branch, dropout_p, seed, offset) if dropout_p else branch)
    return stream, None


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(sys.modules[CounterDropout.__module__], "counter_dropout", plain_dropout)
    monkeypatch.setattr(sys.modules[ResidualNorm.__module__], "residual_norm", plain_residual)


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.drop, self.join = CounterDropout(0.5, seed=3), ResidualNorm(16, dropout_p=0.25, seed=(1 << 63) + 9)

    def forward(self, x):
        return self.join(x, self.drop(x * 2.0))[0] ** 2


def step(net, x, how):
    """The output and the gradient of a step; how: whether the net is recomputed, and by which of torch's ways."""
    x = x.detach().requires_grad_()
    y = net(x) if how == "whole" else checkpoint(net, x, use_reentrant=how == "reentrant")
    (dx,) = torch.autograd.grad(y.sum(), x) if how != "reentrant" else (torch.autograd.backward(y.sum()), x.grad)[1:]
    return y.detach(), dx


@pytest.mark.parametrize("how", ["reentrant", "replayed"])
def test_a_recomputed_call_has_the_first_ones_mask(how):
    """Three steps, recomputed, are the steps of a net that is not; a step's masks are new."""
    x, nets = torch.randn(4, 16), (Net(), Net())
    counters = spiky_amd.mask_counters(nets[1], "cpu")
    assert counters.tolist() == [[3, 1], [9 - (1 << 63), 1]]
    seen = []
    for _ in range(3):
        want, got = step(nets[0], x, "whole"), step(nets[1], x, how)
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        seen.append(got[0])
        counters[:, 1] += 1
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


@pytest.mark.parametrize("how", ["reentrant", "replayed"])
def test_a_recomputed_call_that_is_counted_raises(how):
    """Counted again, it would have the next mask, and the gradient another one than the output."""
    net, x = Net(), torch.randn(4, 16)
    with pytest.raises(RuntimeError, match="mask_counters"):
        step(net, x, how)
    assert (net.drop.calls, net.join.calls) == (1, 1)
    step(net.eval(), x, how)


def test_counters_and_numbers_are_one_state():
    """What one kind of state saves the other goes on from; counters are written in place."""
    x, numbered, counted = torch.randn(4, 16), Net(), Net()
    counters = spiky_amd.mask_counters(counted, "cpu")
    for _ in range(2):
        numbered(x)
        counters[:, 1] += 1
    assert numbered.state_dict()["drop._extra_state"] == counted.state_dict()["drop._extra_state"] == {"seed": 3, "calls": 2}
    want = numbered(x)
    assert torch.equal(counted(x), want)
    other = Net()
    rows = spiky_amd.mask_counters(other, "cpu")
    other.load_state_dict(counted.state_dict())
    assert torch.equal(rows, counters) and torch.equal(other(x), want)
    # copies count for themselves: nothing advances a copy of a counter
    for other in (copy.deepcopy(counted), torch.nn.Sequential(counted)[0]):
        assert torch.equal(other(x), want)
    twin = copy.deepcopy(counted)
    assert twin.drop.counter is None and twin.drop.calls == 2 and counted.drop.counter is not None
    assert torch.equal(spiky_amd.mask_counters(counted, "cpu"), counters)
    assert spiky_amd.mask_counters(torch.nn.Linear(2, 2), "cpu").shape == (0, 2)


def test_a_captured_call_that_is_counted_raises(monkeypatch):
    """Its number would be part of the graph: every replay would drop the same elements."""
    class Captured(torch.Tensor):
        is_cuda = True

    x, capturing = torch.randn(4, 16).as_subclass(Captured), [True]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    drop, join = CounterDropout(0.5), ResidualNorm(16, dropout_p=0.5)
    calls = (lambda: drop(x), lambda: join(x, x))
    for call in calls:
        with pytest.raises(RuntimeError, match="mask_counters"):
            call()
    assert (drop.calls, join.calls) == (0, 0)
    spiky_amd.mask_counters(drop, "cpu"), spiky_amd.mask_counters(join, "cpu")
    for call in calls:
        call()
    capturing[0] = False
    CounterDropout(0.5)(x)
    capturing[0] = True
    join.eval()(x, x), drop.eval()(x)
