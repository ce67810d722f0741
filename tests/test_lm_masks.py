"""The masks of CounterDropout and ResidualNorm in recomputed and captured steps, on the CPU: plain operators in the
place of the library's."""
import copy
import sys

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import spiky_amd
from spiky_amd import CounterDropout, LUTTransformer, ResidualNorm
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


JOIN = dict(vocab_size=20, embedding_dim=16, context_size=4, positional_dim=2, num_layers=2, num_heads=2, n_detectors=4,
            n_anchors_per_detector=3, dropout=0.25, residual_join={})


def joins(model):
    return [m for m in model.modules() if isinstance(m, ResidualNorm)]


def test_ranks_of_equal_weights_have_masks_of_their_own():
    """dropout_seed is the masks' alone; without it they follow seed, as they did."""
    one, two, plain = (LUTTransformer(seed=5, **kw, **JOIN) for kw in (dict(dropout_seed=1), dict(dropout_seed=2), {}))
    for (name, a), b in zip(one.state_dict().items(), two.state_dict().values()):
        assert name.endswith("_extra_state") or torch.equal(a, b), name
    for p, q in zip(one._lut_layers(), two._lut_layers()):
        assert torch.equal(p._detector_anchors, q._detector_anchors)
    assert not {m.seed for m in joins(one)} & {m.seed for m in joins(two)}
    assert len({m.seed for m in joins(one)}) == 4
    assert [m.seed for m in joins(plain)] == [(5 << 16) + n for n in range(4)]
    assert [m.seed for m in joins(LUTTransformer(**JOIN))] == list(range(4))


@pytest.mark.parametrize("counted", [True, False])
def test_a_rank_keeps_its_masks_over_another_ones_checkpoint(counted):
    """A state dict brings its own seeds; seed_dropout gives them back, and leaves the numbers of the calls."""
    one, two = (LUTTransformer(seed=5, dropout_seed=n, **JOIN) for n in (1, 2))
    if counted:
        counters = spiky_amd.mask_counters(two, "cpu")
    want = [m.get_extra_state()["seed"] for m in joins(two)]
    for m in joins(one):
        m.calls = 7
    two.load_state_dict(one.state_dict())
    two.seed_dropout(2)
    assert [m.get_extra_state() for m in joins(two)] == [{"seed": s, "calls": 7} for s in want]
    if counted:
        assert counters.tolist() == [[s, 8] for s in want]


@pytest.mark.parametrize("reentrant", [True, False])
def test_counters_that_move_before_the_backward_pass_raise(reentrant):
    """The recomputed call would read the next mask."""
    net, x = Net(), torch.randn(4, 16, requires_grad=True)
    counters = spiky_amd.mask_counters(net, "cpu")
    for _ in range(2):
        y = checkpoint(net, x, use_reentrant=reentrant)
        counters[:, 1] += 1
        with pytest.raises(RuntimeError, match="after the backward pass"):
            y.sum().backward()
        y = checkpoint(net, x, use_reentrant=reentrant)
        y.sum().backward()
        counters[:, 1] += 1
    copy.deepcopy(net)(x).sum().backward()
