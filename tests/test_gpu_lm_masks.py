"""The masks of the modules' dropout on the GPU in recomputed and in captured steps."""
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


def filled(model):
    """The model with tables of normal values: they start as zeros, and the logits with them."""
    gen = torch.Generator(model.device).manual_seed(6)
    with torch.no_grad():
        for layer in model._lut_layers():
            layer._weights.normal_(0.0, 0.5, generator=gen)
    return model


def check_model_step(got, want):
    """The logits bit for bit.  Gradients pass four layers, whose fp32 atomics come in any order: sums of
    some thousand terms, each off by half a step of 2^-24 of the sum of magnitudes, taken as at most
    four times the largest result: 4 * 4096 * 2^-24.  Another mask moves them by their own size."""
    assert torch.equal(got[0], want[0])
    for a, b in zip(got[1:], want[1:]):
        assert float((a - b).abs().max()) <= 2.0 ** -10 * float(b.abs().max())


def test_a_recomputed_model_is_the_whole_one(cuda_device):
    tokens = torch.randint(0, 50, (4, 8), device=cuda_device)
    join = dict(post_norm="rms", pre_norm="rms", gate=0.5)
    results = []
    for recomputed in (False, True):
        m = filled(small(cuda_device, dropout=0.2, residual_join=join))
        if recomputed:
            mask_counters(m, cuda_device)
        y = checkpoint(m, tokens, use_reentrant=False) if recomputed else m(tokens)
        y.square().sum().backward()
        results.append([y.detach(), *(p.grad for n, p in m.named_parameters() if "_join" in n)])
    assert len(results[0]) == 13
    check_model_step(*results)


def on_a_side_stream(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("within", [True, False])
def test_replays_of_a_captured_step_have_the_eager_steps_masks(cuda_device, within):
    """The counters advance in the captured step, or between its replays."""
    x, eager, net = torch.randn(40, 96, device=cuda_device), Net(cuda_device), Net(cuda_device)
    counters = mask_counters(net, cuda_device)
    start = counters.clone()

    def step(m, advance):
        v = x.clone().requires_grad_()
        y = m(v)
        grads = torch.autograd.grad(y.sum(), [v, *m.parameters()])
        if advance:
            counters[:, 1] += 1
        return [y.detach(), *grads]

    on_a_side_stream(lambda: step(net, within))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(net, within)
    counters.copy_(start)
    seen = []
    for _ in range(4):
        want = step(eager, False)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
        seen.append(captured[0].clone())
        if not within:
            counters[:, 1] += 1
    assert not any(torch.equal(a, b) for a, b in zip(seen, seen[1:]))
    assert net.state_dict()["drop._extra_state"] == eager.state_dict()["drop._extra_state"]
    # a loaded state goes to the graph's counters
    net.load_state_dict({**net.state_dict(), "drop._extra_state": {"seed": 3, "calls": 0},
                         "join._extra_state": {"seed": (1 << 63) + 9, "calls": 0}})
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured[0], seen[0])


def test_a_counted_call_in_a_capture_raises(cuda_device):
    x, net = torch.randn(4, 96, device=cuda_device), Net(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="mask_counters"):
        with torch.cuda.graph(graph):
            net(x)
    assert net.drop.calls == 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = net.eval()(x)
    for _ in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, net(x))


def test_replays_of_a_captured_model_have_the_eager_models_masks(cuda_device):
    tokens = torch.randint(0, 50, (4, 8), device=cuda_device)
    how = dict(dropout=0.2, residual_join=dict(post_norm="rms", pre_norm="rms", gate=0.5))
    eager, m = filled(small(cuda_device, **how)), filled(small(cuda_device, **how))
    counters = mask_counters(m, cuda_device)
    start = counters.clone()

    def step(model):
        leaves = [p for n, p in model.named_parameters() if "_join" in n]
        y = model(tokens)
        return [y.detach(), *torch.autograd.grad(y.square().sum(), leaves)]

    on_a_side_stream(lambda: step(m))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(m)
        counters[:, 1] += 1
    counters.copy_(start)
    seen = []
    for _ in range(3):
        want = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        check_model_step(captured, want)
        seen.append(captured[0].clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])
