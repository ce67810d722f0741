"""Counter-based dropout on the GPU against its definition on whole numbers."""
import numpy as np
import pytest
import torch

from spiky_amd import CounterDropout, counter_dropout
import lm_plain

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def expected(x, p, seed, offset):
    """x times the scale in one 32-bit product, rounded to x's type: the operator's own arithmetic."""
    cols = x.shape[-1] if x.dim() else 1
    rows = x.numel() // cols
    keep = lm_plain.kept(rows, cols, p, seed, offset).reshape(x.shape)
    scale = float(np.float32(1.0 / (1.0 - p))) if p < 1 else 0.0
    return torch.where(keep, (x.float().cpu() * scale), torch.zeros(())).to(x.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 1), (3, 4), (5, 8), (33, 9), (2, 3, 257), (1000, 1), (301, 77),
                                   (2, 5000), (9, 8200), (4096, 16)])
def test_values_are_exactly_the_definitions(cuda_device, dtype, shape):
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(shape, generator=gen).to(dtype)
    y = counter_dropout(x.to(cuda_device), 0.3, 0x123456789ABCDEF0, 0x1_0000_0007)
    assert y.dtype == dtype and y.shape == x.shape
    assert torch.equal(y.cpu(), expected(x, 0.3, 0x123456789ABCDEF0, 0x1_0000_0007))


@pytest.mark.parametrize("p", [0.0, 1e-12, 0.5, 1.0 - 1e-12, 1.0])
def test_ends_of_the_probability(cuda_device, p):
    x = torch.randn(37, 130)
    y = counter_dropout(x.to(cuda_device), p, 3).cpu()
    if p < 1e-6:
        assert torch.equal(y, x * float(np.float32(1.0 / (1.0 - p))))
    elif p > 0.9:
        assert torch.equal(y, torch.zeros_like(x))
    else:
        assert torch.equal(y, expected(x, p, 3, 0))


@pytest.mark.parametrize("p", [0.3, 1.0])
def test_dropped_infinities_and_nan_are_zero(cuda_device, p):
    x = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0]).repeat(64, 16)
    y = counter_dropout(x.to(cuda_device), p, 9).cpu()
    keep = lm_plain.kept(64, 64, p, 9, 0)
    assert torch.equal(y[~keep], torch.zeros(int((~keep).sum())))
    assert torch.equal(torch.isnan(y), torch.isnan(x) & keep)
    assert torch.equal(torch.isinf(y), torch.isinf(x) & keep)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_has_the_same_mask(cuda_device, dtype):
    x = torch.randn(50, 333, device=cuda_device).to(dtype).requires_grad_()
    dy = torch.randn(50, 333, device=cuda_device).to(dtype)
    y = counter_dropout(x, 0.4, -1, 2)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(dx.cpu(), expected(dy.cpu(), 0.4, (1 << 64) - 1, 2))


def test_strided_inputs_have_the_mask_of_their_shape(cuda_device):
    base = torch.randn(6, 5, 48, device=cuda_device)
    for x in (base[:, 2], base[:, :, 3:40], base.transpose(0, 1), base[:, 1:3], base[..., ::2], base[:, :1],
              base[0, 0].expand(4, 48), base[::2, ::2]):
        assert torch.equal(counter_dropout(x, 0.5, 1, 1).cpu(), expected(x.cpu(), 0.5, 1, 1))


def test_types_share_a_mask_and_calls_repeat(cuda_device):
    ones = torch.ones(129, 515, device=cuda_device)
    first = counter_dropout(ones, 0.25, 77, 4)
    assert torch.equal(first, counter_dropout(ones, 0.25, 77, 4))
    for dtype in TYPES[1:]:
        assert torch.equal(first != 0, counter_dropout(ones.to(dtype), 0.25, 77, 4) != 0)
    for other in ((78, 4), (77, 5), (77 + (1 << 32), 4), (77, 4 + (1 << 32))):
        differ = ((first != 0) != (counter_dropout(ones, 0.25, *other) != 0)).float().mean()
        # two independent masks differ at 2 * 0.25 * 0.75 of the elements, off by under 6 deviations
        assert abs(float(differ) - 0.375) < 6 * (0.375 * 0.625 / ones.numel()) ** 0.5


@pytest.mark.parametrize("p", [0.1, 0.5])
def test_share_of_kept_elements(cuda_device, p):
    y = counter_dropout(torch.ones(1024, 1024, device=cuda_device), p, 12345)
    share = float((y != 0).double().mean())
    assert abs(share - (1 - p)) < 6 * (p * (1 - p) / 2 ** 20) ** 0.5


def test_empty(cuda_device):
    for shape in ((0,), (0, 5), (5, 0)):
        assert counter_dropout(torch.zeros(shape, device=cuda_device), 0.5, 1).shape == shape


def test_rows_past_32_bits_of_elements(cuda_device):
    # 2^32 + 2^20 two-byte elements: element offsets pass 32 bits, rows and groups do not
    rows, cols = (1 << 12) + 1, 1 << 20
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device=cuda_device)
    y = counter_dropout(x, 0.5, 6, 1)
    for r in (0, 4095, 4096):
        assert torch.equal((y[r] != 0).cpu(), lm_plain.kept(1, cols, 0.5, 6, 1, row0=r)[0])


def test_seed_tensor_and_graph_replays(cuda_device):
    """A captured call reads [seed, offset] when it runs: each replay has the eager call's mask."""
    x = torch.randn(65, 100, device=cuda_device)
    state = torch.tensor([42, 7], dtype=torch.int64, device=cuda_device)
    assert torch.equal(counter_dropout(x, 0.5, state), counter_dropout(x, 0.5, 42, 7))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        counter_dropout(x, 0.5, state)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = counter_dropout(x, 0.5, state)
    for offset in (7, 8, 9):
        state[1] = offset
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, counter_dropout(x, 0.5, 42, offset))


def test_another_stream(cuda_device):
    x = torch.randn(512, 512, device=cuda_device)
    want = counter_dropout(x, 0.5, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = counter_dropout(x, 0.5, 3)
    side.synchronize()
    assert torch.equal(y, want)


def test_module(cuda_device):
    m = CounterDropout(0.5, seed=11)
    x = torch.randn(8, 64, device=cuda_device, requires_grad=True)
    first, second = m(x), m(x)
    assert torch.equal(first, counter_dropout(x, 0.5, 11, 1)) and torch.equal(second, counter_dropout(x, 0.5, 11, 2))
    other = CounterDropout(0.1)
    other.load_state_dict(m.state_dict())
    other.p = 0.5
    assert torch.equal(other(x), counter_dropout(x, 0.5, 11, 3))
    assert m.eval()(x) is x
