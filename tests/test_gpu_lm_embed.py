"""embed_tokens and its gradient on the GPU against 64-bit sums."""
import math

import pytest
import torch

from spiky_amd import TokenEmbedding, embed_tokens
import lm_tokens_plain as plain

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16
PAIRS = [(F, F), (F, B), (F, H), (B, B), (B, F), (H, H), (H, F)]


def close(got, sums, errors):
    """Within the 32-bit errors, half a step of the result's type, and half its smallest number."""
    eps = torch.finfo(got.dtype)
    bound = errors + (sums.abs() + errors) * eps.eps / 2 + eps.smallest_normal * eps.eps / 2
    worst = ((got.cpu().double() - sums).abs() - bound).max() if sums.numel() else torch.tensor(-1.0)
    assert worst <= 0, float(worst)


def both(device, tokens, vocab, cols, weight=F, out=F, scale=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, cols, generator=gen).to(weight).to(device).requires_grad_()
    dy = torch.randn(*tokens.shape, cols, generator=gen).to(out).to(device)
    y = embed_tokens(tokens, w, scale, dtype=out)
    assert y.dtype == out and torch.equal(y.detach().cpu(), plain.embed(tokens, w, scale, out))
    (dw,) = torch.autograd.grad(y, w, dy)
    assert dw.dtype == weight and dw.shape == w.shape
    close(dw, *plain.embed_gradient(tokens, dy, vocab, scale))
    return w, dy, dw


def text(gen, vocab, *shape):
    """Some tokens frequent, most rare."""
    return ((torch.rand(*shape, generator=gen) ** 6) * vocab).long().clamp_(max=vocab - 1)


@pytest.mark.parametrize("weight,out", PAIRS)
@pytest.mark.parametrize("shape,vocab,cols", [((1,), 1, 1), ((1, 1), 5, 8), ((7,), 3, 5), ((3, 65), 11, 37), ((2, 3, 4), 300, 64),
                                              ((33, 31), 257, 129), ((500,), 40, 1001), ((2, 700), 5000, 260), ((4097,), 17, 16),
                                              ((64,), 70, 4096), ((9,), 8, 9000)])
def test_values_and_gradients(cuda_device, weight, out, shape, vocab, cols):
    gen = torch.Generator().manual_seed(1)
    both(cuda_device, text(gen, vocab, *shape).to(cuda_device), vocab, cols, weight, out, 0.7)


@pytest.mark.parametrize("n,vocab,cols", [(20000, 2, 48), (20000, 262145, 3), (9000, 1500, 130), (70000, 300, 20), (30000, 1, 70),
                                          (3000, 600000, 8)])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_many_tokens(cuda_device, n, vocab, cols, kind):
    """One token many times, tables wider than the sort's workgroups, more rows than tokens."""
    gen = torch.Generator().manual_seed(2)
    both(cuda_device, text(gen, vocab, n).to(kind).to(cuda_device), vocab, cols, out=B)


def test_the_same_token_everywhere(cuda_device):
    for n in (1, 63, 64, 65, 1000, 40000):
        tokens = torch.full((n,), 6, device=cuda_device)
        w, dy, dw = both(cuda_device, tokens, 9, 72)
        assert bool((dw[torch.arange(9) != 6] == 0).all())


def test_tokens_outside_the_table_have_no_row(cuda_device):
    tokens = torch.tensor([[0, -1, 5, 6], [7, 1 << 40, -(1 << 40), 6], [1 << 32, (1 << 32) + 3, -(1 << 31), 1 << 31]])
    w, dy, dw = both(cuda_device, tokens.to(cuda_device), 7, 24, H, F, 3.0)
    narrow = torch.tensor([3, -1, 7, 1 << 30, -(1 << 31), (1 << 31) - 1], dtype=torch.int32)
    both(cuda_device, narrow.to(cuda_device), 7, 24)
    # whatever the gradient holds there
    y = embed_tokens(tokens.to(cuda_device), w, 1.0, dtype=F)
    dy = torch.where((tokens < 0) | (tokens > 6), math.nan, 1.0)[..., None].expand(3, 4, 24).to(cuda_device)
    (dw,) = torch.autograd.grad(y, w, dy)
    assert torch.equal(dw.cpu()[[0, 1, 5, 6]], torch.tensor([1.0, 0.0, 1.0, 2.0], dtype=H)[:, None].expand(4, 24))


def test_empty(cuda_device):
    w = torch.randn(5, 8, device=cuda_device, requires_grad=True)
    none = torch.zeros(3, 0, dtype=torch.int64, device=cuda_device)
    y = embed_tokens(none, w)
    assert y.shape == (3, 0, 8)
    assert torch.equal(torch.autograd.grad(y.sum(), w)[0], torch.zeros_like(w))
    some = torch.tensor([0, 1], device=cuda_device)
    assert torch.equal(embed_tokens(some, w[:0]), torch.zeros(2, 8, device=cuda_device))
    assert embed_tokens(some, w[:, :0]).shape == (2, 0)
    for cut in (w.detach()[:0].requires_grad_(), w.detach()[:, :0].requires_grad_()):
        y = embed_tokens(some, cut)
        assert torch.autograd.grad(y.sum(), cut)[0].shape == cut.shape


def test_views(cuda_device):
    """Tokens, tables and gradients with strides; a scalar token."""
    base = torch.randn(40, 96, device=cuda_device)
    tokens = torch.randint(0, 20, (6, 10), device=cuda_device)
    for w in (base[:20, 3:40], base[::2, :33], base.t()[:20], base[:1].expand(20, 96), base[5:25]):
        leaf = w.detach().requires_grad_()
        for t in (tokens, tokens[:, ::3], tokens.t(), tokens[0, 0]):
            y = embed_tokens(t, leaf, 2.0)
            assert torch.equal(y.detach(), w[t] * 2.0)
            for dy in (torch.ones(1, device=cuda_device).expand_as(y), torch.randn(*t.shape, 2 * w.shape[1], device=cuda_device)[..., ::2],
                       torch.randn(w.shape[1], device=cuda_device).expand_as(y)):
                (dw,) = torch.autograd.grad(y, leaf, dy, retain_graph=True)
                close(dw, *plain.embed_gradient(t, dy, 20, 2.0))


def test_infinities_and_nan_stay_in_their_rows(cuda_device):
    w = torch.randn(6, 16, device=cuda_device)
    w[2], w[4, 3] = math.inf, math.nan
    w.requires_grad_()
    tokens = torch.tensor([1, 2, 4, 3, 1], device=cuda_device)
    y = embed_tokens(tokens, w, 0.5)
    assert torch.equal(y.detach().nan_to_num(nan=7.0), (w.detach() * 0.5)[tokens].nan_to_num(nan=7.0))
    dy = torch.ones(5, 16, device=cuda_device)
    dy[3] = math.nan
    dy[0, 5] = math.inf
    (dw,) = torch.autograd.grad(y, w, dy)
    assert bool(dw[3].isnan().all()) and float(dw[1, 5]) == math.inf
    assert int(dw.isfinite().sum()) == 6 * 16 - 16 - 1


def test_differences(cuda_device):
    """The gradient against differences of a sum of products: it is linear, so they are exact but for rounding."""
    tokens = torch.tensor([[0, 3, 3], [1, 0, 3]], device=cuda_device)
    w = torch.randn(5, 12, device=cuda_device, requires_grad=True)
    c = torch.randn(2, 3, 12, device=cuda_device)
    loss = lambda v: (embed_tokens(tokens, v, 1.5).double() * c.double()).sum()  # noqa: E731
    (dw,) = torch.autograd.grad(loss(w), w)
    for v in range(5):
        for e in (0, 7, 11):
            step = torch.zeros_like(w)
            step[v, e] = 1.0
            with torch.no_grad():
                moved = (loss(w + step) - loss(w - step)) / 2
            # the 6 products of 32 bits on either side are off by half a step of at most 1.5 * 6
            assert abs(float(moved) - float(dw[v, e])) <= (6 * 9 * float(c.abs().max()) + float(dw.abs().max())) * 2.0 ** -23


def test_equal_calls_have_equal_gradients(cuda_device):
    gen = torch.Generator().manual_seed(3)
    tokens = text(gen, 50, 8, 2048).to(cuda_device)
    w = torch.randn(50, 200, device=cuda_device, requires_grad=True)
    dy = torch.randn(8, 2048, 200, device=cuda_device)
    first = torch.autograd.grad(embed_tokens(tokens, w), w, dy)[0]
    for _ in range(5):
        assert torch.equal(first, torch.autograd.grad(embed_tokens(tokens, w), w, dy)[0])


def test_offsets_past_32_bits(cuda_device):
    """A table and a gradient of more than 2^32 elements."""
    cols = 8192
    vocab = (1 << 32) // cols + 9
    w = torch.zeros(vocab, cols, dtype=B, device=cuda_device)
    w[-1], w[-5], w[3] = 1.5, 2.5, 3.5
    tokens = torch.tensor([vocab - 1, 3, vocab - 5, vocab, vocab - 1], device=cuda_device)
    w.requires_grad_()
    y = embed_tokens(tokens, w)
    assert y[:, 0].tolist() == y[:, -1].tolist() == [1.5, 3.5, 2.5, 0.0, 1.5]
    (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert bool((dw[-1] == 2.0).all()) and bool((dw[[3, -5]] == 1.0).all())
    assert int(torch.count_nonzero(dw)) == 3 * cols


def test_another_stream_and_captured_passes(cuda_device):
    gen = torch.Generator().manual_seed(4)
    tokens = text(gen, 900, 4, 600).to(cuda_device)
    w = torch.randn(900, 136, device=cuda_device, requires_grad=True)
    dy = torch.randn(4, 600, 136, device=cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = embed_tokens(tokens, w, 0.5)
        (dw,) = torch.autograd.grad(y, w, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = dw.clone()
    del y, dw
    graph = torch.cuda.CUDAGraph()
    leaf = w.detach().clone().requires_grad_()
    with torch.cuda.graph(graph):
        y = embed_tokens(tokens, leaf, 0.5)
        (dw,) = torch.autograd.grad(y, leaf, dy)
    for turn in range(3):
        dy.mul_(2.0)
        tokens.copy_(tokens.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.detach(), plain.embed(tokens, leaf, 0.5, F).to(cuda_device))
        close(dw, *plain.embed_gradient(tokens, dy, 900, 0.5))
    assert want.shape == dw.shape


def test_tokens_that_change_before_the_gradient_raise(cuda_device):
    w = torch.randn(5, 8, device=cuda_device, requires_grad=True)
    tokens = torch.tensor([1, 2], device=cuda_device)
    y = embed_tokens(tokens, w)
    tokens += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_module(cuda_device):
    torch.manual_seed(0)
    module = TokenEmbedding(11, 24, scale=math.sqrt(24), device=cuda_device)
    tokens = torch.tensor([[1, 5], [5, -1]], device=cuda_device)
    y = module(tokens)
    y.sum().backward()
    assert torch.equal(y.detach().cpu(), plain.embed(tokens, module.weight, math.sqrt(24), F))
    assert module.weight.grad[[1, 5], 0].tolist() == pytest.approx([math.sqrt(24), 2 * math.sqrt(24)], rel=1e-6)
    other = torch.nn.Embedding(11, 24, device=cuda_device)
    other.load_state_dict(module.state_dict())
    assert torch.equal(other.weight, module.weight)
    frozen = module.requires_grad_(False)
    assert not frozen(tokens).requires_grad


REFUSED = [
    (lambda t: embed_tokens(t["i"], t["w"].double()), RuntimeError, "must be float32, bfloat16 or float16"),
    (lambda t: embed_tokens(t["w"], t["w"]), RuntimeError, "int32 or int64"),
    (lambda t: embed_tokens(t["i"].cpu(), t["w"]), RuntimeError, "must be on CUDA"),
    (lambda t: embed_tokens(None, t["w"]), RuntimeError, "must be a torch.Tensor"),
    (lambda t: embed_tokens([1], t["w"]), RuntimeError, "must be a torch.Tensor"),
    (lambda t: embed_tokens(t["i"], t["w"][0]), ValueError, r"must be \[V, E\]"),
    (lambda t: embed_tokens(t["i"], t["w"].bfloat16(), dtype=H), ValueError, "dtype must be"),
    (lambda t: embed_tokens(t["i"], t["w"], dtype=torch.float64), ValueError, "dtype must be"),
    (lambda t: embed_tokens(t["i"], t["w"], dtype="half"), RuntimeError, "torch.dtype"),
    (lambda t: embed_tokens(t["i"], t["w"], "large"), TypeError, "real number"),
    (lambda t: embed_tokens(t["i"], t["w"], math.nan), ValueError, "must be finite"),
    (lambda t: embed_tokens(t["i"], t["w"], -1e39), ValueError, "must be finite"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refusals(cuda_device, case):
    call, kind, message = REFUSED[case]
    t = dict(i=torch.zeros(3, dtype=torch.int64, device=cuda_device), w=torch.zeros(4, 8, device=cuda_device))
    with pytest.raises(kind, match=message):
        call(t)


def test_derivatives_that_there_are_none_of(cuda_device):
    w = torch.randn(4, 8, device=cuda_device, requires_grad=True)
    tokens = torch.tensor([1, 2], device=cuda_device)
    c = torch.randn(2, 8, device=cuda_device, requires_grad=True)
    (dw,) = torch.autograd.grad((embed_tokens(tokens, w) * c).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        torch.autograd.grad(dw.sum(), c)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(w.detach(), torch.ones_like(w))
        with pytest.raises(NotImplementedError, match="no forward-mode derivatives"):
            embed_tokens(tokens, dual)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda x: embed_tokens(tokens, x), w.detach())


@pytest.mark.parametrize("n,vocab,cols,weight,out", [
    (8192, 300, 64, F, F), (8193, 300, 64, F, F), (8192, 20, 65, F, F), (4096, 900, 128, F, F), (4096, 900, 129, F, F),
    (2048, 3000, 512, B, B), (2048, 3000, 513, B, B), (2049, 3000, 512, B, B), (4095, 40, 500, H, H)])
def test_sizes_at_which_another_way_is_taken(cuda_device, n, vocab, cols, weight, out):
    """One launch or three, one slab of columns or two."""
    gen = torch.Generator().manual_seed(5)
    both(cuda_device, text(gen, vocab, n).to(cuda_device), vocab, cols, weight, out, 0.3)


@pytest.mark.parametrize("cols", [24, 320, 1000])
def test_runs_at_the_ends_of_chunks(cuda_device, cols):
    """Chunks of 8, 16 and 32 sorted positions: runs that are as long, one longer, begin with one or inside."""
    for first in (0, 1, 7, 8, 16, 31, 32):
        counts = [first, 8, 9, 7, 16, 17, 15, 32, 33, 31, 64, 65, 63, 1, 0, 0, 2, 1000, 24, 25, 0, 3000, 96, 5200]
        tokens = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
        tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(first))]
        both(cuda_device, tokens.to(cuda_device), len(counts), cols, F, B)
        both(cuda_device, torch.cat([tokens, torch.full((77,), -1)]).to(cuda_device), len(counts) + 3, cols, F, B)


def test_a_capture_beside_an_eager_graph_of_the_same_leaf_is_refused(cuda_device):
    """The eager graph's leaf belongs to the default stream; without it the capture is made."""
    w = torch.randn(64, 16, device=cuda_device, requires_grad=True)
    tokens, dy = torch.randint(0, 64, (9,), device=cuda_device), torch.randn(9, 16, device=cuda_device)
    eager = embed_tokens(tokens, w)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="belongs to the default stream"):
        with torch.cuda.graph(graph):
            torch.autograd.grad(embed_tokens(tokens, w), w, dy)
    del eager
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (dw,) = torch.autograd.grad(embed_tokens(tokens, w), w, dy)
    graph.replay()
    torch.cuda.synchronize()
    close(dw, *plain.embed_gradient(tokens, dy, 64, 1.0))


def test_one_leaf_looked_up_twice(cuda_device):
    """Its gradients add up."""
    w = torch.randn(30, 40, device=cuda_device, requires_grad=True)
    first, second = torch.randint(0, 30, (2, 50), device=cuda_device)
    a, b = torch.randn(2, 50, 40, device=cuda_device)
    ((embed_tokens(first, w) * a).sum() + (embed_tokens(second, w, 2.0) * b).sum()).backward()
    sums, errors = plain.embed_gradient(first, a, 30, 1.0)
    more, others = plain.embed_gradient(second, b, 30, 2.0)
    # the sum of both is rounded once more
    close(w.grad, sums + more, errors + others + (sums.abs() + more.abs()) * 2 * plain.STEP32)
