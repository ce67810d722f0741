"""The gradient of embed_tokens on the GPU for tables of many rows, of which a thread takes several, with tokens
that stand at many positions; and on another stream."""
import pytest
import torch

from spiky_amd import embed_tokens
import lm_tokens_plain as plain

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16


def close(got, sums, errors):
    """Within the 32-bit errors, half a step of the result's type, and half its smallest number."""
    eps = torch.finfo(got.dtype)
    bound = errors + (sums.abs() + errors) * eps.eps / 2 + eps.smallest_normal * eps.eps / 2
    worst = ((got.cpu().double() - sums).abs() - bound).max()
    assert worst <= 0, float(worst)


def check(device, tokens, vocab, cols, weight, out, scale=0.7):
    """Rows that tokens have against their sums in 64 bits, all others against zero."""
    gen = torch.Generator(device).manual_seed(1)
    w = torch.zeros(1, cols, dtype=weight, device=device).expand(vocab, cols).contiguous().requires_grad_()
    dy = torch.randn(*tokens.shape, cols, generator=gen, device=device).to(out)
    (dw,) = torch.autograd.grad(embed_tokens(tokens, w, scale, dtype=out), w, dy)
    assert dw.dtype == weight and dw.shape == w.shape
    there = (tokens >= 0) & (tokens < vocab)
    rows, at = tokens[there].unique(return_inverse=True)
    compact = torch.full_like(tokens, -1)
    compact[there] = at.to(tokens.dtype)
    close(dw[rows.long()], *plain.embed_gradient(compact, dy, len(rows), scale))
    dw[rows.long()] = 0
    assert int(torch.count_nonzero(dw)) == 0


def text(vocab, n, padded=False):
    """Half of the positions are of 12 tokens all over the table, at its ends too, the others of any."""
    gen = torch.Generator().manual_seed(2)
    often = torch.linspace(0, vocab - 1, 12, dtype=torch.float64).round().long()
    tokens = torch.randint(0, vocab, (n,), generator=gen)
    tokens[:n // 2] = often[torch.arange(n // 2) * (torch.arange(n // 2) % 5 + 1) % 12]
    if padded:
        tokens[torch.rand(n, generator=gen) < 0.2] = -1
    return tokens[torch.randperm(n, generator=gen)]


@pytest.mark.parametrize("n,vocab,cols,weight,out", [
    (3000, 17000, 1024, F, F), (3001, 17011, 2041, B, B), (5000, 33000, 1000, F, B), (4000, 140000, 200, H, F),
    (20000, 66000, 512, F, H), (3000, 33000, 1023, H, H)])
def test_several_rows_of_a_thread(cuda_device, n, vocab, cols, weight, out):
    check(cuda_device, text(vocab, n).to(cuda_device), vocab, cols, weight, out)
    check(cuda_device, text(vocab, n, padded=True).int().to(cuda_device), vocab, cols, weight, out)


@pytest.mark.parametrize("n,vocab,cols,weight,out", [
    (6000, 140000, 1024, F, F), (6000, 140000, 1024, F, B), (6001, 140001, 999, F, H), (6000, 140000, 2048, B, B),
    (4000, 70001, 4001, H, F), (300, 140000, 1024, F, B)])
def test_tables_past_the_last_cache(cuda_device, n, vocab, cols, weight, out):
    tokens = text(vocab, 6001)[:n]
    check(cuda_device, tokens.to(cuda_device), vocab, cols, weight, out)


def test_a_gradient_on_another_stream(cuda_device):
    for vocab, cols in ((900, 136), (17000, 1024)):
        tokens = text(vocab, 2400).view(4, 600).to(cuda_device)
        w = torch.randn(vocab, cols, device=cuda_device, requires_grad=True)
        dy = torch.randn(4, 600, cols, device=cuda_device)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = embed_tokens(tokens, w, 0.5)
            (dw,) = torch.autograd.grad(y, w, dy)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y.detach().cpu(), plain.embed(tokens, w, 0.5, F))
        close(dw, *plain.embed_gradient(tokens, dy, vocab, 0.5))
