"""beam_select on the GPU against a full sort in 64 bits."""
import math

import pytest
import torch

from spiky_amd import beam_select, process_logits
import lm_tokens_plain as plain

pytestmark = pytest.mark.gpu

F, B, H = torch.float32, torch.bfloat16, torch.float16


def inputs(searches, beams, vocab, dtype, seed=0, spread=4.0):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(searches, beams, vocab, generator=gen) * spread).to(dtype)
    scores = -10.0 * torch.rand(searches, beams, generator=gen)
    return x, scores, gen


def run(device, x, scores, n=None, **how):
    to = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in how.items()}
    got = beam_select(x.to(device), scores.to(device), n, **to)
    plain.check_select(got, x, scores, x.shape[1] if n is None else n, **how)
    return got


@pytest.mark.parametrize("dtype", [F, B, H])
@pytest.mark.parametrize("searches,beams,vocab,n", [
    (1, 1, 1, 1), (1, 1, 1, 5), (2, 3, 2, 6), (3, 2, 7, 4), (1, 4, 256, 4), (2, 4, 255, 8), (1, 1, 4097, 2), (5, 3, 8192, 5),
    (2, 5, 8193, 10), (3, 2, 20001, 64), (1, 64, 300, 64), (1, 33, 9000, 40), (2, 8, 50001, 16), (1, 2, 262147, 64),
    (70, 1, 130, 1)])
def test_selection(cuda_device, dtype, searches, beams, vocab, n):
    x, scores, gen = inputs(searches, beams, vocab, dtype)
    run(cuda_device, x, scores, n)
    finished = torch.rand(searches, beams, generator=gen) < 0.4
    lengths = torch.randint(0, 30, (searches, beams), generator=gen)
    run(cuda_device, x, scores, n, finished=finished, pad=vocab // 2, lengths=lengths, length_penalty=0.8)


def test_first_step(cuda_device):
    """One beam is alive."""
    x, scores, _ = inputs(2, 4, 5000, F)
    scores[:] = -math.inf
    scores[0, 0], scores[1, 2] = 0.0, -3.0
    x[0, 1], x[1, 0] = math.nan, math.inf  # not read
    got = run(cuda_device, x, scores, 8)
    assert got[1].tolist() == [[0] * 8, [2] * 8]


@pytest.mark.parametrize("dtype", [F, B, H])
@pytest.mark.parametrize("vocab", [5, 300, 9001, 40000])
def test_equal_logits_go_by_token_and_beam(cuda_device, dtype, vocab):
    x = torch.zeros(2, 3, vocab, dtype=dtype)
    got = run(cuda_device, x, torch.zeros(2, 3), 4)
    assert got[1].tolist() == [[0] * 4] * 2 and got[2].tolist() == [[0, 1, 2, 3]] * 2
    # a few values only, everywhere the same ones
    x = (torch.arange(vocab) * 7 % 3).to(dtype).expand(2, 3, vocab).contiguous()
    run(cuda_device, x, torch.zeros(2, 3), 64)
    # equal rows at the odd places of memory that an odd vocabulary gives them
    gen = torch.Generator().manual_seed(1)
    row = (torch.randn(vocab, generator=gen) * 3).to(dtype)
    got = run(cuda_device, row.expand(2, 3, vocab).contiguous(), torch.zeros(2, 3), 6)
    s = got[0].cpu()
    assert s[:, 0].tolist() == s[:, 1].tolist() == s[:, 2].tolist()
    assert got[1][0, :3].tolist() == [0, 1, 2] and len(set(got[2][0, :3].tolist())) == 1


@pytest.mark.parametrize("dtype", [F, B, H])
@pytest.mark.parametrize("left", [0, 1, 3, 200])
def test_masked_tokens(cuda_device, dtype, left):
    """Few tokens that a mask leaves; with -infinity, and with the type's lowest value."""
    for low in (-math.inf, torch.finfo(dtype).min):
        x, scores, gen = inputs(2, 3, 20000, dtype)
        mask = torch.zeros(20000, dtype=torch.bool)
        mask[torch.randperm(20000, generator=gen)[:left]] = True
        x = x.masked_fill(~mask, low)
        got = run(cuda_device, x, scores, 6)
        if low == -math.inf and left == 0:
            assert got[0].tolist() == [[-math.inf] * 6] * 2 and got[2].tolist() == [[0] * 6] * 2


def test_one_beam_masked_whole(cuda_device):
    x, scores, _ = inputs(1, 3, 9000, F)
    x[0, 1] = -math.inf
    got = run(cuda_device, x, scores, 5, pad=77)
    assert 1 not in got[1].tolist()[0]
    got = run(cuda_device, x[:, 1:2], scores[:, 1:2], 3, pad=77)
    assert got[2].tolist() == [[77] * 3] and got[1].tolist() == [[0] * 3]


def test_unknown_scores(cuda_device):
    for value in (math.nan, math.inf):
        for at in (0, 4999, 8999):
            x, scores, _ = inputs(2, 3, 9000, F)
            x[0, 1, at] = value
            got = run(cuda_device, x, scores, 5)
            assert got[1].tolist()[0] == [1] * 5 and got[2].tolist()[0] == [0, 1, 2, 3, 4]
        x, scores, _ = inputs(2, 3, 3, B)
        scores[1, 2] = value
        run(cuda_device, x, scores, 5)
        run(cuda_device, x, scores, 12, finished=torch.tensor([[True, False, False], [False, False, True]]))


@pytest.mark.parametrize("scale", [1e4, 1e30, 3e38])
def test_large_logits(cuda_device, scale):
    x, scores, _ = inputs(2, 3, 5000, F)
    x = (x / x.abs().max()) * scale
    run(cuda_device, x, scores, 6)
    run(cuda_device, -x.abs(), scores, 6)
    run(cuda_device, torch.full_like(x, -scale), scores, 6)


def test_all_finished(cuda_device):
    x, scores, _ = inputs(2, 5, 300, H)
    x[:] = math.nan  # not read
    scores[0, 3] = -math.inf
    done = torch.ones(2, 5, dtype=torch.bool)
    got = run(cuda_device, x, scores, 7, finished=done, pad=9)
    assert bool((got[2] == 9).all())
    run(cuda_device, x[:, :, :0], scores, 7, finished=done, pad=9)


def test_lengths(cuda_device):
    x, scores, gen = inputs(3, 4, 600, F)
    for kind in (torch.int32, torch.int64):
        lengths = torch.randint(-2, 5, (3, 4), generator=gen).to(kind)
        for alpha in (0.0, 0.5, 1.0, -1.0, 8.0, -8.0):
            for finished in (None, torch.rand(3, 4, generator=gen) < 0.5):
                run(cuda_device, x, scores, 9, finished=finished, lengths=lengths, length_penalty=alpha)


def test_views(cuda_device):
    gen = torch.Generator().manual_seed(5)
    base = (torch.randn(12, 3, 2011, generator=gen) * 3).to(B).to(cuda_device)
    scores = -torch.rand(8, 4, generator=gen).to(cuda_device)
    finished = torch.zeros(4, 4, dtype=torch.bool, device=cuda_device)
    finished[1] = True
    for x, s in ((base[:, -1].view(3, 4, 2011), scores[:3]), (base[:, :, 5:1000], scores[:, :3].repeat(2, 1)[:12]),
                 (base[:, 0].unflatten(0, (4, 3)).transpose(0, 1), scores[::3].contiguous()[:, :4]),
                 (base[:2, :1].expand(2, 4, 2011), scores[:4:2]), (base.transpose(1, 2)[:2, :40], scores.repeat(4, 10)[:2, :40])):
        got = beam_select(x, s, 5)
        plain.check_select(got, x.cpu(), s, 5)
    x = base[:4, 0].unflatten(0, (1, 4)).expand(4, 4, 2011)
    got = beam_select(x, scores[:4], 5, finished=finished.t())
    plain.check_select(got, x.cpu(), scores[:4], 5, finished=finished.t().cpu())


def test_many_rows(cuda_device):
    x, scores, _ = inputs(1100, 64, 40, B)
    got = beam_select(x.to(cuda_device), scores.to(cuda_device), 2)
    some = torch.tensor([0, 511, 512, 513, 1023, 1024, 1099])
    plain.check_select([t[some.to(cuda_device)] for t in got], x[some], scores[some], 2)


def test_offsets_past_32_bits(cuda_device):
    vocab = (1 << 30) + 12345
    x = torch.full((1, 5, vocab), -4.0, dtype=B, device=cuda_device)
    x[0, 4, vocab - 1], x[0, 4, 70000], x[0, 3, vocab - 2] = 40.0, 39.0, 38.0
    got = beam_select(x, torch.zeros(1, 5, device=cuda_device), 3)
    assert got[1].tolist() == [[3, 4, 4]] and got[2].tolist() == [[vocab - 2, vocab - 1, 70000]]
    # the others are exp(-42) and exp(-44) each of the first
    want = [-math.log1p(vocab * math.exp(-42.0)), -math.log1p(math.exp(-1.0)), -1.0 - math.log1p(math.exp(-1.0))]
    assert got[0].tolist()[0] == pytest.approx(want, abs=1e-5)


def test_calls_repeat_and_are_captured(cuda_device):
    x, scores, _ = inputs(3, 4, 30000, B)
    x, scores = x.to(cuda_device), scores.to(cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = beam_select(x, scores, 8)
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam_select(x, scores, 8)
    with torch.cuda.graph(other):
        more = beam_select(x, scores, 8)
    for turn in range(3):
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = beam_select(x, scores, 8)
        for a, b, c in zip(got, want, more):
            assert torch.equal(a, b) and torch.equal(c, b)
        if turn == 0:
            assert all(torch.equal(a, b) for a, b in zip(first, want))
        x.copy_(x.flip(2))


def test_after_process_logits(cuda_device):
    x, scores, gen = inputs(2, 4, 1000, H)
    allowed = torch.rand(1000, generator=gen) < 0.2
    y = process_logits(x.to(cuda_device).view(8, 1000), mask=allowed.to(cuda_device), temperature=0.7, dtype=F)
    got = beam_select(y.view(2, 4, 1000), scores.to(cuda_device))
    plain.check_select(got, y.cpu().view(2, 4, 1000), scores, 4)
    assert bool(allowed[got[2].cpu()].all())


REFUSED = [
    (lambda t: beam_select(t["x"][0], t["s"]), ValueError, r"must be \[B, K, V\]"),
    (lambda t: beam_select(t["x"].double(), t["s"]), RuntimeError, "must be float32, bfloat16 or float16"),
    (lambda t: beam_select(t["x"].cpu(), t["s"]), RuntimeError, "must be on CUDA"),
    (lambda t: beam_select(t["x"], None), RuntimeError, "must be a torch.Tensor"),
    (lambda t: beam_select(t["x"], t["s"].cpu()), RuntimeError, "must be on CUDA"),
    (lambda t: beam_select(t["x"], t["s"].double()), RuntimeError, "scores must be float32"),
    (lambda t: beam_select(t["x"], t["s"][:1]), ValueError, "scores must have shape"),
    (lambda t: beam_select(t["x"], t["s"], 0), ValueError, "1 to 64"),
    (lambda t: beam_select(t["x"], t["s"], 65), ValueError, "1 to 64"),
    (lambda t: beam_select(t["x"], t["s"], -1), ValueError, "1 to 64"),
    (lambda t: beam_select(t["x"], t["s"], 2.5), TypeError, "integer"),
    (lambda t: beam_select(t["x"][:, :0], t["s"][:, :0]), ValueError, "1 to 64"),
    (lambda t: beam_select(t["x"].repeat(1, 30, 1), t["s"].repeat(1, 30), 3), ValueError, "1 to 64"),
    (lambda t: beam_select(t["x"], t["s"], finished=t["s"]), RuntimeError, "finished must have dtype bool"),
    (lambda t: beam_select(t["x"], t["s"], finished=t["s"][0] > 0), ValueError, "finished must have shape"),
    (lambda t: beam_select(t["x"], t["s"], lengths=t["s"]), RuntimeError, "int32 or int64"),
    (lambda t: beam_select(t["x"], t["s"], length_penalty=1.0), ValueError, "needs lengths"),
    (lambda t: beam_select(t["x"], t["s"], lengths=t["i"], length_penalty=9.0), ValueError, "-8 to 8"),
    (lambda t: beam_select(t["x"], t["s"], lengths=t["i"], length_penalty=math.nan), ValueError, "-8 to 8"),
    (lambda t: beam_select(t["x"], t["s"], pad=0.5), TypeError, "integer"),
]


@pytest.mark.parametrize("case", range(len(REFUSED)))
def test_refusals(cuda_device, case):
    call, kind, message = REFUSED[case]
    t = dict(x=torch.zeros(2, 3, 8, device=cuda_device), s=torch.zeros(2, 3, device=cuda_device),
             i=torch.zeros(2, 3, dtype=torch.int64, device=cuda_device))
    with pytest.raises(kind, match=message):
        call(t)


def test_no_searches(cuda_device):
    got = beam_select(torch.zeros(0, 3, 8, device=cuda_device), torch.zeros(0, 3, device=cuda_device), 2)
    assert [t.shape for t in got] == [(0, 2)] * 3


def test_zeros_of_both_signs_are_equal(cuda_device):
    for dtype in (F, B, H):
        x = torch.zeros(1, 2, 9000, dtype=dtype)
        x[:, :, ::2] = -0.0
        got = run(cuda_device, x, torch.zeros(1, 2), 5)
        assert got[2].tolist() == [[0, 1, 2, 3, 4]]
        x[:, :, 100:] = -1.0
        got = run(cuda_device, x, torch.tensor([[-0.0, 0.0]]), 5)
        assert got[2].tolist() == [[0, 1, 2, 3, 4]] and got[1].tolist() == [[0] * 5]


@pytest.mark.parametrize("dtype", [F, B])
def test_sorted_logits(cuda_device, dtype):
    """The first candidates side by side, at either end, in many slices."""
    for vocab in (3000, 8200, 70000):
        x = torch.linspace(-30.0, 5.0, vocab).to(dtype).expand(2, 2, vocab).contiguous()
        scores = torch.tensor([[-1.0, -2.5], [-0.25, -0.25]])
        for n in (1, 7, 64):
            run(cuda_device, x, scores, n)
            run(cuda_device, x.flip(2).contiguous(), scores, n)


@pytest.mark.parametrize("beams,n", [(3, 64), (16, 64), (64, 3), (7, 5)])
def test_many_equal_ranks(cuda_device, beams, n):
    """More candidates of one rank than the join lists."""
    for vocab in (40, 9000, 40000):
        x = torch.zeros(2, beams, vocab, dtype=B)
        x[1, :, ::3] = 1.0
        scores = torch.zeros(2, beams)
        run(cuda_device, x, scores, n)
        run(cuda_device, x, scores, n, lengths=torch.full((2, beams), 3), length_penalty=0.5)
