"""The language-model operators where their kernels change form: widths around a piece, a wave, a
workgroup; row counts around a chunk; histories and biases that outgrow a word or a list."""
import pytest
import torch

from spiky_amd import CounterDropout, counter_dropout, process_logits, residual_norm
import lm_plain
from test_gpu_lm_dropout import expected
from test_gpu_lm_logits import check as check_logits, make
from test_gpu_lm_residual import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act,res", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                     (torch.float16, torch.float16)])
@pytest.mark.parametrize("D", [2, 7, 9, 15, 17, 127, 129, 255, 511, 513, 1023, 2047, 2049, 4095, 4097, 8191, 8193, 16383])
def test_rows_that_end_inside_a_piece(cuda_device, act, res, D):
    check(cuda_device, 5, D, act, res, post="layer", pre="layer", gate="channel", biases=True, dropout_p=0.2, seed=9)
    check(cuda_device, 5, D, act, res, gate="full", dropout_p=0.2, seed=9, offset=1 << 40)


@pytest.mark.parametrize("D", [5, 100, 200, 500, 700, 1500, 3001, 5003, 9001])
@pytest.mark.parametrize("full", [True, False])
@pytest.mark.parametrize("rows,gate_rows", [(1537, 1537), (1536, 3), (1530, 510)])
def test_chunks_of_rows(cuda_device, D, full, rows, gate_rows):
    if D > 4000:
        rows, gate_rows = rows // 3, gate_rows // 3
    kw = dict(post="layer", pre="rms", biases=True) if full else {}
    check(cuda_device, rows, D, torch.bfloat16, torch.float32, gate="rows", gate_rows=gate_rows, dropout_p=0.1, seed=2, **kw)


@pytest.mark.parametrize("rows", [1, 2, 255, 257, 1023, 1025, 4097])
def test_few_and_many_rows(cuda_device, rows):
    check(cuda_device, rows, 24, gate="full", biases=True)
    check(cuda_device, rows, 300, torch.float16, gate="channel")


@pytest.mark.parametrize("D", [3, 64, 1001])
def test_gradients_of_some_inputs_only(cuda_device, D):
    """Each gradient is the same whichever others are asked for."""
    gen = torch.Generator().manual_seed(0)
    t = {k: torch.randn(s, generator=gen).to(cuda_device) for k, s in
         dict(r=(40, D), a=(40, D), w1=(D,), b1=(D,), g=(D,), w2=(D,), b2=(D,)).items()}
    dz, dh = torch.randn(40, D, device=cuda_device), torch.randn(40, D, device=cuda_device)

    def grads(names):
        v = {k: x.clone().requires_grad_(k in names) for k, x in t.items()}
        z, h = residual_norm(v["r"], v["a"], post_norm="layer", post_weight=v["w1"], post_bias=v["b1"], gate=v["g"],
                             pre_norm="rms", pre_weight=v["w2"], pre_bias=v["b2"], dropout_p=0.3, seed=1)
        return dict(zip(names, torch.autograd.grad([z, h], [v[k] for k in names], [dz, dh])))

    everything = grads(list(t))
    for k in t:
        assert torch.equal(grads([k])[k], everything[k]), k


def test_unneeded_columns_of_other_lanes_do_not_leak(cuda_device):
    """Columns next to a row's end hold NaN: they are not read, or not used."""
    for dtype in (torch.float32, torch.bfloat16):
        for D in (9, 63, 1001, 5003):
            wide = torch.full((2, 6, D + 40), float("nan"), device=cuda_device).to(dtype)
            wide[..., 11:11 + D] = torch.randn(2, 6, D, device=cuda_device).to(dtype)
            r, a = wide[0, :, 11:11 + D], wide[1, :, 11:11 + D]
            z, h = residual_norm(r, a, post_norm="layer", pre_norm="rms", dropout_p=0.1, seed=1)
            z2, h2 = residual_norm(r.contiguous(), a.contiguous(), post_norm="layer", pre_norm="rms", dropout_p=0.1, seed=1)
            assert torch.isfinite(h.float()).all() and torch.equal(z, z2) and torch.equal(h, h2)
            assert torch.equal(counter_dropout(a, 0.2, 1), counter_dropout(a.contiguous(), 0.2, 1))


def test_rows_past_32_bits_of_elements(cuda_device):
    """Rows are worked out alike wherever they lie: the last of 2^32 elements and some, forward and backward."""
    rows, D = (1 << 19) + 3, 8192
    r, a, dz, dh = (torch.empty(rows, D, dtype=torch.bfloat16, device=cuda_device).normal_() for _ in range(4))
    w = torch.randn(D, device=cuda_device).to(torch.bfloat16)

    def step(at):
        v, b = r[at].detach().requires_grad_(), a[at].detach().requires_grad_()
        z, h = residual_norm(v, b, post_norm="rms", post_weight=w, pre_norm="rms", pre_weight=w)
        return [z.detach(), h.detach(), *torch.autograd.grad([z, h], [v, b], [dz[at], dh[at]])]

    whole, end = step(slice(None)), step(slice(rows - 5, rows))
    assert all(torch.equal(x[-5:], y) for x, y in zip(whole, end))


def test_a_gate_of_no_rows(cuda_device):
    for shape, gate in (((0, 8), (8,)), ((3, 0, 8), (3, 1, 8)), ((2, 0), (0,))):
        g = torch.ones(gate, device=cuda_device, requires_grad=True)
        z, _ = residual_norm(torch.zeros(shape, device=cuda_device), torch.zeros(shape, device=cuda_device), gate=g)
        (dg,) = torch.autograd.grad(z, g, torch.zeros(shape, device=cuda_device))
        assert z.shape == shape and not dg.any()


def test_gradients_of_gradients_raise(cuda_device):
    x = torch.randn(4, 16, device=cuda_device, requires_grad=True)
    for y in (counter_dropout(x, 0.5, 1), residual_norm(x, x, pre_norm="rms")[1]):
        (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated twice"):
            torch.autograd.grad(dx.sum(), x)


def test_a_graph_is_used_once_and_inputs_are_guarded(cuda_device):
    x = torch.randn(4, 16, device=cuda_device, requires_grad=True)
    w = torch.ones(16, device=cuda_device, requires_grad=True)
    z, h = residual_norm(x, x, pre_norm="rms", pre_weight=w)
    (z.sum() + h.sum()).backward()
    with pytest.raises(RuntimeError, match="second time"):
        h.sum().backward()
    z, h = residual_norm(x, x, pre_norm="rms", pre_weight=w)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="inplace"):
        h.sum().backward()


def test_backward_through_the_device_thread_and_accumulation(cuda_device):
    """backward() as programs call it, twice, adds to the leaves' gradients."""
    w = torch.ones(48, device=cuda_device, requires_grad=True)
    x, dy = torch.randn(10, 48, device=cuda_device), torch.randn(10, 48, device=cuda_device)
    residual_norm(x, pre_norm="layer", pre_weight=w)[1].backward(dy)
    once = w.grad.clone()
    residual_norm(x, pre_norm="layer", pre_weight=w)[1].backward(dy)
    assert torch.equal(w.grad, 2 * once)


def test_a_step_on_another_stream(cuda_device):
    w = torch.ones(264, device=cuda_device, requires_grad=True)
    x = torch.randn(500, 264, device=cuda_device)

    def step():
        z, h = residual_norm(x, x, pre_norm="rms", pre_weight=w, dropout_p=0.1, seed=2)
        return [z.detach(), h.detach(), *torch.autograd.grad(h, w, x)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [2, 3, 5, 6, 7, 9, 10, 11, 13, 255, 1021, 4099])
def test_dropout_of_rows_that_end_inside_a_piece(cuda_device, dtype, cols):
    x = torch.randn(37, cols, generator=torch.Generator().manual_seed(1)).to(dtype)
    assert torch.equal(counter_dropout(x.to(cuda_device), 0.4, 99, 3).cpu(), expected(x, 0.4, 99, 3))


def test_dropout_of_a_row_past_32_bits_of_bytes(cuda_device):
    x = torch.ones((1 << 31) + 5, dtype=torch.bfloat16, device=cuda_device)
    y = counter_dropout(x, 0.5, 6, 1)
    tail = y[-1027:].cpu()
    groups = torch.arange(((1 << 31) + 5 - 1027) // 4, ((1 << 31) + 5 + 3) // 4).tolist()
    words = [w for c in groups for w in lm_plain.philox7(c, 0, 1, 0, 6, 0)]
    keep = torch.tensor([w >= 1 << 31 for w in words])[((1 << 31) + 5 - 1027) % 4:][:1027]
    assert torch.equal(tail != 0, keep)


@pytest.mark.parametrize("V", [300, 5000, 200000])
def test_histories_too_long_for_a_word(cuda_device, V):
    """From 2^18 tokens on the slots of sparse biases leave the counts' words."""
    for L in ((1 << 18) - 1, 1 << 18, (1 << 18) + 5):
        s = make(2, V, L, K=300, token=torch.int32, seed=L)
        s["tokens"][0] = 7  # one entry, as often as it can be
        check_logits(cuda_device, s["x"], tokens=s["tokens"], rho=1.2, presence=0.5, frequency=2.0 ** -12, ids=s["ids"],
                     values=s["values"])


@pytest.mark.parametrize("K", [4095, 4096, 4097, 9000])
def test_more_sparse_biases_than_a_chunk_has_entries(cuda_device, K):
    for V in (3, 4096, 6000):
        s = make(2, V, K=K, seed=K)
        check_logits(cuda_device, s["x"], ids=s["ids"], values=s["values"] * 2.0 ** -6)


def test_more_sparse_biases_than_slots_in_a_chunk_of_a_long_history(cuda_device):
    """1024 threads have chunks of 8192 entries of two bytes: more entries with a bias than a word has slots for."""
    s = make(2, 8192, 5000, K=9000, seed=4)
    s["ids"][0] = torch.arange(9000) % 8192
    check_logits(cuda_device, s["x"].to(torch.bfloat16), tokens=s["tokens"], rho=1.2, frequency=0.5, ids=s["ids"],
                 values=s["values"])


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,L", [(60, 150001, 8192), (520, 16385, 8200), (3, 33000, 9000), (130, 20000, 4097)])
def test_long_histories_of_many_rows(cuda_device, out, B, V, L):
    s = make(B, V, L, K=100, token=torch.int32)
    check_logits(cuda_device, s["x"].to(torch.bfloat16), dtype=out, tokens=s["tokens"], lengths=s["lengths"],
                 prompts=s["prompts"], rho=1.3, presence=0.5, frequency=0.125, ids=s["ids"], values=s["values"],
                 mask=torch.rand(V, generator=s["gen"]) < 0.7)


@pytest.mark.parametrize("B,K", [(110, 100), (110, 9000), (30, 40000)])
def test_chunks_that_fill_the_lds(cuda_device, B, K):
    """The largest chunks, and with as many sparse biases smaller ones."""
    s = make(B, 150001, 8192, K=K, token=torch.int32)
    check_logits(cuda_device, s["x"], tokens=s["tokens"], lengths=s["lengths"], rho=1.3, frequency=0.125, ids=s["ids"],
                 values=s["values"] * 2.0 ** -6)


@pytest.mark.parametrize("B", [1, 40, 700])
@pytest.mark.parametrize("V", [1023, 1024, 1025, 2049, 4095, 4096, 4097, 9000])
def test_vocabularies_around_a_chunk(cuda_device, B, V):
    s = make(B, V, 60, K=5)
    check_logits(cuda_device, s["x"].to(torch.bfloat16), tokens=s["tokens"], lengths=s["lengths"], prompts=s["prompts"],
                 rho=1.3, presence=0.5, ids=s["ids"], values=s["values"], bias=torch.randn(B, V).to(torch.float16),
                 mask=torch.rand(B, V, generator=s["gen"]) < 0.7)


def test_temperatures_and_penalties_at_the_ends_of_their_type(cuda_device):
    """A reciprocal that overflows is a division: 0 stays 0, and a value of the same size 1."""
    tiny = 2.0 ** -140
    x = torch.tensor([[0.0, -0.0, tiny, -tiny, 1.0, -1.0]], device=cuda_device)
    got = process_logits(x, temperature=tiny)
    inf = float("inf")
    assert got.tolist() == [[0.0, 0.0, 1.0, -1.0, inf, -inf]]
    got = process_logits(x, tokens=torch.arange(6, device=cuda_device)[None], repetition_penalty=tiny)
    assert got[0, 0] == 0 and got[0, 2] == 1.0 and got[0, 4] == inf


def test_logits_in_place_are_seen_by_autograd(cuda_device):
    x = torch.randn(2, 50, device=cuda_device)
    version = x._version
    assert process_logits(x, out=x, temperature=2.0) is x and x._version > version
    leaf = torch.randn(2, 50, device=cuda_device, requires_grad=True)
    with pytest.raises(ValueError, match="require a gradient"):
        process_logits(x, out=leaf)
    with pytest.raises(ValueError, match="overlap"):
        process_logits(x, out=torch.zeros(1, 50, device=cuda_device).expand(2, 50))
    assert not process_logits(leaf).requires_grad


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(cuda_device):
    """The eager graph's leaves belong to the default stream; without it the capture is made."""
    w = torch.ones(64, device=cuda_device, requires_grad=True)
    x, dy = torch.randn(4, 64, device=cuda_device), torch.randn(4, 64, device=cuda_device)
    calls = (lambda: residual_norm(x, pre_norm="rms", pre_weight=w)[1], lambda: counter_dropout(w, 0.5, 1))
    for call in calls:
        call()
        eager = call()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="belongs to the default stream"):
            with torch.cuda.graph(graph):
                y = call()  # forward alone may be captured
                torch.autograd.grad(y, w, dy[:y.shape[0]] if y.dim() == 2 else dy[0])
        del eager, graph, y
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = call()
            (dw,) = torch.autograd.grad(y, w, dy[:y.shape[0]] if y.dim() == 2 else dy[0])
        for _ in range(3):
            x.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y.detach(), call().detach())
        del y, dw


def test_inference_mode(cuda_device):
    x, w = torch.randn(6, 96, device=cuda_device, requires_grad=True), torch.ones(96, device=cuda_device, requires_grad=True)
    want = [counter_dropout(x, 0.5, 1), *residual_norm(x, x, pre_norm="rms", pre_weight=w), process_logits(x, temperature=2.0)]
    with torch.inference_mode():
        got = [counter_dropout(x, 0.5, 1), *residual_norm(x, x, pre_norm="rms", pre_weight=w)]
        y = x.clone()
        got.append(process_logits(y, out=y, temperature=2.0))
    assert all(torch.equal(a, b) for a, b in zip(want, got)) and not any(t.requires_grad for t in got)


def test_steps_leave_nothing_behind(cuda_device):
    x = torch.randn(64, 256, device=cuda_device, requires_grad=True)
    w = torch.ones(256, device=cuda_device, requires_grad=True)
    state = torch.tensor([1, 2], dtype=torch.int64, device=cuda_device)

    def step():
        z, h = residual_norm(x, counter_dropout(x, 0.1, state), pre_norm="rms", pre_weight=w, dropout_p=0.1, seed=state)
        torch.autograd.grad(z.sum() + process_logits(h.detach(), temperature=2.0).sum() + h.sum(), [x, w])

    step()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        step()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_module_counts_only_training_calls(cuda_device):
    m, x = CounterDropout(0.5, seed=3), torch.randn(4, 32, device=cuda_device)
    m.eval()(x)
    assert m.calls == 0
    assert torch.equal(m.train()(x), counter_dropout(x, 0.5, 3, 1))
