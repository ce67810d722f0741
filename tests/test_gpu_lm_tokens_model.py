"""The operators at both ends of a model together: a LUTTransformer that trains its embedding and is
searched for continuations."""
import pickle

import pytest
import torch

from spiky_amd import LUTTransformer, TokenEmbedding
import lm_tokens_plain as plain

pytestmark = pytest.mark.gpu


def make(device, vocab=61, context=16, **how):
    return LUTTransformer(vocab_size=vocab, embedding_dim=32, context_size=context, positional_dim=4, num_layers=2, num_heads=2,
                          n_detectors=8, n_anchors_per_detector=5, n_anchors_per_detector_attention=3, device=device, seed=2,
                          residual_join=dict(post_norm="rms", pre_norm="rms"), **how)


def fill(model):
    """Tables that hold values."""
    gen = torch.Generator().manual_seed(7)
    with torch.no_grad():
        for layer in model._lut_layers():
            layer._weights.copy_(torch.randn(layer._weights.shape, generator=gen) * 0.3)
    return model


def test_the_embedding_is_frozen_without_options(cuda_device):
    model = make(cuda_device)
    assert type(model.token_embedder) is torch.nn.Embedding and not model.token_embedder.weight.requires_grad
    trained = make(cuda_device, train_embedding=True)
    assert torch.equal(model.token_embedder.weight, trained.token_embedder.weight) and trained.token_embedder.weight.requires_grad
    assert isinstance(make(cuda_device, embedding_scale=2.0).token_embedder, TokenEmbedding)
    assert not make(cuda_device, embedding_scale=2.0).token_embedder.weight.requires_grad
    tokens = torch.randint(0, 61, (3, 16), device=cuda_device)
    fill(model), fill(trained)
    with torch.no_grad():
        assert torch.equal(model(tokens), trained(tokens))
    trained.load_state_dict(model.state_dict())


@pytest.mark.parametrize("scale", [1.0, 3.0])
def test_the_embeddings_gradient(cuda_device, scale):
    model = fill(make(cuda_device, train_embedding=True, embedding_scale=scale))
    seen = []
    model.token_embedder.register_forward_hook(lambda m, a, y: (y.retain_grad(), seen.append(y))[1])
    tokens = torch.randint(0, 61, (5, 16), device=cuda_device)
    torch.nn.functional.cross_entropy(model(tokens)[:, :-1].reshape(-1, 61), tokens[:, 1:].reshape(-1)).backward()
    sums, errors = plain.embed_gradient(tokens, seen[0].grad, 61, scale)
    grad = model.token_embedder.weight.grad
    assert float(grad.abs().max()) > 0
    assert bool(((grad.cpu().double() - sums).abs() <= errors + sums.abs() * plain.STEP32).all())


def test_a_captured_training_step(cuda_device):
    """Forward, gradients and the update of the embedding in one graph, against the same steps run eagerly."""
    torch.manual_seed(0)
    model = fill(make(cuda_device, train_embedding=True))
    other = fill(make(cuda_device, train_embedding=True))
    tokens = torch.randint(0, 61, (4, 16), device=cuda_device)

    def step(m):
        loss = m(tokens)[:, :-1].float().square().mean()
        weight = m.token_embedder.weight
        (g,) = torch.autograd.grad(loss, weight)
        with torch.no_grad():
            weight.sub_(g * 50.0)
        return g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(other)  # scratch grows before the capture
    torch.cuda.current_stream().wait_stream(side)
    other.load_state_dict(model.state_dict())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g = step(other)
    other.load_state_dict(model.state_dict())
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = step(model)
        torch.cuda.synchronize()
        # LUT gradients are committed with atomics in any order: equal within their bar
        assert float((g - want).abs().max()) <= 1e-4 * float(want.abs().max())
        other.load_state_dict(model.state_dict())
        tokens.copy_(torch.randint(0, 61, (4, 16), device=cuda_device))


def test_training_then_searching(cuda_device):
    model = fill(make(cuda_device, train_embedding=True, embedding_scale=1.5))
    optimizer = torch.optim.Adam(model.parameters(), lr=0.01)
    before = model.token_embedder.weight.detach().clone()
    for i in range(3):
        tokens = torch.randint(0, 61, (8, 16), device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(i))
        loss = torch.nn.functional.cross_entropy(model(tokens)[:, :-1].reshape(-1, 61), tokens[:, 1:].reshape(-1))
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
    assert bool((model.token_embedder.weight != before).any(1).all())
    prompt = torch.tensor([[1, 2, 3], [4, 5, 0]], device=cuda_device)
    lengths = torch.tensor([3, 2], device=cuda_device)
    out, scores = model.generate_beams(prompt, 8, 4, lengths=lengths, temperature=0.9)
    assert out.shape == (2, 4, 11) and bool((scores[:, :-1] >= scores[:, 1:]).all())
    assert len({tuple(r) for r in out[0].tolist()}) == 4
    # the scores are the sums of the log-probabilities of the sequences' tokens
    for b, n in enumerate(lengths.tolist()):
        whole = torch.cat([out[b], out.new_zeros(4, 5)], 1)[:, :16]
        with torch.no_grad():
            x = model.eval()(whole).double() / 0.9
        p = torch.log_softmax(x, -1)
        want = sum(p[torch.arange(4), i - 1, whole[:, i]] for i in range(n, n + 8))
        # 8 steps' logits rounded once each by the temperature's reciprocal, and sums of 32 bits
        size = float(x.abs().max()) + float(want.abs().max())
        assert float((want - scores[b].double()).abs().max()) <= 8 * (3 * size + 60) * plain.STEP32


def test_one_beam_is_the_largest_logit(cuda_device):
    model = fill(make(cuda_device))
    prompt = torch.randint(0, 61, (3, 5), device=cuda_device)
    lengths = torch.tensor([5, 1, 3], device=cuda_device)
    out, scores = model.generate_beams(prompt, 20, 1, lengths=lengths)  # past the context
    assert torch.equal(out[:, 0], model.generate(prompt, 20, lengths=lengths, temperature=0.0))
    end = int(out[0, 0, 9])
    short, _ = model.generate_beams(prompt, 20, 1, lengths=lengths, end=end)
    for b, n in enumerate(lengths.tolist()):
        row = out[b, 0, n:].tolist()
        stop = row.index(end) + 1 if end in row else 20
        assert short[b, 0, n:n + 20].tolist() == row[:stop] + [0] * (20 - stop)


def test_options_and_pickles(cuda_device):
    model = fill(make(cuda_device, train_embedding=True))
    prompt = torch.randint(0, 61, (2, 5), device=cuda_device)
    mask = torch.zeros(61, dtype=torch.bool, device=cuda_device)
    mask[[3, 17, 40]] = True
    heat = torch.tensor([0.5, 2.0], device=cuda_device)
    out, scores = model.generate_beams(prompt, 6, 5, end=40, length_penalty=1.0, temperature=heat, mask=mask,
                                       repetition_penalty=1.2, presence_penalty=torch.tensor([0.1, 0.4], device=cuda_device))
    assert set(out[:, :, 5:].unique().tolist()) <= {0, 3, 17, 40}
    with pytest.raises(ValueError, match="no continuation to choose"):
        model.generate_beams(prompt, 2, 2, mask=torch.zeros_like(mask))
    with pytest.raises(ValueError, match="1 to 64"):
        model.generate_beams(prompt, 2, 65)
    again = pickle.loads(pickle.dumps(model.to("cpu"))).to(cuda_device)
    model.to(cuda_device)
    assert torch.equal(again.generate_beams(prompt, 6, 5)[0], model.generate_beams(prompt, 6, 5)[0])
