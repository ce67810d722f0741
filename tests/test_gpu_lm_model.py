"""The language-model operators together: a LUT transformer with joined blocks, and its continuations."""
import os
import sys

import pytest
import torch

from spiky_amd import LUTTransformer, residual_norm

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
import byte_model  # noqa: E402

pytestmark = pytest.mark.gpu


def small(device, embedding_dim=32, dropout=0.0, **kw):
    how = dict(vocab_size=50, embedding_dim=embedding_dim, context_size=8, positional_dim=2, num_layers=2, num_heads=2,
               n_detectors=4, n_anchors_per_detector=4, n_anchors_per_detector_attention=3, device=device, seed=5,
               dropout=dropout)
    return LUTTransformer(**{**how, **kw})


@pytest.mark.parametrize("embedding_dim", [32, (4, 8)])
@pytest.mark.parametrize("no_ffn", [False, True])
def test_plain_joins_are_the_unjoined_model(cuda_device, embedding_dim, no_ffn):
    """Without norms, gate and dropout a join is z + branch, bit for bit: one sum in 32 bits."""
    tokens = torch.randint(0, 50, (3, 8), device=cuda_device)
    plain = small(cuda_device, embedding_dim, no_ffn=no_ffn)
    joined = small(cuda_device, embedding_dim, no_ffn=no_ffn, residual_join={})
    joined.load_state_dict(plain.state_dict(), strict=False)
    with torch.no_grad():
        assert torch.equal(plain(tokens), joined(tokens))


def test_joined_forward_is_its_parts(cuda_device):
    m = small(cuda_device, residual_join=dict(post_norm="rms", pre_norm="layer", gate=0.5, bias=True)).eval()
    tokens = torch.randint(0, 50, (2, 8), device=cuda_device)
    with torch.no_grad():
        z = x = m.token_embedder(tokens)
        for block in m.layers:
            for join, layer in (("attention_join", "attention_lut"), ("ffn_join", "ffn")):
                b = block[layer](x) if layer == "attention_lut" else block[layer](x.reshape(16, 1, 32)).reshape(2, 8, 32)
                j = block[join]
                z, x = residual_norm(z, b, post_norm="rms", post_weight=j.post_weight, post_bias=j.post_bias, gate=j.gate,
                                     pre_norm="layer", pre_weight=j.pre_weight, pre_bias=j.pre_bias)
        want = m.unembedder(x.reshape(16, 1, 32)).reshape(2, 8, 50)
        assert torch.equal(m(tokens), want)


def test_every_parameter_of_a_joined_model_has_a_gradient(cuda_device):
    m = small(cuda_device, dropout=0.1, residual_join=dict(post_norm="rms", pre_norm="rms", gate=0.5))
    tokens = torch.randint(0, 50, (4, 8), device=cuda_device)
    m(tokens).square().sum().backward()
    joins = [p for n, p in m.named_parameters() if "_join" in n]
    assert len(joins) == 12 and all(p.grad is not None and torch.isfinite(p.grad).all() for p in joins)


def test_joins_exclude_batch_norm(cuda_device):
    with pytest.raises(ValueError, match="exclude"):
        small(cuda_device, use_batch_norm=True, residual_join={})


def test_continuations(cuda_device):
    m = small(cuda_device, residual_join=dict(post_norm="rms", pre_norm="rms"))
    prompts = torch.randint(1, 50, (3, 6), device=cuda_device)
    lengths = torch.tensor([6, 1, 4], device=cuda_device)
    mask = torch.zeros(50, dtype=torch.bool, device=cuda_device)
    mask[10:20] = True
    out = m.generate(prompts, 7, lengths=lengths, generator=torch.Generator(cuda_device).manual_seed(1), mask=mask,
                     repetition_penalty=1.2, temperature=0.9)
    assert out.shape == (3, 13) and m.training
    for b, n in enumerate(lengths.tolist()):
        assert torch.equal(out[b, :n], prompts[b, :n])
        new = out[b, n:n + 7]
        assert ((new >= 10) & (new < 20)).all() and not out[b, n + 7:].any()
    again = m.generate(prompts, 7, lengths=lengths, generator=torch.Generator(cuda_device).manual_seed(1), mask=mask,
                       repetition_penalty=1.2, temperature=0.9)
    assert torch.equal(out, again)
    # a row's continuation does not depend on the others
    alone = m.generate(prompts[1:2, :1], 7, temperature=0.0, presence_penalty=0.5)
    among = m.generate(prompts, 7, lengths=lengths, temperature=0.0, presence_penalty=0.5)
    assert torch.equal(alone[0], among[1, :8])
    with pytest.raises(ValueError, match="1 to L"):
        m.generate(prompts, 2, lengths=torch.tensor([0, 1, 2], device=cuda_device))


def test_greedy_continuation_is_the_largest_logit(cuda_device):
    m = small(cuda_device, residual_join=dict(pre_norm="rms"))
    prompt = torch.randint(0, 50, (1, 5), device=cuda_device)
    out = m.generate(prompt, 6, temperature=0.0)
    with torch.no_grad():
        for i in range(5, 11):
            start = max(0, i - 8)
            window = torch.nn.functional.pad(out[:, start:i], (0, 8 - (i - start)))
            assert int(out[0, i]) == int(m.eval()(window)[0, i - start - 1].argmax())


def test_example_learns(cuda_device):
    model = byte_model.make(cuda_device, context=32)
    losses = byte_model.train(model, byte_model.text()[:20000], 30, batch=8)
    assert sum(losses[-5:]) / 5 < losses[0] - 0.5
