"""The joined model on the GPU with tables that hold values, and continuations whose rows differ in
temperature, or that have nothing to choose."""
import pytest
import torch

from spiky_amd import residual_norm
from test_gpu_lm_masks import filled
from test_gpu_lm_model import small

pytestmark = pytest.mark.gpu


def test_each_row_has_its_own_temperature(cuda_device):
    m = filled(small(cuda_device, residual_join=dict(pre_norm="rms")))
    prompts = torch.randint(0, 50, (4, 5), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    largest = m.generate(prompts, 12, temperature=0.0)
    mixed = m.generate(prompts, 12, generator=torch.Generator(cuda_device).manual_seed(1),
                       temperature=torch.tensor([0.0, 5.0, -1.0, 5.0], device=cuda_device))
    assert torch.equal(mixed[[0, 2]], largest[[0, 2]])
    assert not torch.equal(mixed[1], largest[1]) and not torch.equal(mixed[3], largest[3])


@pytest.mark.parametrize("temperature", [1.0, 0.0])
def test_a_row_without_a_token_to_choose_raises(cuda_device, temperature):
    m = filled(small(cuda_device, residual_join=dict(pre_norm="rms")))
    prompts = torch.randint(0, 50, (3, 5), device=cuda_device)
    mask = torch.ones(3, 50, dtype=torch.bool, device=cuda_device)
    mask[1] = False
    with pytest.raises(ValueError, match="no token"):
        m.generate(prompts, 3, temperature=temperature, mask=mask)
    mask[1, 9] = True
    assert m.generate(prompts, 3, temperature=temperature, mask=mask)[1, 5:].tolist() == [9, 9, 9]


def test_largest_logits_of_filled_tables(cuda_device):
    """Without a temperature each new token is the largest logit of the last window, read again by itself."""
    m = filled(small(cuda_device, residual_join=dict(post_norm="rms", pre_norm="layer", gate=0.7, bias=True)))
    prompts = torch.randint(0, 50, (3, 6), generator=torch.Generator().manual_seed(3)).to(cuda_device)
    lengths = torch.tensor([6, 1, 4], device=cuda_device)
    out = m.generate(prompts, 9, lengths=lengths, temperature=0.0)
    assert len(set(out[0].tolist())) > 2
    with torch.no_grad():
        for b, n in enumerate(lengths.tolist()):
            assert torch.equal(out[b, :n], prompts[b, :n])
            for i in range(n, n + 9):
                start = max(0, i - 8)
                window = torch.nn.functional.pad(out[b:b + 1, start:i], (0, 8 - (i - start)))
                assert int(out[b, i]) == int(m.eval()(window)[0, i - start - 1].argmax())


@pytest.mark.parametrize("embedding_dim", [32, (4, 8)])
@pytest.mark.parametrize("no_ffn", [False, True])
def test_plain_joins_of_filled_tables_are_the_unjoined_model(cuda_device, embedding_dim, no_ffn):
    tokens = torch.randint(0, 50, (3, 8), device=cuda_device)
    plain = filled(small(cuda_device, embedding_dim, no_ffn=no_ffn))
    joined = small(cuda_device, embedding_dim, no_ffn=no_ffn, residual_join={})
    joined.load_state_dict(plain.state_dict(), strict=False)
    with torch.no_grad():
        want = plain(tokens)
        assert torch.equal(want, joined(tokens)) and want.abs().max() > 0.1


def test_joined_forward_of_filled_tables_is_its_parts(cuda_device):
    m = filled(small(cuda_device, residual_join=dict(post_norm="rms", pre_norm="layer", gate=0.5, bias=True))).eval()
    tokens = torch.randint(0, 50, (2, 8), device=cuda_device)
    with torch.no_grad():
        z = x = m.token_embedder(tokens)
        for block in m.layers:
            for join, branch in (("attention_join", lambda x: block["attention_lut"](x)),
                                 ("ffn_join", lambda x: block["ffn"](x.reshape(16, 1, 32)).reshape(2, 8, 32))):
                j, b = block[join], branch(x)
                assert b.abs().max() > 0.1
                z, x = residual_norm(z, b, post_norm="rms", post_weight=j.post_weight, post_bias=j.post_bias, gate=j.gate,
                                     pre_norm="layer", pre_weight=j.pre_weight, pre_bias=j.pre_bias)
        assert torch.equal(m(tokens), m.unembedder(x.reshape(16, 1, 32)).reshape(2, 8, 50))
