"""LUTTransformer's joined forward on the CPU, with plain layers and a plain join in the library's place."""
import pickle
import sys

import pytest
import torch

from spiky_amd import LUTTransformer, ResidualNorm

E, S, B, V = 12, 4, 3, 20


class Layer(torch.nn.Module):
    """A product in the place of a LUT layer."""

    def __init__(self, weight):
        super().__init__()
        self.weight = weight

    def forward(self, x):
        y = x.reshape(-1, E) @ self.weight
        return y.reshape(x.shape if x.dim() == 4 else (*x.shape[:-1], -1))


def model(embedding_dim=E, no_ffn=False, **kw):
    gen = torch.Generator().manual_seed(1)
    m = LUTTransformer(vocab_size=V, embedding_dim=embedding_dim, context_size=S, positional_dim=2, num_layers=2, num_heads=2,
                       n_detectors=4, n_anchors_per_detector=3, seed=1, no_ffn=no_ffn, **kw)
    for block in m.layers:
        for name in ("attention_lut", "ffn"):
            if name in block:
                block[name] = Layer(torch.randn(E, E, generator=gen))
    m.unembedder = Layer(torch.randn(E, V, generator=gen))
    return m.eval()


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(sys.modules[ResidualNorm.__module__], "residual_norm",
                        lambda residual, branch, **how: (residual + branch, None))


@pytest.mark.parametrize("embedding_dim", [E, (3, 4)])
@pytest.mark.parametrize("no_ffn", [False, True])
def test_a_joined_forward_keeps_what_the_plain_one_does(embedding_dim, no_ffn):
    """_debug_last_forward: the tokens, the embedding and each layer's branch; kept only if it is a list."""
    tokens = torch.randint(0, V, (B, S))
    seen = []
    for kw in ({}, dict(residual_join={})):
        m = model(embedding_dim, no_ffn, **kw)
        m(tokens)
        assert m._debug_last_forward is None
        m._debug_last_forward = []
        out = m(tokens)
        seen.append([out, *m._debug_last_forward])
    assert len(seen[0]) == len(seen[1]) == 3 + (2 if no_ffn else 4)
    assert all(a.shape == b.shape and torch.equal(a, b) for a, b in zip(*seen))


def test_a_model_pickled_without_joins_runs():
    """One of before there were joins has no attribute of them."""
    m = model()
    want = m(torch.arange(B * S).reshape(B, S))
    del m.__dict__["residual_join"]
    old = pickle.loads(pickle.dumps(m))
    assert "residual_join" not in old.__dict__ and torch.equal(old(torch.arange(B * S).reshape(B, S)), want)


def test_joins_have_the_dropout_of_a_joined_model():
    """No module is made that no call reaches."""
    def dropouts(m):
        return [x for x in m.modules() if isinstance(x, torch.nn.Dropout)]

    assert len(dropouts(model(dropout=0.1))) == 4 and not dropouts(model(dropout=0.1, residual_join={}))
    joined = model(dropout=0.1, residual_join={})
    assert [x.dropout_p for x in joined.modules() if isinstance(x, ResidualNorm)] == [0.1] * 4
