"""LUTTransformer.generate on the CPU: a table of logits for the layers, plain torch for process_logits."""
import math
import sys

import numpy as np
import pytest
import torch

from spiky_amd import LUTTransformer

VOCAB, CONTEXT = 7, 4


class Table(LUTTransformer):
    """The logits of a position are its token's row of a table."""

    def __init__(self, table):
        torch.nn.Module.__init__(self)
        self.context_size = CONTEXT
        self.table = torch.nn.Parameter(table)

    def forward(self, tokens):
        return self.table[tokens.long()]


def plain(logits, *, tokens=None, lengths=None, prompt_lengths=None, temperature=1.0, mask=None):
    """process_logits with a temperature and a mask alone."""
    t = torch.as_tensor(temperature, dtype=logits.dtype).reshape(-1, 1)
    x = torch.where(t > 0, logits / torch.where(t > 0, t, 1.0), logits)
    return x if mask is None else torch.where(mask, x, -math.inf)


@pytest.fixture
def model(monkeypatch):
    monkeypatch.setattr(sys.modules[LUTTransformer.__module__], "process_logits", plain)
    # flat rows, in which a draw seldom meets the largest, and each token's largest another one
    return Table(torch.eye(VOCAB)[(torch.arange(VOCAB) * 3 + 1) % VOCAB] * 0.1)


def greedy(model, tokens, n_new):
    out = tokens.tolist()
    for row in out:
        for _ in range(n_new):
            row.append(int(model.table[row[-1]].argmax()))
    return torch.tensor(out)


def test_each_row_has_its_own_temperature(model):
    """Rows of temperature 0 or less get the largest whatever the other rows do, and those are drawn."""
    prompt = torch.tensor([[1, 2], [3, 4], [5, 6], [0, 1]])
    want = greedy(model, prompt, 20)
    temperature = torch.tensor([0.0, 1.0, -1.0, 1.0])
    out = model.generate(prompt, 20, generator=torch.Generator().manual_seed(0), temperature=temperature)
    assert torch.equal(out[[0, 2]], want[[0, 2]])
    assert not torch.equal(out[1], want[1]) and not torch.equal(out[3], want[3])
    for cold in (torch.zeros(4), 0.0, np.float32(0.0)):
        assert torch.equal(model.generate(prompt, 20, temperature=cold), want)


def test_rows_without_a_temperature_of_their_own_are_drawn_as_ever(model):
    """A tensor of one temperature draws what the number draws."""
    prompt = torch.tensor([[1, 2], [3, 4]])
    one, each = (model.generate(prompt, 9, generator=torch.Generator().manual_seed(4), temperature=t)
                 for t in (0.5, torch.full((2,), 0.5)))
    assert torch.equal(one, each)


@pytest.mark.parametrize("temperature", [1.0, 0.0, torch.tensor([1.0, 0.0, 0.7])])
def test_a_row_without_a_token_to_choose_raises(model, temperature, monkeypatch):
    """A mask that leaves nothing, and NaN: raised by the host, with no draw from what is no distribution."""
    draw, prompt = torch.multinomial, torch.tensor([[1, 2], [3, 4], [5, 6]])
    drawn = []

    def checked(p, *args, **kw):
        drawn.append(bool(torch.isfinite(p).all() and (p.sum(-1) > 0).all()))
        return draw(p, *args, **kw)

    monkeypatch.setattr(torch, "multinomial", checked)
    for row in range(3):
        mask = torch.ones(3, VOCAB, dtype=torch.bool)
        mask[row] = False
        with pytest.raises(ValueError, match="no token"):
            model.generate(prompt, 3, temperature=temperature, mask=mask)
        mask[row, 2] = True
        assert model.generate(prompt, 3, temperature=temperature, mask=mask)[row, 2:].tolist() == [2, 2, 2]
    with torch.no_grad():
        model.table[4, 1] = math.nan
    with pytest.raises(ValueError, match="no token"):
        model.generate(prompt, 3, temperature=temperature)
    assert all(drawn)


def test_submodules_keep_their_mode(model):
    """What was held in evaluation stays there."""
    model.frozen, model.other = torch.nn.Dropout(0.5).eval(), torch.nn.Dropout(0.5)
    for training in (True, False):
        model.training = training
        model.generate(torch.tensor([[1, 2]]), 2)
        assert model.training is training and not model.frozen.training and model.other.training
    modes = []
    model.register_forward_pre_hook(lambda m, _: modes.extend(x.training for x in m.modules()))
    model.generate(torch.tensor([[1, 2]]), 2)
    assert modes and not any(modes)
