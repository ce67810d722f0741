"""LUTTransformer.generate_beams on the CPU: a table of logits for the layers, plain torch for the operators."""
import itertools
import math
import sys

import pytest
import torch

from spiky_amd import LUTTransformer
import lm_tokens_plain

VOCAB, CONTEXT = 5, 4


class Table(LUTTransformer):
    """The logits of a position are its token's row of a table."""

    def __init__(self, table):
        torch.nn.Module.__init__(self)
        self.context_size = CONTEXT
        self.table = torch.nn.Parameter(table)

    def forward(self, tokens):
        assert tokens.shape[1] == CONTEXT
        return self.table[tokens.long()]


def plain_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, temperature=1.0, mask=None, presence_penalty=0.0):
    x = logits
    at = torch.arange(tokens.shape[1])
    answered = (at < lengths[:, None]) & (at >= prompt_lengths[:, None])
    said = torch.zeros_like(x).scatter_add_(1, tokens.long(), answered.to(x.dtype)) > 0
    p = torch.as_tensor(presence_penalty, dtype=x.dtype).reshape(-1, 1)
    x = (x - p * said) / torch.as_tensor(temperature, dtype=x.dtype).reshape(-1, 1)
    return x if mask is None else torch.where(mask, x, -math.inf)


def plain_select(logits, scores, n=None, *, finished=None, pad=0, lengths=None, length_penalty=0.0):
    s, parents, tokens, _ = lm_tokens_plain.select(logits, scores, logits.shape[1] if n is None else n, finished, pad, lengths,
                                                   length_penalty)
    return s.float(), parents, tokens


def plain_reorder(states, parents, out=None):
    moved = [x[torch.arange(x.shape[0])[:, None], parents] for x in states]
    for x, y in zip(out, moved):
        x.copy_(y)
    return out


@pytest.fixture
def model(monkeypatch):
    module = sys.modules[LUTTransformer.__module__]
    monkeypatch.setattr(module, "process_logits", plain_logits)
    monkeypatch.setattr(module, "beam_select", plain_select)
    monkeypatch.setattr(module, "reorder_states", plain_reorder)
    return Table(torch.randn(VOCAB, VOCAB, generator=torch.Generator().manual_seed(3)) * 2.0)


def all_continuations(model, last, n_new, end=None, alpha=0.0, **processing):
    """(rank, score, tokens) of every continuation of a prompt that ends in `last`, the best first."""
    found = {}
    for new in itertools.product(range(VOCAB), repeat=n_new):
        score, before, said, kept = 0.0, last, [], []
        for t in new:
            tokens = torch.tensor([said + [0]])
            x = plain_logits(model.table[before][None], tokens=tokens, lengths=torch.tensor([len(said)]),
                             prompt_lengths=torch.tensor([0]), **processing)[0]
            score += float(torch.log_softmax(x.double(), 0)[t])
            kept.append(t)
            said.append(t)
            before = t
            if t == end:
                break
        row = tuple(kept + [0] * (n_new - len(kept)))
        if score > -math.inf:
            found[row] = (score / len(kept) ** alpha, score, row)
    return sorted(found.values(), reverse=True)


def test_enough_beams_find_the_best(model):
    """With a beam for every continuation but for the last token's, the search is exhaustive."""
    prompt = torch.tensor([[1, 2], [3, 4]])
    out, scores = model.generate_beams(prompt, 2, VOCAB)
    for b in range(2):
        best = all_continuations(model, int(prompt[b, -1]), 2)[:VOCAB]
        assert out[b, :, :2].tolist() == [prompt[b].tolist()] * VOCAB
        assert [tuple(r) for r in out[b, :, 2:].tolist()] == [w[2] for w in best]
        assert scores[b].tolist() == pytest.approx([w[1] for w in best], abs=1e-5)


def test_prompts_of_different_lengths_longer_than_the_context(model):
    prompt = torch.tensor([[1, 2, 3, 4, 1, 2], [3, 9, 9, 9, 9, 9]])
    out, scores = model.generate_beams(prompt, 3, VOCAB * VOCAB, lengths=torch.tensor([6, 1]))
    for b, (length, last) in enumerate(((6, 2), (1, 3))):
        best = all_continuations(model, last, 3)[:4]
        assert [tuple(r) for r in out[b, :4, length:length + 3].tolist()] == [w[2] for w in best]
        assert not out[b, :, length + 3:].any()
        assert scores[b, :4].tolist() == pytest.approx([w[1] for w in best], abs=1e-5)


@pytest.mark.parametrize("alpha", [0.0, 1.0])
def test_beams_end(model, alpha):
    prompt = torch.tensor([[2], [4]])
    out, scores = model.generate_beams(prompt, 3, VOCAB * VOCAB, end=1, length_penalty=alpha)
    for b in range(2):
        best = all_continuations(model, int(prompt[b, 0]), 3, end=1, alpha=alpha)[:3]
        assert [tuple(r) for r in out[b, :3, 1:].tolist()] == [w[2] for w in best]
        assert scores[b, :3].tolist() == pytest.approx([w[1] for w in best], abs=1e-5)


def test_the_search_ends_with_its_beams(model):
    calls = []
    model.register_forward_hook(lambda *a: calls.append(1))
    mask = torch.zeros(VOCAB, dtype=torch.bool)
    mask[1] = True
    out, scores = model.generate_beams(torch.tensor([[2, 3]]), 50, 3, end=1, mask=mask)
    assert len(calls) == 1 and out[0, 0].tolist() == [2, 3, 1] + [0] * 49
    assert scores[0].tolist() == [0.0, -math.inf, -math.inf]


def test_options_of_each_prompt(model):
    prompt = torch.tensor([[2], [2], [4]])
    heat, penalty = torch.tensor([0.5, 2.0, 1.0]), torch.tensor([0.0, 1.0, 3.0])
    mask = torch.ones(3, VOCAB, dtype=torch.bool)
    mask[1, 2], mask[2, 0] = False, False
    out, scores = model.generate_beams(prompt, 3, VOCAB * VOCAB, temperature=heat, presence_penalty=penalty, mask=mask)
    for b in range(3):
        best = all_continuations(model, int(prompt[b, 0]), 3, temperature=float(heat[b]), presence_penalty=float(penalty[b]),
                                 mask=mask[b])[:3]
        assert [tuple(r) for r in out[b, :3, 1:].tolist()] == [w[2] for w in best]
        assert scores[b, :3].tolist() == pytest.approx([w[1] for w in best], abs=1e-5)


def test_refusals(model):
    prompt = torch.tensor([[2], [4]])
    for lengths in (torch.tensor([0, 1]), torch.tensor([1, 2])):
        with pytest.raises(ValueError, match="a prompt has 1 to L tokens"):
            model.generate_beams(prompt, 2, 2, lengths=lengths)
    for beams in (0, -1, 65):
        with pytest.raises(ValueError, match="1 to 64"):
            model.generate_beams(prompt, 0, beams)
    with pytest.raises(ValueError, match="no continuation to choose"):
        model.generate_beams(prompt, 2, 2, mask=torch.zeros(VOCAB, dtype=torch.bool))
    model.table.data[4, 1] = math.nan
    with pytest.raises(ValueError, match="no continuation to choose"):
        model.generate_beams(prompt, 2, 2)


def test_modes_and_prompts_stay(model):
    prompt = torch.tensor([[2, 3]])
    model.train()
    out, scores = model.generate_beams(prompt, 0, 2)
    assert out.tolist() == [[[2, 3]] * 2] and scores.tolist() == [[0.0, -math.inf]] and model.training
    model.generate_beams(prompt, 2, 2)
    assert model.training and prompt.tolist() == [[2, 3]]
