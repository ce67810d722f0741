"""The check of a beam search's choice, on the CPU: it holds for the plain form, and finds each mistake."""
import math

import pytest
import torch

import lm_tokens_plain as plain
from lm_beams_choice import check_choice


def chosen(n, seed=0, **how):
    gen = torch.Generator().manual_seed(seed)
    x, scores = torch.randn(3, 2, 501, generator=gen) * 4, -10 * torch.rand(3, 2, generator=gen)
    got = plain.select(x, scores, n, **how)
    return x, scores, [got[0].float(), got[1], got[2]]


@pytest.mark.parametrize("how", [{}, dict(finished=torch.tensor([[True, False], [False, False], [True, True]]), pad=7),
                                 dict(lengths=torch.tensor([[3, 9], [1, 1], [40, 0]]), length_penalty=0.7)])
def test_the_plain_choice_holds(how):
    for n in (1, 5, 64):
        x, scores, got = chosen(n, **how)
        check_choice(got, x, scores, n, **how)


def test_unknown_and_masked_beams_hold():
    x, scores, _ = chosen(1)
    x[0, 1, 4], x[1] = math.nan, -math.inf
    scores[2, 0] = math.inf
    got = plain.select(x, scores, 6)
    check_choice([got[0].float(), *got[1:3]], x, scores, 6)


@pytest.mark.parametrize("place", [0, 30, 63])
def test_one_wrong_place_is_found(place):
    x, scores, got = chosen(64)
    for wrong in ("token", "parent", "score", "twice", "order"):
        s, p, t = (v.clone() for v in got)
        if wrong == "token":
            t[1, place] = (t[1, place] + 17) % 501
        elif wrong == "parent":
            p[1, place] = 1 - p[1, place]
        elif wrong == "score":
            s[1, place] += 1e-3
        elif wrong == "twice":
            other = place - 1 if place else 1
            s[1, place], p[1, place], t[1, place] = s[1, other], p[1, other], t[1, other]
        else:  # two of one beam
            i, j = [k for k in range(64) if p[1, k] == p[1, place]][:2] if place < 32 else \
                [k for k in range(64) if p[1, k] == p[1, place]][-2:]
            for v in (s, t):
                v[1, i], v[1, j] = v[1, j].clone(), v[1, i].clone()
        with pytest.raises(AssertionError):
            check_choice((s, p, t), x, scores, 64)
