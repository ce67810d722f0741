"""Plain 64-bit forms of the embedding's gradient and of a beam search's step, on the CPU, with the
magnitudes that the tolerances of their tests are counted in."""
import math

import numpy as np
import torch

STEP32 = 2.0 ** -24  # half a step of float32, relative


def embed(tokens, weight, scale, dtype):
    """The operator's own arithmetic: one 32-bit product, rounded to dtype."""
    t, w = tokens.cpu().long(), weight.detach().cpu()
    there = (t >= 0) & (t < w.shape[0])
    y = torch.zeros(*t.shape, w.shape[1])
    y[there] = w[t[there]].float() * torch.tensor(scale, dtype=torch.float32)
    return y.to(dtype)


def embed_gradient(tokens, dy, vocab, scale):
    """The sums, and for each the bound of its rounding errors in 32 bits: a sum of m terms has m - 1
    additions, each off by at most half a step of a partial sum, and one product behind it."""
    t, d = tokens.cpu().reshape(-1).long(), dy.detach().cpu().double().reshape(tokens.numel(), -1)
    there = (t >= 0) & (t < vocab)
    scale = float(np.float32(scale))
    sums = torch.zeros(vocab, d.shape[1], dtype=torch.float64).index_add_(0, t[there], d[there]) * scale
    sizes = torch.zeros_like(sums).index_add_(0, t[there], d[there].abs()) * abs(scale)
    counts = torch.bincount(t[there], minlength=vocab).double()[:, None]
    return sums, sizes * (counts + 1.0) * STEP32


def select(logits, scores, n, finished=None, pad=0, lengths=None, length_penalty=0.0):
    """(scores, parents, tokens, ranks): the first n candidates of each search, and their ranks."""
    x = logits.detach().cpu().double().numpy()
    score = scores.cpu().double().numpy()
    B, K, V = x.shape
    found = []
    for b in range(B):
        s, beam, logit, token, rank = [], [], [], [], []
        for k in range(K):
            done = finished is not None and bool(finished[b, k])
            if score[b, k] == -math.inf:
                continue
            if done:
                at, value, key = np.array([pad]), score[b, k:k + 1], np.zeros(1)
            else:
                row = x[b, k]
                unknown = np.isnan(row).any() or (row == math.inf).any() or not score[b, k] < math.inf
                if unknown:
                    at, value, key = np.arange(V), np.full(V, math.nan), np.zeros(V)
                else:
                    at = np.flatnonzero(row > -math.inf)
                    key = row[at]
                    top = key.max(initial=-math.inf)
                    value = key - top - (math.log(np.exp(key - top).sum()) if len(key) else 0.0) + score[b, k]
            length = 1.0
            if lengths is not None:
                length = max(1.0, float(lengths[b, k]) + (0.0 if done else 1.0))
            with np.errstate(invalid="ignore"):
                r = value / length ** length_penalty
            s.append(value)
            beam.append(np.full(len(at), k))
            logit.append(key)
            token.append(at)
            rank.append(np.where(np.isnan(r), math.inf, r))
        s, beam, logit, token, rank = (np.concatenate(v) if v else np.zeros(0) for v in (s, beam, logit, token, rank))
        order = np.lexsort((token, -logit, beam, -rank))[:n]
        rows = [(s[i], int(beam[i]), int(token[i]), rank[i]) for i in order]
        rows += [(-math.inf, 0, pad, -math.inf)] * (n - len(rows))
        found.append(rows)
    return tuple(torch.tensor([[r[i] for r in rows] for rows in found], dtype=torch.int64 if i in (1, 2) else torch.float64)
                 .reshape(B, n) for i in range(4))


def select_tolerance(vocab, want):
    """The sum of exponentials: at most 44 additions in a row and one rounding of each exponential (4
    half steps), and exponents off by 3 half steps of their size, whose average under the softmax is at
    most log(vocab); the result is rounded once more."""
    return (48 + 3 * math.log(max(vocab, 2))) * STEP32 + want.abs().nan_to_num(posinf=0.0, neginf=0.0) * STEP32


def check_select(got, logits, scores, n, **how):
    """The scores, and the choice: equal but where candidates of two beams are nearer than the tolerance."""
    want = select(logits, scores, n, **how)
    s, parents, tokens = (t.cpu() for t in got)
    assert s.dtype == torch.float32 and parents.dtype == tokens.dtype == torch.int64
    bound = select_tolerance(logits.shape[-1], want[0])
    assert torch.equal(s.isnan(), want[0].isnan()) and torch.equal(s == -math.inf, want[0] == -math.inf)
    # infinities that are equal have no difference
    assert not ((s.double() - want[0]).abs() > bound).any()
    differ = (parents != want[1]) | (tokens != want[2])
    if differ.any():
        rank = want[3]
        near = torch.zeros_like(differ)
        gap = (rank[:, 1:] - rank[:, :-1]).abs() <= 2 * bound[:, 1:]
        near[:, 1:] |= gap
        near[:, :-1] |= gap & (want[1][:, 1:] != want[1][:, :-1])
        near[:, -1] = True  # the next one may be as near
        assert not (differ & ~near).any(), (got, want)
        assert float(differ.float().mean()) < 0.05
