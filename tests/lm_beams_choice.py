"""What a beam search's step has chosen, each place looked up in 64 bits: beside lm_tokens_plain.check_select, which
compares with a full sort, this holds every returned (beam, token) to its own score, order and rank."""
import math

import numpy as np
import torch

import lm_tokens_plain as plain


def check_choice(got, logits, scores, n, finished=None, pad=0, lengths=None, length_penalty=0.0):
    """Each returned score is its candidate's; candidates of a beam are its first ones, in their exact order, none
    twice; and the rank of every place is the wanted one's to the error of two scores.

    A beam's scores in 64 bits have one error in common, of its sum of exponentials (plain.select_tolerance without
    the rounding of the result); ranks have it divided by length^length_penalty, and rounding errors of 64 bits."""
    s, parents, tokens = (t.cpu() for t in got)
    x, score = logits.detach().cpu().double().numpy(), scores.cpu().double().numpy()
    B, K, V = x.shape
    want = plain.select(logits, scores, n, finished, pad, lengths, length_penalty)
    error = float(plain.select_tolerance(V, torch.zeros(1, dtype=torch.float64)))
    for b in range(B):
        done = [finished is not None and bool(finished[b, k]) for k in range(K)]
        length = [1.0 if lengths is None else max(1.0, float(lengths[b, k]) + (not done[k])) ** length_penalty for k in range(K)]
        # ranks of one search are taken in their order, so an error of any beam's may move all of them
        worst = max((error / length[k] for k in range(K) if not done[k] and score[b, k] > -math.inf), default=0.0)
        of_beam = {}
        for j in range(n):
            p, t, found, rank = int(parents[b, j]), int(tokens[b, j]), float(s[b, j]), float(want[3][b, j])
            if rank == -math.inf:  # no candidates are left
                assert (found, p, t) == (-math.inf, 0, pad), (b, j)
                continue
            assert score[b, p] != -math.inf, (b, j)
            if done[p]:
                assert t == pad and p not in of_beam, (b, j)
                of_beam[p] = [t]
                true = score[b, p]
            else:
                if p not in of_beam:
                    of_beam[p] = []
                of_beam[p].append(t)
                row = x[b, p]
                unknown = np.isnan(row).any() or (row == math.inf).any() or not score[b, p] < math.inf
                top = row.max() if not unknown else 0.0
                true = math.nan if unknown else row[t] - top - math.log(np.exp(row - top).sum()) + score[b, p]
            if math.isnan(true):
                assert math.isnan(found) and rank == math.inf, (b, j)
                continue
            assert true > -math.inf, (b, j)
            if math.isinf(true):
                assert found == true and rank == true, (b, j)
                continue
            assert abs(found - true) <= (0.0 if done[p] else error + abs(true) * plain.STEP32), (b, j, found, true)
            assert abs(true / length[p] - rank) <= 2 * worst + 1e-12 * abs(rank), (b, j, true / length[p], rank)
        for k, chosen in of_beam.items():
            if done[k]:
                continue
            row = x[b, k]
            unknown = np.isnan(row).any() or (row == math.inf).any() or not score[b, k] < math.inf
            first = np.arange(V) if unknown else np.lexsort((np.arange(V), -row))
            assert chosen == first[:len(chosen)].tolist(), (b, k, chosen, first[:len(chosen)].tolist())
