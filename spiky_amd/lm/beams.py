"""A step of a beam search: the selection over beams and vocabulary, and the states that follow it."""
from .. import _native


def beam_select(logits, scores, n=None, *, finished=None, pad=0, lengths=None, length_penalty=0.0):
    """(scores, parents, tokens), each [B, n]: of the continuations of K beams in each of B searches,
    the n of largest score, the largest first.

    Beam k continued by token v has the score

        s = scores[k] + log_softmax(logits[k])[v]

    and a beam that has finished has one continuation, the token `pad`, with its own score.  They are
    ordered by s / length ** length_penalty, where length is lengths[k], plus 1 if the beam has not
    finished, and at least 1; of equal ones, the lower beam comes first, then the larger logit, then
    the lower token.  `scores` of the result are s itself.  Continuations of score -infinity (masked
    tokens, and all of a beam whose score is -infinity, as the others' before a search's first step)
    are not chosen: where there are fewer than n, the rest is -infinity, beam 0 and `pad`.  A beam that
    has not finished and whose score or logits hold NaN or +infinity has scores of NaN, which rank as
    +infinity, in the order of its tokens.

    logits: [B, K, V], float32, bfloat16 or float16 on a HIP device, the vocabulary contiguous, rows at
    any distance.  scores: float32 [B, K].  n: K without.  finished: bool [B, K].  lengths: int32 or
    int64 [B, K].  K and n are at most 64, the penalty -8 to 8.  Scores are float32, parents and tokens
    int64; the order is that of the scores in 64 bits, over exponentials and sums of them in 32.  There
    is no gradient."""
    return _native.lm().beam_select(logits, scores, n, finished, pad, lengths, length_penalty)


def reorder_states(states, parents, out=None):
    """states[b, parents[b, j]] at [b, j], for one tensor [B, K, ...] or a list or tuple of them, of any
    types and shapes behind the same [B, K]; zeros where a parent is outside 0..K-1.

    parents: int32 or int64 [B, n].  Returns new tensors, a list where the states are one, or `out`:
    tensors of the results' shapes that share no memory with the states, or `states` themselves, which
    are then reordered in place (n = K, at most 64; beams that stay where they are cost nothing).  A
    cache of which some positions are in use is passed as a view of these, without a copy where the
    dimensions behind [B, K] are contiguous but for one, as they have to be of `out`.  There is no
    gradient."""
    return _native.lm().reorder_states(states, parents, out)
