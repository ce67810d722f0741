"""Tangents that the steps of a beam search do not have; checked before the device is."""
import pytest
import torch
from torch.autograd import forward_ad

from spiky_amd import beam_select, reorder_states


def test_tangents_are_refused():
    x, scores, parents = torch.randn(2, 3, 4), torch.randn(2, 3), torch.zeros(2, 3, dtype=torch.int64)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: beam_select(dual(x), scores), lambda: beam_select(x, dual(scores)),
                     lambda: reorder_states(dual(x), parents), lambda: reorder_states([x, dual(x)], parents),
                     lambda: reorder_states(x, parents, out=dual(x)), lambda: reorder_states((x, x), parents, out=(x, dual(x)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
    for call in (lambda: beam_select(x, scores), lambda: reorder_states([x, x], parents, out=[x, x])):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call()
