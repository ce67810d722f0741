"""Dropout whose mask is a function of a counter and is never stored."""
import torch

from .. import _native
from .common import CountedMasks, check_probability


def counter_dropout(x, p, seed, offset=0):
    """x / (1 - p) where an element is kept, 0 where it is dropped (infinities and NaN too).

    Whether the element at row r, column c of x, seen as rows of its last dimension, is kept is a
    function of (seed, offset, r, c): word c % 4 of Philox4x32-7 under key `seed` and counter
    (c // 4, r, offset), kept from floor(p * 2**32 + 1/2) on.  So the same call gives the same
    mask, for any type, stride or size of launch, and the backward pass makes it again.  Use
    another offset for each call of a step.

    x: float32, bfloat16 or float16 on a HIP device, any shape.  seed, offset: whole numbers of
    64 bits, or seed an int64 device tensor of [seed, offset], read when the kernels run (for
    graphs whose replays advance it in place, after the backward pass).  Tensors with forward-mode
    tangents are refused."""
    return _native.lm().dropout(x, p, seed, offset)


class CounterDropout(CountedMasks, torch.nn.Module):
    """nn.Dropout over counter_dropout: call number n of a module in training uses offset n.

    Modules of one model take different seeds.  The calls' number is part of the state dict, so a
    resumed run goes on with masks that it has not used.  Inside a backward pass (recomputed by
    torch.utils.checkpoint) and in a captured graph a call raises, unless the model has
    mask_counters."""

    def __init__(self, p=0.5, seed=0):
        super().__init__()
        check_probability(p)
        self.p = float(p)
        self.count_masks(seed)

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        return counter_dropout(x, self.p, *self.next_mask(x))

    def extra_repr(self):
        return f"p={self.p}, seed={self.seed}"
