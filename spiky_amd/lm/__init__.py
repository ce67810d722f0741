"""Operators around the LUT blocks of a language model: dropout, the residual join, logits."""
from .common import mask_counters  # noqa: F401
from .dropout import CounterDropout, counter_dropout  # noqa: F401
from .logits import process_logits  # noqa: F401
from .residual import ResidualNorm, residual_norm  # noqa: F401
