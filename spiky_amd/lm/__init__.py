"""Operators around the LUT blocks of a language model: token embeddings, dropout, the residual join,
logits, and the steps of a beam search."""
from .beams import beam_select, reorder_states  # noqa: F401
from .common import mask_counters  # noqa: F401
from .dropout import CounterDropout, counter_dropout  # noqa: F401
from .embedding import TokenEmbedding, embed_tokens  # noqa: F401
from .logits import process_logits  # noqa: F401
from .residual import ResidualNorm, residual_norm  # noqa: F401
