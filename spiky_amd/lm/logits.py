"""What happens to logits before a token is chosen: penalties, biases, temperature, masks."""
from .. import _native


def process_logits(logits, *, tokens=None, lengths=None, prompt_lengths=None, repetition_penalty=1.0,
                   presence_penalty=0.0, frequency_penalty=0.0, bias=None, bias_ids=None, bias_values=None,
                   temperature=1.0, mask=None, out=None, dtype=None):
    """Logits [B, V] made ready for the choice of each row's next token.  In this order:

        x = logits + bias + the sum of a row's bias_values at its bias_ids
        x = x / repetition_penalty where x > 0, else x * repetition_penalty,
            for entries among the row's tokens
        x = x - frequency_penalty * n - presence_penalty
            for entries that n > 0 of the row's tokens after the prompt are
        x = x / temperature              (rows of temperature 0 or less stay as they are)
        x = -inf where the mask leaves an entry out, whatever it holds; a row whose mask leaves
            nothing is all -inf

    logits: float32, bfloat16 or float16, columns contiguous, rows at any distance (the last
    positions of a [B, S, V] tensor need no copy).  tokens: int32 or int64 [B, L], of which a
    row's first `lengths` count (all, without) and of those the first `prompt_lengths` are its
    prompt (none, without); lengths beyond 0..L are taken as the nearest of these.  Tokens and
    bias ids outside 0..V-1 count nowhere.  Penalties and temperature: a number, or [B] for each
    row.  bias: [V] or [B, V], any of the three types.  bias_ids: [K] or [B, K] with float32
    bias_values of that shape; ids that repeat add up, in their order.  mask: bool [V] or [B, V],
    True where allowed, or int32 [ceil(V / 32)] or [B, ceil(V / 32)] with entry v in bit v % 32 of
    word v // 32.

    Returns a tensor of the logits' type, or of `dtype` float32, or `out`, which may be `logits` and
    else shares no memory with them or another argument.
    There is no gradient."""
    return _native.lm().process_logits(logits, tokens, lengths, prompt_lengths, repetition_penalty, presence_penalty,
                                       frequency_penalty, bias, bias_ids, bias_values, temperature, mask, out, dtype)
