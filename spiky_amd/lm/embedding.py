"""The lookup of token embeddings, with scaling and the gradient of the table."""
import torch

from .. import _native


def embed_tokens(tokens, weight, scale=1.0, dtype=None):
    """scale * weight[tokens], of shape [*tokens.shape, E]; zeros for tokens outside 0..V-1, such as
    the -1 of a padded batch.

    tokens: int32 or int64 on a HIP device, any shape.  weight: [V, E], float32, bfloat16 or float16,
    rows at any distance.  The result has the weight's type, or `dtype`: float32, or any of the three
    beside a float32 weight.  scale: a number, finite in 32 bits; each product is rounded to 32 bits and
    then to the result's type.

    The gradient of the weight is dense: scale times the sum of the output's gradient over a token's
    positions, zeros for tokens that do not occur.  Sums are 32-bit, over the positions sorted by token
    and in an order that the tokens alone decide, and are rounded once, to the weight's type.  So equal
    calls have equal gradients.  There are no forward-mode derivatives and no gradients of gradients."""
    return _native.lm().embed_tokens(tokens, weight, scale, dtype)


class TokenEmbedding(torch.nn.Module):
    """A trained table of token embeddings: embed_tokens with `weight` [num_embeddings, embedding_dim],
    from a normal distribution, and `scale`.  Its state dict is that of nn.Embedding."""

    def __init__(self, num_embeddings, embedding_dim, scale=1.0, device=None, dtype=None):
        super().__init__()
        self.num_embeddings, self.embedding_dim, self.scale = num_embeddings, embedding_dim, float(scale)
        self.weight = torch.nn.Parameter(torch.empty(num_embeddings, embedding_dim, device=device, dtype=dtype))
        torch.nn.init.normal_(self.weight)

    def forward(self, tokens):
        return embed_tokens(tokens, self.weight, self.scale)

    def extra_repr(self):
        return f"{self.num_embeddings}, {self.embedding_dim}, scale={self.scale}"
