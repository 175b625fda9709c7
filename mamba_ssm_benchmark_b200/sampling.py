"""The next token of every sequence from its logits and a given uniform number, on sm_100a.

Of w = exp((logits - max) / temperature), in this order:
  * the ``top_k`` largest are kept;
  * of these, largest first, as many as it takes for their sum to reach ``top_p`` of all of theirs;
  * of these what is at least ``min_p`` (a share of the largest weight, which is 1).
The token is the first, by index, where the running sum of the kept weights passes ``uniforms`` times their sum.  Equal
logits rank by index, the lowest first.  Sums are exact whole numbers (units of 2^-42 of the largest weight), so a token
depends neither on how a row is split over the GPU nor on the batch around it.
"""

from . import _native as nat


def sample_tokens(logits, uniforms, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """One token per row: (B,) int64.

    logits: (B, V) float32 or bfloat16, V at most 2^20, unit stride along V (other layouts are copied); uniforms: (B,)
    float32 in [0, 1).  temperature (0: the largest logit), top_k (None or 0: all), top_p (None or 1: all) and min_p
    (None or 0: all) are numbers, or (B,) tensors with a setting for every row.  A row with a NaN, without a logit above
    -inf or with a NaN temperature gives -1.  Not differentiable."""
    return nat.glue().sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p)
