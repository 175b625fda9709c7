"""Rows of a table by token, scaled, and the table's gradient, on sm_100a.

    y[t] = scale weight[idx[t]],   dweight[v] = scale * (sum of dy[t] over the t with idx[t] = v)

The gradient sums a token's places in their order, in float32 and above: results are reproducible.
"""

from . import _native as nat


def embedding(idx, weight, scale=1.0):
    """scale * weight[idx], shaped (*idx.shape, C) and in weight's dtype.

    idx: int64 or int32 token ids of any shape; weight: (V, C) float32 or bfloat16, unit stride along C (other layouts
    are copied); scale: a number.  Differentiable with respect to weight.  An id outside 0 .. V-1 gives a row of NaN and no
    gradient, and sets a bit of the device error word."""
    return nat.glue().embedding(idx, weight, scale, False)
