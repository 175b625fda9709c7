"""Rows of a table by token, scaled, and the table's gradient, on sm_100a.

    y[t] = scale weight[idx[t]],   dweight[v] = scale * (sum of dy[t] over the t with idx[t] = v)

The gradient sums a token's places in their order, in float32 and above: results are reproducible.
"""

import torch

from . import _native as nat


def embedding(idx, weight, scale=1.0):
    """scale * weight[idx], shaped (*idx.shape, C) and in weight's dtype.

    idx: int64 or int32 token ids of any shape; weight: (V, C) float32 or bfloat16, unit stride along C (other layouts
    are copied); scale: a number.  Differentiable with respect to weight.  An id outside 0 .. V-1 gives a row of NaN and no
    gradient, and sets a bit of the device error word."""
    if weight.dim() != 2 or weight.numel() == 0:
        raise ValueError(f"weight must be (vocabulary, channels) with no empty axis, got {tuple(weight.shape)}")
    if idx.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"idx must be int64 or int32, got {idx.dtype}")
    if idx.numel() == 0:
        raise ValueError(f"idx must have no empty axis, got {tuple(idx.shape)}")
    if weight.dtype not in nat.DTYPES:
        raise TypeError(f"weight must be float32 or bfloat16, got {weight.dtype}")
    if not weight.is_cuda:
        raise RuntimeError("the sm_100a embedding needs CUDA tensors (this package has no CPU path)")
    if idx.device != weight.device:
        raise ValueError("all tensors must be on one device")
    C = weight.shape[1]
    if weight.stride(1) != 1 and C != 1:
        weight = weight.contiguous()
    y = nat.glue().embedding(idx.reshape(-1).contiguous(), weight, float(scale))
    return y if idx.dim() == 1 else y.reshape(*idx.shape, C)
