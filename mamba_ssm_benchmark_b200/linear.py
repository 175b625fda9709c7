"""Products of 8-bit rows with bias, activation and residual in one kernel on the sm_100a tensor cores.

    y = act(x_scale * w_scale * (x8 @ weight8^T) + bias) + residual

x8 and its scales come from ``rms_norm_fp8`` or ``quantize_fp8``, weight8 and its scales from ``quantize_fp8`` of a weight, once.
For answering, not for training: 8-bit weights have no gradient.
"""

import torch
import torch.nn as nn

from . import _native as nat
from .norm import quantize_fp8

E4M3 = torch.float8_e4m3fn


def linear_fp8(x8, x_scale, weight8, weight_scale, bias=None, activation=None, residual=None, dtype=None):
    """y: (..., N) in ``dtype`` (float32 or bfloat16; default: the residual's, else bfloat16).

    x8: (..., K) and weight8: (N, K) in float8_e4m3fn, rows that start at multiples of 16 bytes as ``quantize_fp8`` lays them
    out (others are copied); x_scale: (...), weight_scale: (N) float32; bias: (N) or None; activation: None or "silu";
    residual: shaped like y and in its dtype, or None.  Sums are float32."""
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    return nat.glue().linear_fp8(x8, x_scale, weight8, weight_scale, bias, activation is not None, residual, dtype)


class Fp8Linear(nn.Module):
    """A linear map without bias whose weight is held in 8 bits with a scale for every row, made from ``weight`` (N, K) on the
    GPU.  Its buffers move with a model and are not cast with it."""

    def __init__(self, weight):
        super().__init__()
        w8, scale = quantize_fp8(weight.detach())
        self.out_features, self.in_features = weight.shape
        self.dtype = weight.dtype if weight.dtype in nat.DTYPES else torch.float32
        rows = torch.zeros(w8.shape[0], -(-w8.shape[1] // 16) * 16, dtype=torch.uint8, device=w8.device)
        rows[:, :w8.shape[1]] = w8.view(torch.uint8)
        # bytes, which a cast of the model leaves alone; rows of whole 16 bytes
        self.register_buffer("weight8", rows)
        self.register_buffer("weight_scale", scale)

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, x, residual=None, dtype=None):
        """x: (..., K) values, which are put into 8 bits row by row, or the pair (x8, scale).  The result is in ``dtype``; by
        default in the residual's dtype, x's, or the weight's before it was put into 8 bits."""
        if dtype is None:
            dtype = residual.dtype if residual is not None else self.dtype if isinstance(x, tuple) else x.dtype
        x8, scale = x if isinstance(x, tuple) else quantize_fp8(x)
        w8 = self.weight8.view(E4M3)
        return linear_fp8(x8, scale, w8 if w8.shape[1] == self.in_features else w8[:, :self.in_features], self.weight_scale,
                          residual=residual, dtype=dtype)
