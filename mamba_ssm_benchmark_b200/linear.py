"""Products of 8-bit rows with bias, activation and residual in one kernel on the sm_100a tensor cores.

    y = act(x_scale * w_scale * (x8 @ weight8^T) + bias) + residual

x8 and its scales come from ``rms_norm_fp8`` or ``quantize_fp8``, weight8 and its scales from ``quantize_fp8`` of a weight, once.
For answering, not for training: 8-bit weights have no gradient.
"""

import torch
import torch.nn as nn

from . import _native as nat
from .norm import _dense, quantize_fp8

E4M3 = torch.float8_e4m3fn


def linear_fp8(x8, x_scale, weight8, weight_scale, bias=None, activation=None, residual=None, dtype=None):
    """y: (..., N) in ``dtype`` (float32 or bfloat16; default: the residual's, else bfloat16).

    x8: (..., K) and weight8: (N, K) in float8_e4m3fn, rows that start at multiples of 16 bytes as ``quantize_fp8`` lays them
    out (others are copied); x_scale: (...), weight_scale: (N) float32; bias: (N) or None; activation: None or "silu";
    residual: shaped like y and in its dtype, or None.  Sums are float32."""
    if x8.dtype != E4M3 or weight8.dtype != E4M3:
        raise TypeError(f"x8 and weight8 must be float8_e4m3fn, got {x8.dtype} and {weight8.dtype}")
    if weight8.dim() != 2 or x8.dim() < 1 or x8.numel() == 0 or weight8.numel() == 0:
        raise ValueError(f"x8 must be (..., K) and weight8 (N, K) with no empty axis, got {tuple(x8.shape)} and {tuple(weight8.shape)}")
    N, K = weight8.shape
    shape = x8.shape[:-1]
    if x8.shape[-1] != K:
        raise ValueError(f"x8 must have weight8's {K} columns, got {tuple(x8.shape)}")
    if x_scale.shape != shape or weight_scale.shape != (N,):
        raise ValueError(f"the scales must be {tuple(shape)} and ({N},), got {tuple(x_scale.shape)} and {tuple(weight_scale.shape)}")
    if x_scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
        raise TypeError("the scales must be float32")
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias must be ({N},), got {tuple(bias.shape)}")
    if dtype is None:
        dtype = residual.dtype if residual is not None else torch.bfloat16
    if dtype not in nat.DTYPES:
        raise TypeError(f"dtype must be float32 or bfloat16, got {dtype}")
    if residual is not None and (residual.shape != (*shape, N) or residual.dtype != dtype):
        raise ValueError(f"residual must be {(*shape, N)} in {dtype}, got {tuple(residual.shape)} in {residual.dtype}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x_scale, weight_scale, bias, residual)):
        raise RuntimeError("linear_fp8 has no gradient: call it under torch.no_grad()")
    if not x8.is_cuda:
        raise RuntimeError("the sm_100a products need CUDA tensors (this package has no CPU path)")
    dev = x8.device
    for t in (x_scale, weight8, weight_scale, bias, residual):
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on one device")
    if bias is not None:
        bias = bias.to(torch.float32).contiguous()
    if residual is not None:
        residual = _dense(residual.reshape(-1, N))
    y = nat.glue().linear_fp8(x8.reshape(-1, K), x_scale.reshape(-1).contiguous(), weight8, weight_scale.contiguous(), bias,
                              residual, activation == "silu", dtype == torch.bfloat16)
    return y if len(shape) == 1 else y.reshape(*shape, N)


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
