"""Group norm over channels-last tensors, with an activation and a gate, on sm_100a.

    n = (x - mean) / sqrt(var + eps),   y = act(n weight + bias) * silu(z)

x is (samples, ..., C): the statistics of a sample and group run over every position between the
first and the last axis and over the group's C / groups channels.  A two-dimensional x, (tokens,
heads * width) with ``groups = heads``, is the norm of every head of every token; with
``center=False`` (no mean is subtracted) and ``z`` it is the gated norm behind a mixer's heads,
with ``center=False`` and a constant weight the length normalisation of queries and keys.

``rms_norm`` is the norm of a residual stream: it adds the residual, keeps the sum and norms it, in one pass; ``rms_norm_fp8``
gives the result in 8 bits with a scale for every row, as ``linear_fp8`` takes it, and ``quantize_fp8`` only that.

Statistics and sums are float32; x, z and their gradients are read and written in float32 or
bfloat16 (a mix is promoted to float32 first); weight, bias and their gradients are float32 inside.
Parameter gradients are summed in a fixed order: results are reproducible.
"""

import torch

from . import _native as nat


def _dense(t):
    """A layout that the kernels read: unit stride along the channels."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(t, name, C):
    if t is None:
        return None
    if t.dim() != 1 or t.shape[0] != C:
        raise ValueError(f"{name} must be ({C},), got {tuple(t.shape)}")
    return (t if t.dtype == torch.float32 else t.to(torch.float32)).contiguous()


def _flat(t, dtype):
    """(samples, C) or (samples, positions, C) in the kernels' type; one position is the two-dimensional case."""
    if t is None:
        return None
    if t.dtype != dtype:
        t = t.to(dtype)
    if t.dim() > 2:
        t = t.reshape(t.shape[0], -1, t.shape[-1])
        if t.shape[1] == 1:
            t = t[:, 0]
    return _dense(t)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, z=None, center=True):
    """y = act(group_norm(x) * weight + bias) * silu(z), shaped like x and in x's dtype.

    x: (samples, C) or (samples, ..., C), float32 or bfloat16, unit stride along C (other layouts are
    copied); groups divides C; weight, bias: (C) or None; activation: None or "silu"; z: the gate,
    shaped like x, or None; center: subtract the mean (False: root-mean-square norm).
    Differentiable with respect to x, weight, bias and z."""
    if x.dim() < 2:
        raise ValueError(f"x must be (samples, ..., C), got {tuple(x.shape)}")
    C, in_dtype, shape = x.shape[-1], x.dtype, x.shape
    if x.numel() == 0:
        raise ValueError(f"x must have no empty axis, got {tuple(shape)}")
    if not isinstance(groups, int) or groups < 1 or C % groups != 0:
        raise ValueError(f"groups must divide C={C}, got {groups!r}")
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    if z is not None and z.shape != shape:
        raise ValueError(f"z must be shaped like x {tuple(shape)}, got {tuple(z.shape)}")
    eps, center = float(eps), bool(center)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps!r}")
    if in_dtype == torch.float64 or (z is not None and z.dtype == torch.float64):
        raise TypeError("float64 is not supported by the sm_100a kernels; use float32 or bfloat16")
    if not x.is_cuda:
        raise RuntimeError("the sm_100a group norm needs CUDA tensors (this package has no CPU path)")
    dev = x.device
    for t in (weight, bias, z):
        if t is not None and t.device != dev:
            raise ValueError("all tensors must be on one device")
    dtype = in_dtype if in_dtype in nat.DTYPES and (z is None or z.dtype == in_dtype) else torch.float32
    x, z = _flat(x, dtype), _flat(z, dtype)
    weight, bias = _param(weight, "weight", C), _param(bias, "bias", C)
    y = nat.glue().group_norm(x, groups, weight, bias, z, eps, activation == "silu", center)
    if y.shape != shape:
        y = y.reshape(shape)
    return y if in_dtype == dtype else y.to(in_dtype)


def rms_norm(x, weight=None, residual=None, eps=1e-5):
    """total = x + residual, y = total / sqrt(mean(total^2) + eps) * weight: y without a residual, (y, total) with one.

    x: (..., C), float32 or bfloat16, unit stride along C (other layouts are copied); residual: shaped like x, or None;
    weight: (C) or None.  y is in x's dtype, total in the wider of x's and the residual's; what is normed is total as it is
    kept.  Differentiable with respect to x, weight and residual, whose gradients are one tensor where x and residual
    have one dtype (as those of x + residual are)."""
    out = nat.glue().rms_norm(x, weight, residual, eps, False)
    return out[0] if residual is None else tuple(out)


def rms_norm_fp8(x, weight=None, residual=None, eps=1e-5):
    """``rms_norm`` with y in 8 bits: (y8, scale) or, with a residual, (y8, scale, total).

    y8: float8_e4m3fn, shaped like x, rows that start at multiples of 16 bytes; scale: (...) float32, the row's largest |y|
    (at least 1e-30) / 448; y is about y8 * scale.  No gradient."""
    return tuple(nat.glue().rms_norm_fp8(x, weight, residual, eps, True))


def quantize_fp8(x):
    """x (..., C) in 8 bits with a scale for every row: (x8, scale) as ``rms_norm_fp8`` gives them.  No gradient."""
    return tuple(nat.glue().rms_norm_fp8(x, None, None, 0.0, False))
