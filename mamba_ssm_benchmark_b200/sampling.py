"""The next token of every sequence from its logits and a given uniform number, on sm_100a.

Of w = exp((logits - max) / temperature), in this order:
  * the ``top_k`` largest are kept;
  * of these, largest first, as many as it takes for their sum to reach ``top_p`` of all of theirs;
  * of these what is at least ``min_p`` (a share of the largest weight, which is 1).
The token is the first, by index, where the running sum of the kept weights passes ``uniforms`` times their sum.  Equal
logits rank by index, the lowest first.  Sums are exact whole numbers (units of 2^-42 of the largest weight), so a token
depends neither on how a row is split over the GPU nor on the batch around it.
"""

import torch

from . import _native as nat
from .norm import _dense

MAX_VOCAB = 1 << 20


def _setting(name, value, B, dev, default, lo, hi, dtype=torch.float64):
    """(tensor or None, number): settings by row go to the kernel as they are."""
    if value is None:
        return None, default
    if isinstance(value, torch.Tensor):
        if value.shape != (B,):
            raise ValueError(f"{name} must be a number or a ({B},) tensor, got {tuple(value.shape)}")
        if value.device != dev:
            raise ValueError("all tensors must be on one device")
        return value.to(dtype).contiguous(), default
    value = int(value) if dtype == torch.int64 else float(value)
    if not lo <= value <= hi:
        raise ValueError(f"{name} must be in {lo} .. {hi}, got {value}")
    return None, value


def sample_tokens(logits, uniforms, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """One token per row: (B,) int64.

    logits: (B, V) float32 or bfloat16, V at most 2^20, unit stride along V (other layouts are copied); uniforms: (B,)
    float32 in [0, 1).  temperature (0: the largest logit), top_k (None or 0: all), top_p (None or 1: all) and min_p
    (None or 0: all) are numbers, or (B,) tensors with a setting for every row.  A row with a NaN, without a logit above
    -inf or with a NaN temperature gives -1.  Not differentiable."""
    if logits.dim() != 2 or logits.numel() == 0:
        raise ValueError(f"logits must be (B, V) with no empty axis, got {tuple(logits.shape)}")
    B, V = logits.shape
    if V > MAX_VOCAB:
        raise ValueError(f"the vocabulary must be at most {MAX_VOCAB}, got {V}")
    if uniforms.shape != (B,):
        raise ValueError(f"uniforms must be ({B},), got {tuple(uniforms.shape)}")
    if logits.dtype == torch.float64 or uniforms.dtype != torch.float32:
        raise TypeError(f"logits must be float32 or bfloat16 and uniforms float32, got {logits.dtype} and {uniforms.dtype}")
    dev = logits.device
    temperature, temperature0 = _setting("temperature", temperature, B, dev, 1.0, 0.0, float("inf"))
    top_k, top_k0 = _setting("top_k", top_k, B, dev, 0, 0, 1 << 62, torch.int64)
    top_p, top_p0 = _setting("top_p", top_p, B, dev, 1.0, 0.0, 1.0)
    min_p, min_p0 = _setting("min_p", min_p, B, dev, 0.0, 0.0, 1.0)
    if not logits.is_cuda:
        raise RuntimeError("the sm_100a sampling needs CUDA tensors (this package has no CPU path)")
    if uniforms.device != dev:
        raise ValueError("all tensors must be on one device")
    logits = _dense(logits.detach() if logits.dtype in nat.DTYPES else logits.detach().to(torch.float32))
    return nat.glue().sample_tokens(logits, uniforms.detach().contiguous(), temperature, temperature0, top_k, top_k0, top_p,
                                    top_p0, min_p, min_p0)
