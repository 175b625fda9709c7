"""Plain restatements of the gated delta rule and of the channels-last group norm, in the type of their
inputs (the tests pass float64), by their definitions: position by position, and differentiable by autograd."""

import torch


def gated_delta_rule(q, k, v, g, beta, h0=None, scale=None):
    """(o, last): S <- e^g S + beta k (v - e^g S^T k)^T, o = scale S^T q, over positions.
    q, k (B, L, Hk, dk); v (B, L, Hv, dv); g, beta (B, L, Hv); h0 (B, Hv, dk, dv) or None."""
    B, L, Hv, dv = v.shape
    Hk, dk = q.shape[2:]
    scale = dk ** -0.5 if scale is None else scale
    q, k = (t.repeat_interleave(Hv // Hk, dim=2) for t in (q, k))
    S = torch.zeros(B, Hv, dk, dv, dtype=v.dtype, device=v.device) if h0 is None else h0
    out = []
    for i in range(L):
        S = S * torch.exp(g[:, i])[..., None, None]
        miss = v[:, i] - torch.einsum("bhkv,bhk->bhv", S, k[:, i])
        S = S + torch.einsum("bhk,bhv->bhkv", k[:, i], beta[:, i][..., None] * miss)
        out.append(scale * torch.einsum("bhkv,bhk->bhv", S, q[:, i]))
    return torch.stack(out, dim=1), S


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, silu=False, z=None, center=True):
    """silu?(norm(x) weight + bias) silu(z), x (samples, ..., C), statistics over all but the sample axis
    and over the channels of a group."""
    xs = x.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    mean = xs.mean(dim=(1, 3), keepdim=True) if center else torch.zeros_like(xs[:, :1, :, :1])
    var = (xs - mean).square().mean(dim=(1, 3), keepdim=True)
    y = ((xs - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    y = y if weight is None else y * weight
    y = y if bias is None else y + bias
    y = y * torch.sigmoid(y) if silu else y
    return y if z is None else y * (z * torch.sigmoid(z))
