"""Group norm over channels-last tensors, with an activation and a gate, on sm_100a.

    n = (x - mean) / sqrt(var + eps),   y = act(n weight + bias) * silu(z)

x is (samples, ..., C): the statistics of a sample and group run over every position between the
first and the last axis and over the group's C / groups channels.  A two-dimensional x, (tokens,
heads * width) with ``groups = heads``, is the norm of every head of every token; with
``center=False`` (no mean is subtracted) and ``z`` it is the gated norm behind a mixer's heads,
with ``center=False`` and a constant weight the length normalisation of queries and keys.

Statistics and sums are float32; x, z and their gradients are read and written in float32 or
bfloat16 (a mix is promoted to float32 first); weight, bias and their gradients are float32 inside.
Parameter gradients are summed in a fixed order: results are reproducible.
"""

import torch

from . import _native as nat


def _view(t, positions):
    """ssm_view of a (samples, positions, C) tensor; a 2-D one has a single position."""
    return nat.view2(t) if positions == 1 else nat.view3(t)


def _workspace(shape, groups, backward, dev):
    n = nat.norm_workspace_bytes(*shape, groups, backward)
    return torch.empty(n, dtype=torch.uint8, device=dev), n


def _forward(x, weight, bias, z, groups, eps, silu, center, want_stats):
    (N, P, C), dev = _dims(x), x.device
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats = torch.empty((N, groups, 2), dtype=torch.float32, device=dev) if want_stats else None
    ws, wsb = _workspace((N, P, C), groups, False, dev)
    with torch.cuda.device(dev):
        rc = nat.lib().ssm_group_norm_fwd(N, P, C, groups, _view(x, P), nat.ptr(weight), nat.ptr(bias), eps,
                                          int(center), int(silu), _view(z, P), _view(y, P), nat.ptr(stats),
                                          ws.data_ptr(), wsb, nat.stream_of(dev))
    nat.check(rc, "ssm_group_norm_fwd")
    return y, stats


def _dims(x):
    return (x.shape[0], 1, x.shape[1]) if x.dim() == 2 else tuple(x.shape)


class GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, z, groups, eps, silu, center):
        y, stats = _forward(x, weight, bias, z, groups, eps, silu, center, True)
        ctx.save_for_backward(x, weight, bias, z, stats)
        ctx.args = groups, silu, center
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, z, stats = ctx.saved_tensors
        groups, silu, center = ctx.args
        (N, P, C), dev = _dims(x), x.device
        dy = _dense(dy.to(x.dtype))
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dz = torch.empty(x.shape, dtype=x.dtype, device=dev) if z is not None else None
        dw = torch.empty(C, dtype=torch.float32, device=dev) if weight is not None else None
        db = torch.empty(C, dtype=torch.float32, device=dev) if bias is not None else None
        ws, wsb = _workspace((N, P, C), groups, True, dev)
        with torch.cuda.device(dev):
            rc = nat.lib().ssm_group_norm_bwd(N, P, C, groups, _view(x, P), nat.ptr(weight), nat.ptr(bias), int(center),
                                              int(silu), _view(z, P), nat.ptr(stats), _view(dy, P), _view(dx, P),
                                              nat.ptr(dw), nat.ptr(db), _view(dz, P), ws.data_ptr(), wsb,
                                              nat.stream_of(dev))
        nat.check(rc, "ssm_group_norm_bwd")
        return dx, dw, db, dz, None, None, None, None


def _dense(t):
    """A layout the kernels read: unit stride along the channels, no negative or broadcast trouble."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _param(t, name, C):
    if t is None:
        return None
    if tuple(t.shape) != (C,):
        raise ValueError(f"{name} must be ({C},), got {tuple(t.shape)}")
    return t.to(torch.float32).contiguous()


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, z=None, center=True):
    """y = act(group_norm(x) * weight + bias) * silu(z), shaped like x and in x's dtype.

    x: (samples, C) or (samples, ..., C), float32 or bfloat16, unit stride along C (other layouts are
    copied); groups divides C; weight, bias: (C) or None; activation: None or "silu"; z: the gate,
    shaped like x, or None; center: subtract the mean (False: root-mean-square norm).
    Differentiable with respect to x, weight, bias and z."""
    if x.dim() < 2:
        raise ValueError(f"x must be (samples, ..., C), got {tuple(x.shape)}")
    C = x.shape[-1]
    if min(x.shape) < 1:
        raise ValueError(f"x must have no empty axis, got {tuple(x.shape)}")
    if not isinstance(groups, int) or groups < 1 or C % groups != 0:
        raise ValueError(f"groups must divide C={C}, got {groups!r}")
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be 'silu' or None, got {activation!r}")
    if z is not None and z.shape != x.shape:
        raise ValueError(f"z must be shaped like x {tuple(x.shape)}, got {tuple(z.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps!r}")
    acts = [t for t in (x, z) if t is not None]
    if any(t.dtype == torch.float64 for t in acts):
        raise TypeError("float64 is not supported by the sm_100a kernels; use float32 or bfloat16")
    if not x.is_cuda:
        raise RuntimeError("the sm_100a group norm needs CUDA tensors (this package has no CPU path)")
    if any(t is not None and t.device != x.device for t in (weight, bias, z)):
        raise ValueError("all tensors must be on one device")
    ct = x.dtype if x.dtype in nat.DTYPES and all(t.dtype == x.dtype for t in acts) else torch.float32
    weight, bias = _param(weight, "weight", C), _param(bias, "bias", C)

    def flat(t):
        if t is None:
            return None
        t = t.to(ct)
        if t.dim() > 2:      # (samples, positions, C); one position is the two-dimensional case
            t = t.reshape(t.shape[0], -1, C)
            t = t[:, 0] if t.shape[1] == 1 else t
        return _dense(t)

    xf, zf = flat(x), flat(z)
    tensors = [t for t in (xf, weight, bias, zf) if t is not None]
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        y = GroupNormFn.apply(xf, weight, bias, zf, groups, float(eps), activation == "silu", bool(center))
    else:
        y, _ = _forward(xf, weight, bias, zf, groups, float(eps), activation == "silu", bool(center), False)
    return y.reshape(x.shape).to(x.dtype)
