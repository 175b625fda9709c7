"""The gated delta rule on sm_100a: chunked forward and backward, and the one-token state update.

Per value head, with a matrix state S (dk, dv):

    S_t = exp(g_t) S_{t-1} + beta_t k_t (v_t - exp(g_t) S_{t-1}^T k_t)^T,    o_t = scale S_t^T q_t

``gated_delta_rule`` takes a sequence and is differentiable; ``gated_delta_state_update`` takes one token
and updates the state in place (decoding).  They stand next to ``selective_scan`` and
``selective_state_update``: same order of results, same handling of types and errors.  State, sums and
gradients of states are float32; q, k, v and o are read and written in float32 or bfloat16 when q, k and
v share the type, any other mix is promoted to float32.
"""

import torch

from . import _native as nat

MAX_KEY_WIDTH = 128


def _check(q, k, v, g, beta, state, state_name):
    """Shapes of (B, L, heads, width) arguments; returns (B, L, Hk, Hv, dk, dv)."""
    if q.dim() != 4 or k.shape != q.shape:
        raise ValueError(f"q and k must be (B, L, Hk, dk) of equal shape, got {tuple(q.shape)} / {tuple(k.shape)}")
    B, L, Hk, dk = q.shape
    if v.dim() != 4 or tuple(v.shape[:2]) != (B, L):
        raise ValueError(f"v must be (B, L, Hv, dv) with B={B}, L={L}, got {tuple(v.shape)}")
    Hv, dv = v.shape[2:]
    if min(B, L, Hk, Hv, dk, dv) < 1:
        raise ValueError(f"q and v must have no empty axis, got {tuple(q.shape)} / {tuple(v.shape)}")
    if Hv % Hk != 0:
        raise ValueError(f"the {Hv} value heads must be a multiple of the {Hk} key heads")
    if dk > MAX_KEY_WIDTH:
        raise ValueError(f"the key width must be at most {MAX_KEY_WIDTH} for the sm_100a kernels, got {dk}")
    for name, t in (("g", g), ("beta", beta)):
        if tuple(t.shape) != (B, L, Hv):
            raise ValueError(f"{name} must be (B, L, Hv) = {(B, L, Hv)}, got {tuple(t.shape)}")
    if state is not None and tuple(state.shape) != (B, Hv, dk, dv):
        raise ValueError(f"{state_name} must be (B, Hv, dk, dv) = {(B, Hv, dk, dv)}, got {tuple(state.shape)}")
    tensors = [t for t in (q, k, v, g, beta, state) if t is not None]
    if any(t.dtype == torch.float64 for t in tensors):
        raise TypeError("float64 is not supported by the sm_100a kernels; use float32 or bfloat16")
    if not q.is_cuda:
        raise RuntimeError("the sm_100a gated delta rule needs CUDA tensors (this package has no CPU path)")
    if any(t.device != q.device for t in tensors):
        raise ValueError("all tensors must be on one device")
    return B, L, Hk, Hv, dk, dv


def _act(t, dtype):
    t = t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _common_dtype(*ts):
    return ts[0].dtype if ts[0].dtype in nat.DTYPES and all(t.dtype == ts[0].dtype for t in ts) else torch.float32


def _empty(shape, dtype, dev):
    return torch.empty(shape, dtype=dtype, device=dev)


def _forward(q, k, v, g, beta, h0, scale, save):
    B, L, Hk, dk = q.shape
    Hv, dv = v.shape[2:]
    dims, dev = (B, L, Hk, Hv, dk, dv), q.device
    o = _empty((B, L, Hv, dv), q.dtype, dev)
    last = _empty((B, Hv, dk, dv), torch.float32, dev)
    saved = _empty(nat.gated_delta_saved_bytes(dims, q.dtype), torch.uint8, dev) if save else None
    wsb = nat.gated_delta_workspace_bytes(dims, q.dtype, False)
    ws = _empty(wsb, torch.uint8, dev)
    with torch.cuda.device(dev):
        rc = nat.lib().ssm_gated_delta_fwd(*dims, nat.heads4(q), nat.heads4(k), nat.heads4(v), nat.view3(g),
                                           nat.view3(beta), nat.ptr(h0), scale, nat.heads4(o), nat.ptr(last),
                                           nat.ptr(saved), ws.data_ptr(), wsb, nat.stream_of(dev))
    nat.check(rc, "ssm_gated_delta_fwd")
    return o, last, saved


class GatedDeltaFn(torch.autograd.Function):
    """(o, last) of the gated delta rule.  Keeps the state entering every 64 positions and the chunks'
    corrected values for the backward."""

    @staticmethod
    def forward(ctx, q, k, v, g, beta, h0, scale):
        o, last, saved = _forward(q, k, v, g, beta, h0, scale, True)
        ctx.save_for_backward(q, k, v, g, beta, h0, saved)
        ctx.scale = scale
        return o, last

    @staticmethod
    def backward(ctx, do, dlast):
        q, k, v, g, beta, h0, saved = ctx.saved_tensors
        B, L, Hk, dk = q.shape
        Hv, dv = v.shape[2:]
        dims, dev = (B, L, Hk, Hv, dk, dv), q.device
        do = _act(do, q.dtype)
        dlast = None if dlast is None else dlast.to(torch.float32).contiguous()
        dq, dk_, dv_ = (_empty(t.shape, q.dtype, dev) for t in (q, k, v))
        dg, dbeta = (_empty((B, L, Hv), torch.float32, dev) for _ in range(2))
        dh0 = None if h0 is None else _empty(h0.shape, torch.float32, dev)
        wsb = nat.gated_delta_workspace_bytes(dims, q.dtype, True)
        ws = _empty(wsb, torch.uint8, dev)
        with torch.cuda.device(dev):
            rc = nat.lib().ssm_gated_delta_bwd(*dims, nat.heads4(q), nat.heads4(k), nat.heads4(v), nat.view3(g),
                                               nat.view3(beta), ctx.scale, saved.data_ptr(), nat.heads4(do),
                                               nat.ptr(dlast), nat.heads4(dq), nat.heads4(dk_), nat.heads4(dv_),
                                               nat.ptr(dg), nat.ptr(dbeta), nat.ptr(dh0), ws.data_ptr(), wsb,
                                               nat.stream_of(dev))
        nat.check(rc, "ssm_gated_delta_bwd")
        return dq, dk_, dv_, dg, dbeta, dh0, None


def gated_delta_rule(q, k, v, g, beta, h0=None, scale=None):
    """Returns (o, last): o (B, L, Hv, dv) in v's dtype, last (B, Hv, dk, dv) float32.

    q, k: (B, L, Hk, dk); v: (B, L, Hv, dv), Hv a multiple of Hk (key head h // (Hv // Hk) serves value
    head h); g: (B, L, Hv), the log of the decay (at most 0; -inf resets the state); beta: (B, L, Hv), the
    step of the correction; h0: (B, Hv, dk, dv) or None (zeros); scale: of o, default dk ** -0.5.
    Any strides.  Differentiable with respect to all six tensors."""
    _check(q, k, v, g, beta, h0, "h0")
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    out_dtype, ct = v.dtype, _common_dtype(q, k, v)
    q, k, v = (_act(t, ct) for t in (q, k, v))
    g, beta = (_act(t, torch.float32) for t in (g, beta))
    h0 = None if h0 is None else h0.to(torch.float32).contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, h0)):
        o, last = GatedDeltaFn.apply(q, k, v, g, beta, h0, scale)
    else:
        o, last, _ = _forward(q, k, v, g, beta, h0, scale, False)
    return o.to(out_dtype), last


def gated_delta_state_update(state, q, k, v, g, beta, scale=None, out=None):
    """One token; ``state`` (B, Hv, dk, dv) float32 is updated in place.  q, k: (B, Hk, dk); v: (B, Hv, dv);
    g, beta: (B, Hv).  Returns o (B, Hv, dv) in v's dtype (``out`` if given: that shape, q, k and v's common
    type).  No synchronisation; capturable in a CUDA graph."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3 or g.dim() != 2 or beta.dim() != 2:
        raise ValueError(f"q, k and v must be (B, H, width) and g, beta (B, H), got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}, {tuple(g.shape)}, {tuple(beta.shape)}")
    q, k, v, g, beta = (t.unsqueeze(1) for t in (q, k, v, g, beta))
    B, _, Hk, Hv, dk, dv = _check(q, k, v, g, beta, state, "state")
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 (B, Hv, dk, dv) tensor")
    scale = float(dk ** -0.5 if scale is None else scale)
    out_dtype, ct = v.dtype, _common_dtype(q, k, v)
    q, k, v = (_act(t, ct) for t in (q, k, v))
    g, beta = (_act(t, torch.float32) for t in (g, beta))
    if out is None:
        o = _empty((B, Hv, dv), ct, state.device)
    else:
        if tuple(out.shape) != (B, Hv, dv) or out.dtype != ct or out.device != state.device or \
                (out.stride(-1) != 1 and dv != 1):
            raise ValueError(f"out must be a ({B}, {Hv}, {dv}) {ct} tensor with unit inner stride")
        o = out
    with torch.cuda.device(state.device):
        rc = nat.lib().ssm_gated_delta_state_update(B, Hk, Hv, dk, dv, state.data_ptr(), nat.heads4(q), nat.heads4(k),
                                                    nat.heads4(v), nat.view3(g), nat.view3(beta), scale,
                                                    nat.heads4(o.unsqueeze(1)), nat.stream_of(state.device))
    nat.check(rc, "ssm_gated_delta_state_update")
    return o if out is not None else o.to(out_dtype)
