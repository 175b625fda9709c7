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


def _check(q, k, v, g, beta, state, state_name, rank):
    """Checks (B, L, heads, width) arguments (rank 4) or one token's (B, heads, width) (rank 3); returns
    (B, L, Hk, Hv, dk, dv)."""
    qs, vs = q.shape, v.shape
    lead = "(B, L" if rank == 4 else "(B"
    if len(qs) != rank or k.shape != qs:
        raise ValueError(f"q and k must be {lead}, Hk, dk) of equal shape, got {tuple(qs)} / {tuple(k.shape)}")
    if len(vs) != rank or vs[:-2] != qs[:-2]:
        raise ValueError(f"v must be {lead}, Hv, dv) with {lead}) = {tuple(qs[:-2])}, got {tuple(vs)}")
    Hk, dk = qs[-2:]
    Hv, dv = vs[-2:]
    B, L = qs[0], qs[1] if rank == 4 else 1
    if q.numel() == 0 or v.numel() == 0:
        raise ValueError(f"q and v must have no empty axis, got {tuple(qs)} / {tuple(vs)}")
    if Hv % Hk != 0:
        raise ValueError(f"the {Hv} value heads must be a multiple of the {Hk} key heads")
    if dk > MAX_KEY_WIDTH:
        raise ValueError(f"the key width must be at most {MAX_KEY_WIDTH} for the sm_100a kernels, got {dk}")
    if g.shape != vs[:-1] or beta.shape != vs[:-1]:
        raise ValueError(f"g and beta must be {lead}, Hv) = {tuple(vs[:-1])}, got {tuple(g.shape)} / {tuple(beta.shape)}")
    if state is not None and state.shape != (B, Hv, dk, dv):
        raise ValueError(f"{state_name} must be (B, Hv, dk, dv) = {(B, Hv, dk, dv)}, got {tuple(state.shape)}")
    if not q.is_cuda:
        raise RuntimeError("the sm_100a gated delta rule needs CUDA tensors (this package has no CPU path)")
    dev = q.device
    for t in (q, k, v, g, beta, state):
        if t is None:
            continue
        if t.dtype == torch.float64:
            raise TypeError("float64 is not supported by the sm_100a kernels; use float32 or bfloat16")
        if t.device != dev:
            raise ValueError("all tensors must be on one device")
    return B, L, Hk, Hv, dk, dv


def _act(t, dtype):
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _common_dtype(q, k, v):
    return q.dtype if q.dtype in nat.DTYPES and k.dtype == q.dtype and v.dtype == q.dtype else torch.float32


def gated_delta_rule(q, k, v, g, beta, h0=None, scale=None):
    """Returns (o, last): o (B, L, Hv, dv) in v's dtype, last (B, Hv, dk, dv) float32.

    q, k: (B, L, Hk, dk); v: (B, L, Hv, dv), Hv a multiple of Hk (key head h // (Hv // Hk) serves value
    head h); g: (B, L, Hv), the log of the decay (at most 0; -inf resets the state); beta: (B, L, Hv), the
    step of the correction; h0: (B, Hv, dk, dv) or None (zeros); scale: of o, default dk ** -0.5.
    Any strides.  Differentiable once with respect to all six tensors.  A value that is not finite reaches no
    output before its position; gradients are defined for finite inputs."""
    _check(q, k, v, g, beta, h0, "h0", 4)
    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    out_dtype, ct = v.dtype, _common_dtype(q, k, v)
    q, k, v = _act(q, ct), _act(k, ct), _act(v, ct)
    g, beta = _act(g, torch.float32), _act(beta, torch.float32)
    if h0 is not None:
        h0 = _act(h0, torch.float32).contiguous()
    o, last = nat.glue().gated_delta(q, k, v, g, beta, h0, scale)
    return (o if out_dtype == ct else o.to(out_dtype)), last


def gated_delta_state_update(state, q, k, v, g, beta, scale=None, out=None):
    """One token; ``state`` (B, Hv, dk, dv) float32 is updated in place.  q, k: (B, Hk, dk); v: (B, Hv, dv);
    g, beta: (B, Hv).  Returns o (B, Hv, dv) in v's dtype (``out`` if given: that shape, q, k and v's common
    type).  No synchronisation; capturable in a CUDA graph."""
    B, _, _, Hv, dk, dv = _check(q, k, v, g, beta, state, "state", 3)
    if state.dtype != torch.float32 or not state.is_contiguous():
        raise ValueError("state must be a contiguous float32 (B, Hv, dk, dv) tensor")
    scale = float(dk ** -0.5 if scale is None else scale)
    out_dtype, ct = v.dtype, _common_dtype(q, k, v)
    q, k, v = _act(q, ct), _act(k, ct), _act(v, ct)
    g, beta = _act(g, torch.float32), _act(beta, torch.float32)
    if out is not None and (out.shape != (B, Hv, dv) or out.dtype != ct or out.device != state.device or
                            (out.stride(-1) != 1 and dv != 1)):
        raise ValueError(f"out must be a ({B}, {Hv}, {dv}) {ct} tensor with unit inner stride")
    o = nat.glue().gated_delta_step(state, q, k, v, g, beta, scale, out)
    return o if out is not None or out_dtype == ct else o.to(out_dtype)
