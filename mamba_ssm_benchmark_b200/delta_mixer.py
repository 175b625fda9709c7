"""A gated delta-rule mixer: the token mixer around ``gated_delta_rule``, next to ``MambaMixer``.

    q, k, v, z = in_proj(u);   q, k, v = silu(causal depthwise conv)        (causal_conv1d)
    q, k = each head scaled to length 1                                     (group_norm, uncentred)
    g = -exp(A_log) softplus(gate + dt_bias),   beta = sigmoid(gate')
    o = gated delta rule                                                    (gated_delta_rule)
    out = out_proj(norm of every head of o * silu(z))                       (group_norm with a gate)

The projections stay torch GEMMs; everything between them runs on this package's kernels.  ``forward`` has
``MambaMixer``'s three paths (training, prefill with a state, one token with a state) and its state's attributes
(``conv``, ``ssm``), so ``MambaLM(mixer="delta")``, ``generate`` and ``GraphDecoder`` work with either mixer.
"""

import math
from types import SimpleNamespace

import torch
import torch.nn as nn
import torch.nn.functional as F

from .conv import causal_conv1d
from .delta import MAX_KEY_WIDTH, gated_delta_rule, gated_delta_state_update
from .mixer import _Holder, _softplus_inverse
from .norm import group_norm


class GatedDeltaMixer(nn.Module):
    """d_model: width of the input; expand * d_model channels inside, in value heads of head_dim channels that
    share key_heads key heads (default half as many) of the same width, at most MAX_KEY_WIDTH."""

    def __init__(self, d_model, head_dim=64, key_heads=None, expand=2, d_conv=4, dt_min=1e-3, dt_max=0.1):
        super().__init__()
        if not 1 <= head_dim <= MAX_KEY_WIDTH:
            raise ValueError(f"head_dim must be 1 to {MAX_KEY_WIDTH} for the sm_100a kernels, got {head_dim}")
        self.d_inner, self.head_dim, self.d_conv = expand * d_model, head_dim, d_conv
        if self.d_inner % head_dim != 0:
            raise ValueError(f"the inner width {self.d_inner} must be a multiple of head_dim={head_dim}")
        self.heads = self.d_inner // head_dim
        self.key_heads = key_heads if key_heads is not None else max(1, self.heads // 2)
        if self.heads % self.key_heads != 0:
            raise ValueError(f"the {self.heads} value heads must be a multiple of the {self.key_heads} key heads")
        self.d_key = self.key_heads * head_dim
        self.d_conv_in = 2 * self.d_key + self.d_inner                     # q, k, v
        self.in_proj = _Holder((self.d_conv_in + self.d_inner, d_model))   # and z
        self.gate_proj = _Holder((2 * self.heads, d_model))                # decay, beta
        self.conv = _Holder((self.d_conv_in, 1, d_conv), (self.d_conv_in,))
        self.out_proj = _Holder((d_model, self.d_inner))
        self.A_log = nn.Parameter(torch.empty(self.heads))
        self.dt_bias = nn.Parameter(torch.empty(self.heads))
        self.norm_weight = nn.Parameter(torch.empty(self.d_inner))
        # x / rms(x) * head_dim^-1/2 has length 1
        self.register_buffer("unit", torch.full((2 * self.d_key,), head_dim ** -0.5), persistent=False)
        self.reset_parameters(dt_min, dt_max)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        # moved with the module but not cast with it: rounded to bf16, keys would be up to 0.2 % off length 1
        self.unit = torch.full_like(self.unit, self.head_dim ** -0.5, dtype=torch.float32)
        return self

    @torch.no_grad()
    def reset_parameters(self, dt_min=1e-3, dt_max=0.1):
        """Decay rates in [1, 16], step sizes log-uniform in [dt_min, dt_max] through softplus; projections and
        conv uniform in +-1/sqrt(fan_in)."""
        for holder in (self.in_proj, self.gate_proj, self.conv, self.out_proj):
            bound = 1.0 / math.sqrt(holder.weight[0].numel())
            holder.weight.uniform_(-bound, bound)
            if holder.bias is not None:
                holder.bias.uniform_(-bound, bound)
        self.A_log.uniform_(1.0, 16.0).log_()
        dt = torch.empty(self.heads).uniform_(math.log(dt_min), math.log(dt_max)).exp_()
        self.dt_bias.copy_(_softplus_inverse(dt))
        self.norm_weight.fill_(1.0)

    def init_state(self, batch, max_len, device, dtype=torch.float32):
        """Decode state: the last d_conv - 1 conv inputs and every value head's (key, value) matrix; its size does
        not depend on max_len."""
        del max_len
        return SimpleNamespace(conv=torch.zeros(batch, self.d_conv_in, self.d_conv - 1, device=device, dtype=dtype),
                               ssm=torch.zeros(batch, self.heads, self.head_dim, self.head_dim, device=device,
                                               dtype=torch.float32))

    def forward(self, u, state=None, pos=0):
        del pos
        Bsz, L, _ = u.shape
        H, d = self.heads, self.head_dim
        xz = F.linear(u, self.in_proj.weight)
        x, z = xz[..., :self.d_conv_in], xz[..., self.d_conv_in:]
        gate = F.linear(u, self.gate_proj.weight).float()
        g = -torch.exp(self.A_log.float()) * F.softplus(gate[..., :H] + self.dt_bias.float())
        beta = torch.sigmoid(gate[..., H:])
        conv_state = None if state is None else state.conv
        if conv_state is not None:
            x = x.to(conv_state.dtype)
        x = causal_conv1d(x, self.conv.weight, self.conv.bias, conv_state=conv_state, update_state=conv_state is not None)
        x = x.reshape(Bsz * L, self.d_conv_in)
        qk = group_norm(x[:, :2 * self.d_key], 2 * self.key_heads, self.unit, eps=1e-6, center=False)
        q, k = qk.reshape(Bsz, L, 2, self.key_heads, d).unbind(2)
        v = x[:, 2 * self.d_key:].reshape(Bsz, L, H, d)
        if state is not None and L == 1:
            o = gated_delta_state_update(state.ssm, q[:, 0], k[:, 0], v[:, 0], g[:, 0], beta[:, 0])
        else:
            o, last = gated_delta_rule(q, k, v, g, beta, h0=None if state is None else state.ssm)
            if state is not None:
                state.ssm.copy_(last)
        o = group_norm(o.reshape(Bsz * L, self.d_inner), H, self.norm_weight, z=z.reshape(Bsz * L, self.d_inner),
                       center=False)
        return F.linear(o.reshape(Bsz, L, self.d_inner), self.out_proj.weight)
