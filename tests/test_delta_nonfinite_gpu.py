"""A non-finite value in an input of the gated delta rule reaches no output before its position: by the recurrence the state
is what it was up to there.  Outputs before it are held bit by bit to those of the call without it (a zero above a diagonal
times anything finite adds nothing), outputs from it on are not finite."""

import pytest
import torch
from test_delta_gpu import _inputs

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import gated_delta_rule

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
NAN, INF = float("nan"), float("inf")

# every chain kernel: (B, L, Hk, Hv, dk, dv), type, channels a CTA
FORMS = [((1, 200, 1, 2, 64, 48), F32, 16), ((1, 200, 1, 2, 64, 40), BF16, 16), ((2, 200, 1, 2, 128, 33), F32, 16),
         ((1, 200, 2, 2, 100, 48), BF16, 16), ((5, 200, 4, 8, 64, 64), F32, 32), ((5, 200, 4, 8, 128, 64), BF16, 32),
         ((16, 200, 4, 8, 64, 128), F32, 128), ((16, 200, 4, 8, 64, 100), BF16, 128), ((16, 200, 8, 8, 128, 128), BF16, 128)]


@pytest.mark.parametrize("shape,dtype,channels", FORMS)
@pytest.mark.parametrize("name,value", [("v", NAN), ("v", INF), ("v", -INF), ("k", NAN), ("k", INF), ("q", NAN), ("beta", NAN),
                                        ("g", NAN)])
@pytest.mark.parametrize("at", [0, 30, 64 + 15, 64 + 44, 128 + 63])
def test_outputs_before_a_non_finite_input(shape, dtype, channels, name, value, at):
    assert nat.delta_channels(*shape, dtype) == channels
    t, *_ = _inputs(*shape, dtype=dtype, seed=sum(shape))
    t = {n: x.to(DEV) for n, x in t.items()}
    with torch.no_grad():
        clean, _ = gated_delta_rule(**t)
        if name in ("q", "k", "v"):
            t[name][0, at, -1, 3] = value                       # one channel of one head
        else:
            t[name][0, at, -1] = value
        o, last = gated_delta_rule(**t)
        lv = {n: x.clone().requires_grad_() for n, x in t.items()}
    o2 = gated_delta_rule(**lv)[0].detach()                      # the training form of the kernel
    assert torch.equal(o[:, :at], clean[:, :at]) and torch.equal(o[1:], clean[1:])
    assert torch.equal(o.isnan(), o2.isnan()) and torch.equal(o2[:, :at], clean[:, :at])
    H, group = shape[3], shape[3] // shape[2]
    heads = slice(H - 1, H) if name in ("v", "g", "beta") else slice(H - group, H)
    assert torch.equal(o[:, :, :heads.start], clean[:, :, :heads.start])
    later, state = o[0, at:, heads], last[0, heads]
    if name == "v":                                               # a channel of its own
        rest = [i for i in range(shape[5]) if i != 3]
        assert torch.equal(o[..., rest], clean[..., rest])
        later, state = later[..., 3], state[..., 3]
    if name == "q":
        assert torch.equal(o[:, at + 1:], clean[:, at + 1:]) and torch.isfinite(last).all()
        later, state = later[:1], later[:1]
    assert not torch.isfinite(later).any() and not torch.isfinite(state).any()
    assert nat.read_device_error() == 0


@pytest.mark.parametrize("shape,dtype,channels", FORMS)
def test_divergence_is_not_hidden(shape, dtype, channels):
    """Keys far longer than 1: the state grows by a factor of up to beta |k|^2 a position and overflows, in the triangular
    inverse first.  Once the recurrence (in float64) is beyond float32's range, outputs are not finite, and never something
    finite instead.  (Up to 15 outputs in front of an overflow inside a chunk may go with it.)"""
    t, *_ = _inputs(*shape, dtype=dtype, h0=False, seed=sum(shape))
    t["k"] = t["k"] * 100
    t["g"], t["beta"] = torch.zeros_like(t["g"]), torch.ones_like(t["beta"])
    t = {n: x if x is None else x[:1].to(DEV).expand(shape[0], *x.shape[1:]).contiguous() for n, x in t.items()}
    with torch.no_grad():
        o, last = gated_delta_rule(**t)
        S = torch.zeros(shape[3], shape[4], shape[5], dtype=torch.float64, device=DEV)
        group, size = shape[3] // shape[2], []
        for i in range(shape[1]):
            k = t["k"][0, i].double().repeat_interleave(group, 0)
            S = S + k[..., None] * (t["v"][0, i].double() - (S * k[..., None]).sum(1))[:, None]
            size.append(S.abs().amax(1).amin())              # of the smallest channel
    size = torch.stack(size)
    over = ~(size <= 1e42)                                   # float64 overflows too
    assert int(over.sum()) > 20
    assert not torch.isfinite(o[:, over]).any() and not torch.isfinite(last).any()
