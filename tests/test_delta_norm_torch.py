"""What torch asks of the gated delta rule and the group norm beside values and gradients: forward-mode derivatives and
tracing are refused, and what a backward does not read may change before it."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from mamba_ssm_benchmark_b200 import gated_delta_rule, gated_delta_state_update, group_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _delta():
    gen = torch.Generator().manual_seed(0)
    randn = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    return {"q": randn(1, 70, 1, 16), "k": 0.2 * randn(1, 70, 1, 16), "v": randn(1, 70, 2, 24), "g": -randn(1, 70, 2).abs(),
            "beta": torch.sigmoid(randn(1, 70, 2)), "h0": randn(1, 2, 16, 24)}


def _norm():
    gen = torch.Generator().manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    return {"x": randn(6, 64), "weight": randn(64), "bias": randn(64), "z": randn(6, 64)}


def _step(state, **kw):
    return gated_delta_state_update(state, *(kw[n][:, 0] for n in ("q", "k", "v", "g", "beta")))


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(grad):
    """For every input alone, whether or not something also wants a gradient."""
    with fwAD.dual_level():
        for make, call in ((_delta, gated_delta_rule), (_norm, lambda **kw: group_norm(groups=4, **kw))):
            for name in make():
                t = make()
                if grad:
                    t = {n: x.requires_grad_() for n, x in t.items()}
                t[name] = fwAD.make_dual(t[name], torch.ones_like(t[name]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(**t)
        t = _delta()
        state = t.pop("h0")
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _step(state, **{**t, "v": fwAD.make_dual(t["v"], t["v"])})
        assert torch.isfinite(_step(state, **t)).all()           # without a tangent a level changes nothing


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_tracing_is_refused():
    t, n = _delta(), _norm()
    for fn in (lambda q: gated_delta_rule(**{**t, "q": q}), lambda q: _step(t["h0"].clone(), **{**t, "q": q})):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(fn, (t["q"],), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: group_norm(x, 4), (n["x"],), check_trace=False)


def test_state_updated_in_place_before_the_backward():
    """Truncated back-propagation: the state buffer takes the last state while the graph of the call that read it is alive."""
    t = _delta()
    t["q"].requires_grad_()
    o, last = gated_delta_rule(**t)
    (want,) = torch.autograd.grad(o.sum() + last.sum(), t["q"], retain_graph=True)
    t["h0"].copy_(last.detach())
    (got,) = torch.autograd.grad(o.sum() + last.sum(), t["q"])
    assert torch.equal(got, want)


def test_gradient_of_the_first_state():
    t = {n: x.requires_grad_() for n, x in _delta().items()}
    o, last = gated_delta_rule(**{**t, "h0": t["h0"].transpose(2, 3).contiguous().transpose(2, 3)})
    (a,) = torch.autograd.grad(o.sum() + last.sum(), t["h0"])
    o, last = gated_delta_rule(**{**t, "h0": t["h0"]})
    (b,) = torch.autograd.grad(o.sum() + last.sum(), t["h0"])
    assert a.shape == t["h0"].shape and torch.equal(a, b)
