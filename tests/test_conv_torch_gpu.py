"""causal_conv1d under torch's forward-mode derivatives and torch.jit.trace, without anything that wants a gradient."""

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from mamba_ssm_benchmark_b200 import causal_conv1d

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_forward_mode_is_refused():
    gen = torch.Generator().manual_seed(0)
    t = [torch.randn(*s, generator=gen).to(DEV) for s in ((2, 20, 16), (16, 4), (16,))]
    with fwAD.dual_level():
        want = causal_conv1d(*t)
        for i in range(3):
            args = list(t)
            args[i] = fwAD.make_dual(t[i], torch.ones_like(t[i]))
            with pytest.raises(NotImplementedError):
                causal_conv1d(*args)
    assert torch.equal(causal_conv1d(*t), want)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_a_trace_computes():
    gen = torch.Generator().manual_seed(1)
    x, y, w = (torch.randn(*s, generator=gen).to(DEV) for s in ((2, 20, 16), (2, 20, 16), (16, 4)))
    traced = torch.jit.trace(lambda u: causal_conv1d(u, w), (x,), check_trace=False)
    assert torch.equal(traced(y), causal_conv1d(y, w))
