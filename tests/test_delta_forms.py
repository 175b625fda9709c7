"""The gated delta rule's chain kernels, each by name: strips of 16 channels, one or two to a CTA, and tcgen05 with 128.  The
library's choice of a form is asserted first (CPU), so that a change of its rule cannot leave a form untested; then every
form runs in both types, with and without a first state, in training and inference (GPU).

Tolerances as in test_delta_gpu.py."""

import ctypes

import pytest
import torch
from test_delta_gpu import F32_TOL, NAMES, _compare, _err, _inputs, _run

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import gated_delta_rule, gated_delta_state_update
from oracle import delta_oracle as O

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16

# (B, L, Hk, Hv, dk, dv), types, channels a CTA: lengths that end inside a chunk, widths that fill no tile
FORMS = [
    ((1, 130, 2, 4, 64, 48), (F32, BF16), 16), ((2, 70, 2, 2, 100, 40), (F32, BF16), 16), ((16, 70, 4, 8, 128, 128), (F32,), 16),
    ((5, 130, 4, 8, 64, 64), (F32,), 32), ((5, 130, 4, 8, 100, 50), (BF16,), 32), ((8, 70, 7, 21, 128, 48), (BF16,), 32),
    ((5, 130, 4, 8, 64, 64), (BF16,), 16), ((16, 70, 4, 16, 48, 16), (BF16,), 16),
    ((16, 130, 4, 8, 64, 128), (F32, BF16), 128), ((8, 199, 8, 16, 48, 100), (F32, BF16), 128),
    ((16, 65, 8, 8, 64, 144), (F32, BF16), 128), ((16, 130, 4, 8, 128, 128), (BF16,), 128),
    ((8, 70, 5, 15, 100, 90), (BF16,), 128), ((150, 1, 1, 1, 33, 112), (F32, BF16), 128),
]
CASES = [(shape, dtype, channels) for shape, dtypes, channels in FORMS for dtype in dtypes]


@pytest.mark.parametrize("shape,dtype,channels", CASES)
def test_choice(shape, dtype, channels):
    assert [nat.delta_channels(*shape, dtype, backward) for backward in (False, True)] == [channels] * 2


@pytest.mark.parametrize("heads,dk,dv,dtype,channels", [
    (385, 128, 48, BF16, (32, 32)), (200, 64, 48, BF16, (16, 16)), (385, 64, 48, BF16, (16, 16)), (100, 128, 48, BF16, (32, 32)),
    (200, 64, 48, F32, (32, 32)), (148, 128, 128, BF16, (128, 128)), (50, 64, 128, BF16, (128, 16)),
    (128, 128, 48, BF16, (128, 128)), (128, 64, 48, F32, (128, 128)), (4, 128, 48, BF16, (16, 16)),
])
def test_choice_is_the_fastest_measured(heads, dk, dv, dtype, channels):
    """Shapes at which another choice took at least 8 % more for 1024 positions."""
    assert tuple(nat.delta_channels(1, 1024, heads, heads, dk, dv, dtype, backward) for backward in (False, True)) == channels


def test_choice_refusals():
    n = ctypes.c_int32(0)
    plan = lambda *a: nat.lib().ssm_gated_delta_plan(*a)
    assert plan(1, 1, 1, 1, 16, 16, nat.SSM_F32, 0, None) == nat.SSM_ERR_INVALID
    assert plan(1, 1, 2, 3, 16, 16, nat.SSM_F32, 0, ctypes.byref(n)) == nat.SSM_ERR_INVALID
    assert plan(1, 1, 1, 1, 16, 16, 7, 0, ctypes.byref(n)) == nat.SSM_ERR_DTYPE


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype,channels", CASES)
@pytest.mark.parametrize("h0,scale", [(True, None), (False, 0.37)])
def test_form(shape, dtype, channels, h0, scale):
    t, do, dlast = _inputs(*shape, dtype=dtype, h0=h0, seed=sum(shape))
    got = _run(lambda **kw: gated_delta_rule(**kw, scale=scale), t, do, dlast, lambda x: x.to(DEV))
    want = _run(lambda **kw: O.gated_delta_rule(**kw, scale=scale), t, do, dlast, lambda x: x.to(DEV).double())
    _compare(got, {n: x.cpu() for n, x in want.items()})
    d = {n: None if x is None else x.to(DEV) for n, x in t.items()}
    with torch.no_grad():                      # inference saves nothing
        o, last = gated_delta_rule(**d, scale=scale)
    assert torch.equal(o, got["o"]) and torch.equal(last, got["last"])
    again = _run(lambda **kw: gated_delta_rule(**kw, scale=scale), t, do, dlast, lambda x: x.to(DEV))
    for n, x in got.items():
        assert torch.equal(again[n], x), n
    assert nat.read_device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 1, 2, 32, 24), (64, 2, 4, 128, 64)])       # one channel a lane, four
def test_scale_of_the_state_update(shape):
    B, Hk, Hv, dk, dv = shape
    t, *_ = _inputs(B, 1, Hk, Hv, dk, dv, seed=7)
    state = t["h0"].to(DEV)
    o = gated_delta_state_update(state, *(t[n][:, 0].to(DEV) for n in NAMES[:5]), scale=-0.37)
    want_o, want_s = O.gated_delta_rule(**{n: x.double() for n, x in t.items()}, scale=-0.37)
    assert _err(o, want_o[:, 0]) <= F32_TOL and _err(state, want_s) <= F32_TOL
    assert nat.read_device_error() == 0
