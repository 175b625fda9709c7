"""The channels-last group norm where its kernels work on rows, channels or layouts at the edge, against its definition in
float64.  Tolerances as in test_norm_gpu.py, from the same count of roundings."""

import pytest
import torch
from test_norm_gpu import F32_TOL, _entering, _inputs, _run

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import group_norm
from oracle import delta_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert nat.read_device_error() == 0


def _hold(got, want, entering, factor=1.0):
    """Every result of `got` against `want`: dx against the size of what enters it, all others against their own."""
    for n, w in want.items():
        assert got[n].shape == w.shape and bool(torch.isfinite(got[n]).all()), n
        off, size = float((got[n].cpu().double() - w).norm()), float(w.norm())
        bound = factor * F32_TOL * (max(size, entering) if n == "dx" else size)
        assert off <= bound + (got[n].dtype == torch.bfloat16) * 2.0 ** -8 * size, (n, off, size)


@pytest.mark.parametrize("shape,groups", [((1, 512), 8), ((7, 512), 8), ((8, 512), 8), ((33, 96), 3), ((1000, 72), 9),
                                          ((9, 2100), 1), ((5, 16400), 1), ((2, 17, 64), 4)])
@pytest.mark.parametrize("silu,gate", [(False, False), (True, False), (True, True)])
def test_eps_of_zero(shape, groups, silu, gate):
    """Rows that fill no CTA: the lanes beside them have no variance, and with eps = 0 no finite rstd."""
    t, dy = _inputs(shape, torch.float32, seed=sum(shape), gate=gate)
    got = _run(lambda x, **kw: group_norm(x, groups, eps=0.0, activation="silu" if silu else None, **kw), t, dy,
               lambda x: x.to(DEV))
    want = _run(lambda x, **kw: O.group_norm(x, groups, eps=0.0, silu=silu, **kw), t, dy, lambda x: x.double())
    _hold(got, want, _entering(t, dy, groups, silu, True))
