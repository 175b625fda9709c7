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


def _windows(t, C):
    return t.unfold(0, C, 1)                 # rows that overlap: strides (1, 1)


@pytest.mark.parametrize("which", ["x", "z", "both"])
def test_overlapping_rows(which):
    """x, z or both as sliding windows over one array: results and gradients are those of the rows, each for itself."""
    rows, C, groups = 37, 64, 4
    t, dy = _inputs((rows, C), torch.float32, seed=11, gate=True)
    gen = torch.Generator().manual_seed(12)
    long = {n: torch.randn(rows + C - 1, generator=gen) for n in ("x", "z")}
    for n in long:
        if which in (n, "both"):
            t[n] = _windows(long[n], C)
    want = _run(lambda x, **kw: O.group_norm(x, groups, **kw), t, dy, lambda x: x.double().contiguous())
    leaves = {n: (_windows(long[n].to(DEV), C) if which in (n, "both") and n in long else x.to(DEV)).requires_grad_()
              for n, x in t.items()}
    assert any(x.stride() == (1, 1) for x in leaves.values())
    y = group_norm(leaves["x"], groups, leaves["weight"], leaves["bias"], z=leaves["z"])
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(DEV))
    _hold({"y": y.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}, want, _entering(t, dy, groups, False, True))


def test_overlapping_positions():
    """The same with more than one position: strides (5, 3, 1)."""
    base = torch.randn(5 * 2 + 3 * 8 + 64, generator=torch.Generator().manual_seed(13))
    shape, strides = (3, 9, 64), (5, 3, 1)
    t, dy = _inputs(shape, torch.float32, seed=14, gate=False)
    t["x"] = base.as_strided(shape, strides)
    want = _run(lambda x, **kw: O.group_norm(x, 4, **kw), t, dy, lambda x: x.double().contiguous())
    leaves = {n: (base.to(DEV).as_strided(shape, strides) if n == "x" else x.to(DEV)).requires_grad_() for n, x in t.items()}
    y = group_norm(leaves["x"], 4, leaves["weight"], leaves["bias"])
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(DEV))
    _hold({"y": y.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}, want, _entering(t, dy, 4, False, True))


def test_more_groups_than_a_grid_holds():
    """2^31 (sample, group) pairs: every one has its statistics, in both directions.  Samples are independent, so slices of
    the results are held against the definition of the same slice; dx is exact 0 up to rounding with two elements a group,
    so the groups here are one channel at two positions with a weight, and dx is held against the size of what enters."""
    N, P, C = 2 ** 21, 2, 1024
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 130 * 2 ** 30:
        pytest.skip("needs 130 GB")
    gen = torch.Generator(device=DEV).manual_seed(21)
    x = torch.empty(N, P, C, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    w = (1.0 + 0.1 * torch.randn(C, generator=gen, device=DEV)).requires_grad_()
    slices = (slice(0, 3), slice(N // 2 - 1, N // 2 + 2), slice(N - 3, N))
    dy = torch.zeros_like(x)
    for sl in slices:
        dy[sl].normal_(generator=gen)
    x.requires_grad_()
    y = group_norm(x, C, w)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    want_dw = torch.zeros(C, dtype=torch.float64)
    for sl in slices:
        t = {"x": x.detach()[sl].cpu(), "weight": w.detach().cpu(), "bias": torch.zeros(C)}
        want = _run(lambda x, **kw: O.group_norm(x, C, **kw), t, dy[sl].cpu(), lambda x: x.double())
        want_dw += want["dweight"]
        _hold({"y": y.detach()[sl], "dx": dx[sl]}, {n: want[n] for n in ("y", "dx")}, _entering(t, dy[sl].cpu(), C, False, True))
    off = float((dw.cpu().double() - want_dw).norm())
    assert off <= F32_TOL * float(want_dw.norm())
    del x, y, dx, dy
    torch.cuda.empty_cache()


@pytest.mark.parametrize("shape", [(65536, 2, 64), (1 << 24, 8), (1, 1 << 22, 8), (3001, 4100)])
def test_parameter_gradients_of_many_rows(shape):
    """A constant gradient: every rounding of a running sum may go the same way.  One fp32 sum has at most 256 rows, and a
    dozen more roundings follow before fp64: 270 * 2^-24 of the terms' sizes; dbias has terms of one sign."""
    x = torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(31), device=DEV)
    w, b = (torch.ones(shape[-1], device=DEV, requires_grad=True) for _ in range(2))
    dy = torch.full_like(x, 1.3)
    dw, db = torch.autograd.grad(group_norm(x, 1, w, b, center=False), [w, b], dy)
    bound = 270 * 2.0 ** -24
    n = x.double()
    n = n / (n.square().mean(dim=tuple(range(1, x.dim())), keepdim=True) + 1e-5).sqrt()
    over = tuple(range(x.dim() - 1))
    want = float(dy[(0,) * x.dim()].double()) * (x.numel() // shape[-1])
    assert float((db.double() - want).abs().max()) <= bound * want
    scale = float(dy[(0,) * x.dim()].double())
    assert bool(((dw.double() - scale * n.sum(over)).abs() <= (bound + F32_TOL) * scale * n.abs().sum(over)).all())


@pytest.mark.parametrize("shape,groups", [((3, 300, 64), 4), ((40, 64), 4), ((3, 2100), 1), ((3, 16400), 1)])
def test_infinite_elements_without_centring(shape, groups):
    """x / rms with an infinite element in a group: rms is infinite, so the element itself gives NaN and its group's others 0;
    in the first row, in a later one, and of both signs at once.  Other groups are what they are."""
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(41))
    x.view(shape[0], -1)[0, 3], x[1].view(-1)[-1] = float("inf"), float("-inf")
    x[2].view(-1)[0], x[2].view(-1)[5] = float("inf"), float("-inf")
    want = O.group_norm(x.double(), groups, center=False)
    y = group_norm(x.to(DEV), groups, center=False).cpu()
    assert int(want.isnan().sum()) == 4 and torch.equal(y.isnan(), want.isnan())
    assert torch.equal(y == 0, want == 0)
    fine = ~want.isnan()
    assert float((y[fine] - want[fine]).norm()) <= F32_TOL * float(want[fine].norm())
