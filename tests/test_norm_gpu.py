"""GPU parity of the channels-last group norm (ssm_group_norm_fwd / _bwd) against its definition in float64
(oracle/delta_oracle.py).

Tolerances, on ||difference|| / ||reference||: float32 results pass a dozen roundings of 2^-24 and approximate
exponentials of a few 2^-23, and their sums have at most 32 rounded partial sums in a row: 64 * 2^-24 = 4e-6, taken
as 5e-6; bfloat16 results add one rounding of at most 2^-8.  dx is what its terms leave when the group's mean and
its component along x are taken out, so its error is held against the size of the term that enters, rstd e w, which is
the gradient with the statistics held fixed; with two elements in a group nearly all of it is taken out.
"""

import pytest
import torch

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import group_norm
from oracle import delta_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32_TOL = 5e-6


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert nat.read_device_error() == 0


def _inputs(shape, dtype, seed, gate, affine=True):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)
    t = {"x": (randn(*shape) * 2.0 + 0.5).to(dtype)}
    if affine:
        t["weight"], t["bias"] = 1.0 + 0.2 * randn(shape[-1]), 0.2 * randn(shape[-1])
    if gate:
        t["z"] = randn(*shape).to(dtype)
    return t, randn(*shape).to(dtype)


def _run(fn, t, dy, cast, **kw):
    leaves = {n: cast(x).detach().clone().requires_grad_() for n, x in t.items()}
    y = fn(leaves["x"], weight=leaves.get("weight"), bias=leaves.get("bias"), z=leaves.get("z"), **kw)
    grads = torch.autograd.grad(y, list(leaves.values()), cast(dy))
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}


def _err(a, b):
    b = b.double()
    return float((a.cpu().double() - b).norm() / b.norm().clamp_min(1e-300))


def _check(t, dy, groups, silu, center):
    got = _run(lambda x, **kw: group_norm(x, groups, activation="silu" if silu else None, center=center, **kw), t, dy,
               lambda x: x.to(DEV))
    want = _run(lambda x, **kw: O.group_norm(x, groups, silu=silu, center=center, **kw), t, dy, lambda x: x.double())
    for n, w in want.items():
        half = got[n].dtype == torch.bfloat16
        assert got[n].shape == w.shape, n
        off, size = float((got[n].cpu().double() - w).norm()), float(w.norm())
        bound = F32_TOL * (max(size, _entering(t, dy, groups, silu, center)) if n == "dx" else size)
        assert off <= bound + half * 2.0 ** -8 * size, (n, off, size)
    return got


def _entering(t, dy, groups, silu, center):
    """The size of dx with mean and rstd held fixed."""
    x = t["x"].double().requires_grad_()
    xs = x.detach().reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
    mean = xs.mean(dim=(1, 3), keepdim=True) if center else torch.zeros_like(xs[:, :1, :, :1])
    rstd = ((xs - mean).square().mean(dim=(1, 3), keepdim=True) + 1e-5).rsqrt()
    y = ((x.reshape(xs.shape) - mean) * rstd).reshape(x.shape)
    y = y * t["weight"].double() + t["bias"].double() if "weight" in t else y
    y = y * torch.sigmoid(y) if silu else y
    y = y * torch.nn.functional.silu(t["z"].double()) if "z" in t else y
    return float(torch.autograd.grad(y, x, dy.double())[0].norm())


TOKENS = [((1, 64), 1), ((7, 512), 8), ((33, 96), 3), ((5, 40), 5), ((300, 1024), 8), ((9, 330), 11), ((4, 4096), 2),
          ((1000, 72), 9), ((2, 5120), 40),
          # groups that eight warps share, and that no registers hold
          ((70, 2100), 1), ((3, 4098), 2), ((9, 2099), 1), ((5, 16400), 1)]
SEQUENCES = [((2, 17, 64), 4), ((1, 1, 64), 8), ((3, 101, 30), 5), ((2, 6, 7, 48), 3), ((1, 700, 96), 1), ((5, 2, 24), 24)]


@pytest.mark.parametrize("shape,groups", TOKENS + SEQUENCES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("silu,gate,center", [(False, True, False), (True, False, True), (True, True, True)])
def test_forward_and_gradients(shape, groups, dtype, silu, gate, center):
    t, dy = _inputs(shape, dtype, seed=sum(shape) + groups, gate=gate)
    got = _check(t, dy, groups, silu, center)
    with torch.no_grad():
        d = {n: x.to(DEV) for n, x in t.items()}
        y = group_norm(d["x"], groups, d["weight"], d["bias"], activation="silu" if silu else None, z=d.get("z"),
                       center=center)
    assert y.dtype == dtype and torch.equal(y, got["y"])


@pytest.mark.parametrize("shape,groups", [((6, 64), 2), ((2, 9, 64), 2)])
def test_without_parameters(shape, groups):
    t, dy = _inputs(shape, torch.float32, seed=3, gate=False, affine=False)
    _check(t, dy, groups, False, True)


def test_gradients_against_differences():
    """<grad, d> against central differences of the float64 definition."""
    t, dy = _inputs((3, 8, 24), torch.float32, seed=4, gate=True)
    got = _run(lambda x, **kw: group_norm(x, 3, activation="silu", **kw), t, dy, lambda x: x.to(DEV))
    gen = torch.Generator().manual_seed(9)
    base = {n: x.double() for n, x in t.items()}
    for n in t:
        d = torch.randn(t[n].shape, generator=gen, dtype=torch.float64)
        lo, hi = (float((O.group_norm(groups=3, silu=True, **{**base, n: base[n] + s * 1e-5 * d}) * dy).sum())
                  for s in (-1, 1))
        g = got["d" + n].cpu().double()
        assert abs(float((g * d).sum()) - (hi - lo) / 2e-5) <= F32_TOL * float(g.norm() * d.norm()), n


@pytest.mark.parametrize("shape,groups", [((8, 256), 2), ((2, 500, 32), 2)])
def test_large_common_offset(shape, groups):
    """A mean 1000 times the deviation: the inputs themselves carry 2^-24 * 1000 of the deviation, so results are
    held to 1000 times the usual bound's share of one rounding."""
    t, dy = _inputs(shape, torch.float32, seed=5, gate=False)
    t["x"] = t["x"] + 2000.0
    got = _run(lambda x, **kw: group_norm(x, groups, **kw), t, dy, lambda x: x.to(DEV))
    want = _run(lambda x, **kw: O.group_norm(x, groups, **kw), t, dy, lambda x: x.double())
    for n in want:
        assert _err(got[n], want[n]) <= 1000 * 2.0 ** -24 * 4, n


def test_constant_groups_are_finite():
    """No deviation at all: rstd = eps^-1/2, the output is the bias."""
    x = torch.full((4, 64), 3.0, device=DEV)
    b = torch.randn(64, device=DEV)
    assert torch.equal(group_norm(x, 4, None, b), b.expand(4, 64))
    assert torch.equal(group_norm(x.view(2, 2, 64), 4, None, b), b.expand(2, 2, 64))


def test_strides_and_alignment():
    """x and z as halves of one tensor at an odd offset: equal to dense copies; the gradient of a broadcast input sums."""
    pack = torch.randn(50, 2 * 96 + 3, device=DEV)
    x, z = pack[:, 1:97], pack[:, 98:194]
    assert x.data_ptr() % 16 != 0
    y = group_norm(x, 3, z=z, center=False)
    assert _err(y, O.group_norm(x.double().cpu(), 3, z=z.double().cpu(), center=False)) <= F32_TOL
    xt = torch.randn(96, 50, device=DEV).t()
    assert torch.equal(group_norm(xt, 3), group_norm(xt.contiguous(), 3))
    row = torch.randn(1, 96, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(group_norm(row.expand(50, 96), 3, z=z).sum(), row)
    one = row.detach().double().cpu().requires_grad_()
    (w,) = torch.autograd.grad(O.group_norm(one.expand(50, 96), 3, z=z.double().cpu()).sum(), one)
    assert _err(g, w) <= 50 * F32_TOL          # fifty rows cancel into one


def test_determinism_and_streams():
    t, dy = _inputs((4, 900, 128), torch.bfloat16, seed=6, gate=True)
    run = lambda: _run(lambda x, **kw: group_norm(x, 4, activation="silu", **kw), t, dy, lambda x: x.to(DEV))
    a, side = run(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = run()
    torch.cuda.current_stream().wait_stream(side)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_refusals():
    x = torch.zeros(4, 6, 32, device=DEV)
    with pytest.raises(ValueError, match="groups"):
        group_norm(x, 5)
    with pytest.raises(ValueError, match="empty"):
        group_norm(x[:0], 4)
    with pytest.raises(ValueError, match="samples"):
        group_norm(x[0, 0], 4)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 4, activation="relu")
    with pytest.raises(ValueError, match="z must"):
        group_norm(x, 4, z=x[:, :3])
    with pytest.raises(ValueError, match="weight"):
        group_norm(x, 4, torch.ones(31, device=DEV))
    with pytest.raises(ValueError, match="eps"):
        group_norm(x, 4, eps=-1.0)
    with pytest.raises(TypeError, match="float64"):
        group_norm(x.double(), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        group_norm(x.cpu(), 4)
    with pytest.raises(ValueError, match="one device"):
        group_norm(x, 4, torch.ones(32))
