"""Edges of the operators around a language model's mixers that their other tests pass by.  u = 2^-24."""

import pytest
import torch

from mamba_ssm_benchmark_b200 import embedding, quantize_fp8, rms_norm, rms_norm_fp8, sample_tokens
from oracle import lm_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: U, BF16: 2.0 ** -8}


def _randn(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dtype)


def _within(got, want, bound):
    """|got - want| <= bound, element by element."""
    assert got.shape == want.shape
    off = (got.detach().double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-300)).max())


@pytest.mark.parametrize("shape", [(8,), (4, 8), (2, 4, 8), (2, 3, 2, 24), (1, 1, 8), (3, 5, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_leaves_do_not_share_memory(shape, dtype):
    """x and residual have one gradient; kept by leaves of any number of axes, each adds the next one to its own memory."""
    x, r = (_randn(*shape, seed=i, dtype=dtype).requires_grad_() for i in (1, 2))
    w = torch.ones(shape[-1], device=DEV)

    def step():
        y, total = rms_norm(x, w, residual=r)
        assert y.shape == total.shape == x.shape
        (y.float().sum() + total.float().square().sum()).backward()

    step()
    first = x.grad.clone()
    assert torch.equal(r.grad, first) and x.grad.data_ptr() != r.grad.data_ptr()
    step()
    assert torch.equal(x.grad, 2 * first) and torch.equal(r.grad, 2 * first)
    x.grad.zero_()
    assert torch.equal(r.grad, 2 * first)
    x.grad = r.grad = None
    rms_norm(x, w, residual=r)[1].sum().backward()          # only the sum is used
    assert x.grad.data_ptr() != r.grad.data_ptr()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rms_norm_of_any_layout(dtype):
    """Axes in another order, broadcast, cut and stepped over, as x, residual and gradients: as of dense copies."""
    a = _randn(4, 6, 5, 48, seed=1, dtype=dtype)
    views = [a[:, :, 0], a[:, 2], a[1:, ::2, 1:4], a.transpose(0, 2), a.transpose(1, 3), a[..., 3:40], a[:, :1].expand(4, 6, 5, 48),
             a[0, 0, 0].expand(7, 3, 48), a[:, :, :, :1], a[:, :, :1, :1], a[0, :1, 0], a[..., 1], a[0].movedim(0, -1), a.flip(0)[None]]
    for i, v in enumerate(views):
        dense = v.contiguous().clone()
        C = v.shape[-1]
        w = 1 + 0.1 * _randn(C, seed=2)
        dy = _randn(*v.shape[::-1], seed=3, dtype=dtype).permute(*range(v.dim() - 1, -1, -1))
        results = []
        for x, r, g in ((v, v, dy), (dense, dense, dy.contiguous())):
            x, r, wl = (t.detach().requires_grad_() for t in (x, r, w))
            y, total = rms_norm(x, wl, residual=r)
            alone = rms_norm(x, wl)
            with torch.no_grad():
                y8, scale, t8 = rms_norm_fp8(x, wl, residual=r)
            results.append([y.detach(), total.detach(), alone.detach(), y8.float(), scale, t8, *torch.autograd.grad([y, total, alone], [x, r, wl], [g, g, g])])
        for k, (p, q) in enumerate(zip(*results)):
            # a layout that is not aligned adds a row's values in another order: 2 x 27 u, then a step of the type
            tol = 54 * U + 2 * HALF[p.dtype] if k != 3 else 2.0 ** -3
            assert p.shape == q.shape and p.dtype == q.dtype, (i, k)
            assert float((p.double() - q.double()).norm()) <= tol * float(q.double().norm()), (i, k)


@pytest.mark.parametrize("C", [8200, 20001, 1 << 17, 1 << 20, 1 << 24])
@pytest.mark.parametrize("xd,rd", [(F32, None), (F32, F32), (BF16, F32)])
def test_rms_norm_of_very_long_rows(C, xd, rd):
    """Equal values, whose roundings add up instead of cancelling.  A sum passes 16 additions of a thread, a rounding of those in
    float64 and 9 of the warps': 26 u, of which half reaches the root; the root (4 u), inv_c and two products: 27 u of a value as of any
    row; of a gradient 64 u of its terms' sizes."""
    x = torch.full((1, C), 1.7, device=DEV, dtype=xd)
    r = None if rd is None else torch.full((1, C), 0.6, device=DEV, dtype=rd)
    w = torch.full((C,), 1.1, device=DEV)
    dy = torch.full((1, C), 0.3, device=DEV)
    dy[:, ::2] = 0.9
    dy = dy.to(xd)
    lv = [t.clone().requires_grad_() for t in (x, w)] + ([] if r is None else [r.clone().requires_grad_()])
    out = rms_norm(lv[0], lv[1], residual=lv[2] if r is not None else None)
    y, total = out if r is not None else (out, x)
    grads = torch.autograd.grad(y, lv, dy)
    t = total.detach().double()
    rstd = (t.square().mean() + 1e-5).rsqrt()
    n, g = t * rstd, dy.double() * w.double()
    _within(y, n * w.double(), (27 * U + HALF[xd]) * (n * w.double()).abs())
    mean = (g * n).mean()
    dx, size = rstd * (g - n * mean), rstd * (g.abs() + n.abs() * mean.abs())
    _within(grads[0], dx, 64 * U * size + HALF[xd] * dx.abs())
    _within(grads[1], dy.double()[0] * n[0], 64 * U * (dy.double()[0] * n[0]).abs())
    if r is not None:
        _within(grads[2], dx, 64 * U * size + U * dx.abs())
    y8, scale = rms_norm_fp8(total.detach(), w)
    want = float((n * w.double()).abs().max()) / 448
    assert abs(float(scale) / want - 1) <= 29 * U
    assert bool((y8.float() == 448).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("longest", [64, 127])
def test_embedding_gradient_of_the_longest_chunks(longest, dtype):
    """Runs of 127 places and of one in turn: with as many places as here a chunk is nominally 64 long and ends where a run does, so
    a whole run of 127 is one chunk.  Equal values: 126 additions whose roundings add up, u of the sum each, then the scale and half
    a step."""
    turns, C = 1200, 48
    count = torch.tensor([longest, 128 - longest], device=DEV).repeat(turns)
    idx = torch.repeat_interleave(torch.arange(2 * turns, device=DEV), count)
    assert len(idx) == 128 * turns >= 64 * 148 * 12
    W = torch.zeros(2 * turns, C, device=DEV, dtype=dtype, requires_grad=True)
    dy = torch.full((len(idx), C), 1 / 3, device=DEV).to(dtype)
    dw, = torch.autograd.grad(embedding(idx, W, 1.7), W, dy)
    want = count[:, None].double() * float(dy[0, 0].double()) * 1.7
    _within(dw, want.expand(-1, C), ((126 + 2) * U + HALF[dtype]) * want)
    assert torch.equal(dw, torch.autograd.grad(embedding(idx, W, 1.7), W, dy)[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [4, 900, 3000, 60000, 400000])
def test_sample_the_widest_range(V, dtype):
    """Logits from the type's lowest value to its highest, whose distances a float32 does not hold, at temperatures where they matter
    and at ones where they do not; some masked.  Up to 2 V 2^-42 of the largest weight may lie between two tokens at a border."""
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.linspace(-1, 1, V, device=DEV).double()[torch.randperm(V, device=DEV, generator=g)] * torch.finfo(dtype).max
    logits = torch.stack([logits.to(dtype), logits.to(dtype).masked_fill(torch.rand(V, device=DEV, generator=g) < 0.3, float("-inf"))])
    logits[1, V // 2] = torch.finfo(dtype).max
    u = torch.tensor([0.03, 0.97], device=DEV)
    for at in (u, u.flip(0)):
        for T in (1.0, 1e36, 1e37, 2e37, 1e39, 1e300, float("inf")):
            for kw in (dict(), dict(top_k=V - 2), dict(top_p=0.9), dict(top_k=V // 2, top_p=0.9), dict(top_k=600), dict(min_p=0.9), dict(top_p=0.01)):
                got = sample_tokens(logits, at, temperature=T, **kw).tolist()
                for b in range(2):
                    l = logits[b].double()
                    want = O.sample(l, float(at[b].double()), temperature=T, **kw)
                    between = torch.exp((l[min(got[b], want) + 1:max(got[b], want)] - l.max()) / T).nan_to_num(0.0)
                    assert got[b] == want or float(between.sum()) < 2 * V * 2.0 ** -42, (T, kw, b, got[b], want)


@pytest.mark.parametrize("residual", [False, True])
def test_rms_norm_gradient_against_differences_of_its_own_forward(residual):
    """Along random directions, x, residual and weight together and each alone: (f(+h) - f(-h)) / 2h of the float32 forward.
    Each f is off by 28 u of every |y c| (27 u and the rounding) and u of every |total c|, so the quotient by that over h; the step
    itself by what the same quotient of the float64 definition is off at h against h / 1000, whose own error is (h / 1000)^2; a gradient by
    64 u of its terms' sizes, at most 64 u (|g| + |n| mean|g n|) rstd <= 1000 u here."""
    rows, C, h = 6, 96, 2.0 ** -6
    x, w, r = _randn(rows, C, seed=1), 1 + 0.1 * _randn(C, seed=2), 2 * _randn(rows, C, seed=3)
    cy, ct = _randn(rows, C, seed=4), _randn(rows, C, seed=5)
    leaves = [x, w] + ([r] if residual else [])

    def loss(norm, at):
        out = norm(at[0], at[1], *at[2:])
        y, total = out if residual else (out, None)
        return float((y.double() * cy.double()).sum() + ((total.double() * ct.double()).sum() if residual else 0.0))

    own = lambda x, w, r=None: rms_norm(x, w, residual=r)
    exact = lambda x, w, r=None: O.rms_norm(x, w, r) if residual else O.rms_norm(x, w)[0]
    out = own(*leaves)
    y, total = (t.double() for t in out) if residual else (out.double(), None)
    noise = float(28 * U * (y.abs() * cy.abs()).sum() + (U * (total.abs() * ct.abs()).sum() if residual else 0.0)) / h
    for moved in [tuple(range(len(leaves)))] + [(i,) for i in range(len(leaves))]:
        d = [_randn(*t.shape, seed=20 + i) if i in moved else torch.zeros_like(t) for i, t in enumerate(leaves)]
        quotient = lambda norm, at, d, h: (loss(norm, [a + h * b for a, b in zip(at, d)]) - loss(norm, [a - h * b for a, b in zip(at, d)])) / (2 * h)
        # the points as float32 has them, exactly h d to either side
        at = [(t * 2 ** 10).round() / 2 ** 10 for t in leaves]
        d = [(t * 2 ** 10).round() / 2 ** 10 for t in d]
        lv = [t.clone().requires_grad_() for t in at]
        grads = torch.autograd.grad(own(*lv), lv, (cy, ct) if residual else cy)
        wide = [t.double() for t in at], [t.double() for t in d]
        step = abs(quotient(exact, *wide, h) - quotient(exact, *wide, h / 1000))
        got = sum(float((g.double() * b.double()).sum()) for g, b in zip(grads, d))
        size = sum(float(b.abs().double().sum()) for b in d)
        assert abs(got - quotient(own, at, d, h)) <= noise + step + 1e-5 + 1000 * U * size, moved


@pytest.mark.parametrize("xd,rd", [(BF16, None), (BF16, BF16), (BF16, F32), (F32, F32)])
def test_rms_norm_gradient_along_the_row(xd, rd):
    """The norm does not change as its row grows: the mean of g n takes away what g has along the row, and without it the
    derivative would be the sum of g n, ten times the bound in bf16 and more in float32.  That is left by eps and dtotal, exactly known; the bound is the gradient's
    own rounding and 64 u of its terms."""
    rows, C = 5, 1000
    x, w = _randn(rows, C, seed=1, dtype=xd), 1 + 0.1 * _randn(C, seed=2)
    r = None if rd is None else _randn(rows, C, seed=3).to(rd)
    lv = [x.clone().requires_grad_()] + ([] if r is None else [r.clone().requires_grad_()])
    out = rms_norm(lv[0], w, residual=lv[1] if r is not None else None)
    y, total = out if r is not None else (out, x)
    t = total.detach().double()
    rstd = (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    n = t * rstd
    dy = (n + 0.3 * _randn(rows, C, seed=4)).to(xd)
    ct = 0.01 * _randn(rows, C, seed=5).to(total.dtype)
    grads = torch.autograd.grad(out, lv, (dy, ct) if r is not None else dy)
    g = dy.double() * w.double()
    want = (g * n * 1e-5 * rstd.square()).sum(-1) + (0.0 if r is None else (ct.double() * t).sum(-1))
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + (0.0 if r is None else ct.double().abs())
    for d in grads:
        bound = ((64 * U * size + HALF[d.dtype] * d.double().abs()) * t.abs()).sum(-1)
        _within((d.double() * t).sum(-1), want, bound)
        assert bool(((g * n).sum(-1) > 100 * bound).all() if d.dtype == F32 else ((g * n).sum(-1) > 10 * bound).all())


@pytest.mark.parametrize("T", [1, 31, 1023, 1024, 1025, 1500, 2048, 4096, 16384, 16385])
@pytest.mark.parametrize("V", [3, 511, 512, 70000])
def test_embedding_gradient_on_both_sides_of_the_sorts_borders(T, V):
    """One CTA, eight and sixteen, a pass or two: whole numbers, whose sums are exact."""
    g = torch.Generator(device=DEV).manual_seed(T)
    idx = torch.randint(0, V, (T,), device=DEV, generator=g)
    W = torch.zeros(V, 8, device=DEV, requires_grad=True)
    dy = torch.randint(-4, 5, (T, 8), device=DEV, generator=g).float()
    dw, = torch.autograd.grad(embedding(idx, W), W, dy)
    assert torch.equal(dw.double(), O.embedding_grad(idx, dy, V, 1.0)[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("C", [96, 2560, 9000])
def test_values_next_to_the_borders_of_e4m3(C, norm, dtype):
    """Rows full of values near the middle between two e4m3, off it by up to 16 float32 steps.  y / scale = t w 448 / max|t w|: the
    products t w (of the value and of the largest one), the quotient and the last product round, u each; a value further than that from the middle
    goes to its nearest."""
    g = torch.Generator(device=DEV).manual_seed(C)
    rows = 300
    mids = torch.tensor([(8 + k + 0.5) * 2.0 ** e for e in range(-4, 5) for k in range(8)], device=DEV).double()
    mids = mids[mids < 440]
    big = torch.exp(4 * torch.randn(rows, 1, device=DEV, generator=g)).to(dtype)
    off = torch.randint(-16, 17, (rows, C), device=DEV, generator=g).double() * 2.0 ** -23
    w = 1 + 0.1 * torch.randn(C, device=DEV, generator=g) if norm else torch.ones(C, device=DEV)
    v = mids[torch.randint(0, len(mids), (rows, C), device=DEV, generator=g)] * (1 + off) * (1 - 2 * torch.randint(0, 2, (rows, C), device=DEV, generator=g))
    x = (v * big.double() / 448 / w.double()).to(dtype)
    x[:, 5] = big[:, 0]
    x[:, 5] *= 2
    y8, scale = rms_norm_fp8(x, w) if norm else quantize_fp8(x)
    t = x.double() * w.double()
    v = t * 448 / t.abs().amax(-1, keepdim=True)
    half = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 4)
    _within(y8.double(), v, half + (4 if norm else 2) * U * (1 + 2 * U) * v.abs())
    y = O.rms_norm(x.double(), w.double())[0] if norm else t
    want = y.abs().amax(-1) / 448
    _within(scale, want, (27 + 2) * U * want)
