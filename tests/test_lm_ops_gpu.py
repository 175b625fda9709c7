"""The operators around a language model's mixers against their definitions in float64 (oracle/lm_oracle.py).

Bounds, with u = 2^-24 and half a step h of the result's type (2^-24 fp32, 2^-8 bf16) relative to the value:
  * rms_norm: a row's sum of squares passes at most 32 + 5 + 8 additions, half of whose error reaches the root; the root, the
    quotient and two products add one u each: 27 u of every value, then h.
  * its gradient: the same of each of its terms' sizes; of the weight: chains of 256 rows, 30 u before: 286 u of the sum of
    absolute terms.
  * embedding's gradient: chunks of at most 64 places, joined in float64: 64 u of the sum of absolute terms.
  * linear_fp8: an instruction adds 32 exact products to an fp32 accumulator and may truncate (2 u of what it has so far),
    and up to seven parts of K are added: (K / 32 + 64) 2 u of the sum of absolute terms; SiLU's slope is below 1.1, its own
    error 2^-20 of its argument; then h.
Tokens and ranks have no tolerance."""

import pytest
import torch

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import embedding, linear_fp8, quantize_fp8, rms_norm, rms_norm_fp8, sample_tokens
from oracle import lm_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
HALF = {F32: U, BF16: 2.0 ** -8}


def _gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, device=DEV, generator=_gen(seed)).to(dtype)


def _within(got, want, bound, what=""):
    """|got - want| <= bound, element by element (bound a tensor or a number)."""
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (what, float((off / torch.as_tensor(bound).clamp_min(1e-300)).max()))


# ---- embedding ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,V,C,scale", [(1, 1, 1, 1.0), (8, 256, 256, 1.0), (33, 50, 330, 3.5), (700, 3, 7, 1.0), (5, 100000, 96, 0.1),
                                         (4097, 700, 130, 16.0), (20000, 300, 64, 1.0), (3000, 5000, 2561, 1.0)])
def test_embedding(T, V, C, scale, dtype):
    W = _randn(V, C, seed=1, dtype=dtype).requires_grad_()
    idx = (torch.rand(T, device=DEV, generator=_gen(2)) ** 3 * V).long().clamp_max(V - 1)
    dy = _randn(T, C, seed=3, dtype=dtype)
    y = embedding(idx, W, scale)
    assert torch.equal(y, (W.detach().float() * scale).to(dtype)[idx])
    dw, = torch.autograd.grad(y, W, dy)
    assert dw.dtype == dtype
    want, size = O.embedding_grad(idx, dy, V, scale)
    _within(dw, want, 66 * U * size + HALF[dtype] * want.abs())
    assert torch.equal(dw, torch.autograd.grad(embedding(idx, W, scale), W, dy)[0])     # bit by bit


def test_embedding_one_token_everywhere():
    """A run over all chunks; every other row is zero."""
    W = _randn(300, 64).requires_grad_()
    for T in (64, 65, 5000, 70000):
        idx = torch.full((T,), 7, device=DEV)
        dy = torch.rand(T, 64, device=DEV, generator=_gen(T)) + 1.0
        dw, = torch.autograd.grad(embedding(idx, W), W, dy)
        want = dy.double().sum(0)
        _within(dw[7], want, 66 * U * want)
        dw[7] = 0.0
        assert not dw.any()


@pytest.mark.parametrize("T", [4095, 4097, 16385, 131072, 131073, 300001])
def test_embedding_of_many_tokens(T):
    """Every form of the sort: one CTA, eight, sixteen, more places than stay in registers.  Whole numbers: sums are exact."""
    V = 3000
    idx = (torch.rand(T, device=DEV, generator=_gen(T)) ** 4 * V).long().clamp_max(V - 1)
    W = torch.zeros(V, 8, device=DEV, requires_grad=True)
    dy = torch.randint(-4, 5, (T, 8), device=DEV, generator=_gen(1)).float()
    dw, = torch.autograd.grad(embedding(idx.int(), W), W, dy)
    assert torch.equal(dw.double(), O.embedding_grad(idx, dy, V, 1.0)[0])


@pytest.mark.parametrize("V", [511, 512, 513, 262143, 262144, 300000])
def test_embedding_sorts_every_digit(V):
    """Places by token where a pass more or less is needed, the first and last ids among them."""
    idx = torch.cat([torch.tensor([V - 1, 0, V - 1, 511 % V, V // 2], device=DEV),
                     torch.randint(0, V, (9000,), device=DEV, generator=_gen(V))])
    W = torch.zeros(V, 4, device=DEV, requires_grad=True)
    dy = torch.randint(-8, 9, (len(idx), 4), device=DEV, generator=_gen(1)).float()      # sums are exact
    dw, = torch.autograd.grad(embedding(idx, W), W, dy)
    assert torch.equal(dw.double(), O.embedding_grad(idx, dy, V, 1.0)[0])


def test_embedding_layouts_and_ids():
    W = _randn(40, 24)
    idx = torch.randint(0, 40, (3, 5), device=DEV, generator=_gen(0))
    assert torch.equal(embedding(idx, W), W[idx])
    assert torch.equal(embedding(idx.int(), W), W[idx])
    assert torch.equal(embedding(idx.t(), W), W[idx.t()])
    wide = _randn(40, 70)
    for view in (wide[:, 3:27], wide[:, 4:28], wide.t()[:40, :24], wide[::2, :24]):
        rows = idx % view.shape[0]
        assert torch.equal(embedding(rows, view), view[rows])
        v = view.detach().requires_grad_()
        dy = _randn(3, 5, 24, seed=4)
        dw, = torch.autograd.grad(embedding(rows, v), v, dy)
        want, size = O.embedding_grad(rows.flatten(), dy.flatten(0, 1), len(view), 1.0)
        _within(dw, want, 66 * U * size + U * want.abs())
    v = W.clone().requires_grad_()
    dw, = torch.autograd.grad(embedding(idx, v).sum(), v)               # a broadcast gradient
    assert torch.equal(dw, torch.bincount(idx.flatten(), minlength=40).float()[:, None].expand(40, 24))


def test_embedding_ids_outside_the_table():
    W = _randn(10, 33).requires_grad_()
    idx = torch.tensor([3, -1, 10, 9, 1 << 40, 3], device=DEV)
    nat.read_device_error()
    y = embedding(idx, W)
    assert nat.read_device_error() == 2
    bad = torch.tensor([False, True, True, False, True, False], device=DEV)
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], W.detach()[idx[~bad]])
    dy = _randn(6, 33, seed=1)
    dw, = torch.autograd.grad(y, W, dy)
    want, _ = O.embedding_grad(idx[~bad], dy[~bad], 10, 1.0)
    _within(dw, want, 4 * U * dy.abs().sum(0).double())
    y = embedding(torch.tensor([-5, 12], device=DEV), W)
    dw, = torch.autograd.grad(y, W, dy[:2])
    assert not dw.any()
    assert nat.read_device_error() == 2


# ---- RMS norm ---------------------------------------------------------------------------------------
TYPES = [(F32, None), (BF16, None), (F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)]
SHAPES = [(1, 1), (1, 256), (3, 7), (5, 330), (700, 33), (2, 1024), (33, 2560), (9, 4095), (4, 5120), (3, 8192), (2, 8194), (2, 20001)]


@pytest.mark.parametrize("xd,rd", TYPES)
@pytest.mark.parametrize("rows,C", SHAPES)
def test_rms_norm(rows, C, xd, rd):
    x = _randn(rows, C, seed=1, dtype=xd).requires_grad_()
    r = None if rd is None else (2 * _randn(rows, C, seed=2)).to(rd).requires_grad_()
    w = (1 + 0.1 * _randn(C, seed=3)).requires_grad_()
    out = rms_norm(x, w, residual=r)
    leaves = [t for t in (x, w, r) if t is not None]
    dy = _randn(rows, C, seed=4, dtype=xd)
    if r is None:
        y, total, dt = out, x.detach(), None
        grads = torch.autograd.grad(y, leaves, dy)
    else:
        y, total = out
        wide = torch.promote_types(xd, rd)
        assert total.dtype == wide and torch.equal(total, (x.detach().float() + r.detach().float()).to(wide))
        dt = _randn(rows, C, seed=5, dtype=wide)
        grads = torch.autograd.grad([y, total], leaves, [dy, dt])
    t, wd, g = total.detach().double(), w.detach().double(), dy.double() * w.detach().double()
    rstd = (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    n = t * rstd
    assert y.dtype == xd
    _within(y, n * wd, (27 * U + HALF[xd]) * (n * wd).abs(), "y")
    c = (g * n).mean(-1, keepdim=True)
    dx = rstd * (g - n * c) + (0.0 if dt is None else dt.double())
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) + (0.0 if dt is None else dt.double().abs())
    _within(grads[0], dx, 64 * U * size + HALF[xd] * dx.abs(), "dx")
    _within(grads[1], (dy.double() * n).sum(0), 290 * U * (dy.double() * n).abs().sum(0), "dw")
    if r is not None:
        assert grads[2].dtype == rd
        _within(grads[2], dx, 64 * U * size + HALF[rd] * dx.abs(), "dr")


@pytest.mark.parametrize("xd,rd", [(F32, None), (F32, F32), (BF16, BF16), (BF16, F32)])
def test_rms_norm_gradient_against_differences(xd, rd):
    """Along a random direction, in steps of the float32 forward that its roundings allow: 1e-3 of the derivative."""
    x, r, w = _randn(6, 96, seed=1, dtype=xd), _randn(6, 96, seed=2), 1 + 0.1 * _randn(96, seed=3)
    r = None if rd is None else r.to(rd)
    cy, ct = _randn(6, 96, seed=4), _randn(6, 96, seed=5)
    loss = lambda x, w, r: (rms_norm(x, w, residual=r) * cy).sum() if r is None else \
        sum((a * b).sum() for a, b in zip(rms_norm(x, w, residual=r), (cy, ct)))
    lv = [t.clone().requires_grad_() for t in (x, w) + (() if r is None else (r,))]
    grads = torch.autograd.grad(loss(*lv, *((None,) if r is None else ())), lv)
    def exact(x, w, r):
        y, total = O.rms_norm(x, w, r)
        return (y * cy.double()).sum() + (0.0 if r is None else (total * ct.double()).sum())
    for i, g in enumerate(grads):
        d = _randn(*g.shape, seed=10 + i).double()
        at = [t.detach().double() for t in lv]
        at = at + [None] * (3 - len(at))
        h = 1e-5
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + h * d, at[i] - h * d
        want = float((exact(*plus) - exact(*minus)) / (2 * h))
        got = float((g.double() * d).sum())
        size = float((g.double() * d).abs().sum())
        # total is rounded to its type before it is normed, and every gradient to its own
        assert abs(got - want) <= (1e-5 + 4 * max(HALF[xd], HALF[rd or xd], HALF[g.dtype]) * (0 if F32 is xd else 1)) * size, (i, got, want)


def test_rms_norm_of_many_rows():
    """The weight's gradient over more rows than one fp32 sum takes, and rows whose sum is all that matters."""
    for rows, C in ((70000, 32), (300000, 8), (3000, 512)):
        x, w = _randn(rows, C, seed=1), (1 + 0.1 * _randn(C, seed=2)).requires_grad_()
        dy = torch.rand(rows, C, device=DEV, generator=_gen(3))
        dw, = torch.autograd.grad(rms_norm(x.abs(), w), w, dy)
        t = x.abs().double()
        n = t * (t.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        want = (dy.double() * n).sum(0)
        _within(dw, want, 290 * U * want)
        assert torch.equal(dw, torch.autograd.grad(rms_norm(x.abs(), w), w, dy)[0])


def test_rms_norm_partial_uses():
    x, r = _randn(5, 64, seed=1).requires_grad_(), _randn(5, 64, seed=2).requires_grad_()
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, total = rms_norm(x, w, residual=r)
    g = torch.autograd.grad(total.sum(), [x, r, w], retain_graph=True)      # the norm's result is not used
    assert torch.equal(g[0], torch.ones_like(x)) and torch.equal(g[1], torch.ones_like(r)) and not g[2].any()
    gx, = torch.autograd.grad(y.sum(), [x], retain_graph=True)              # the sum is not used
    both = torch.autograd.grad([y.sum(), total.sum()], [x, r])
    assert float((both[0] - gx - 1).abs().max()) < 1e-5
    assert torch.equal(rms_norm(x.detach()), rms_norm(x.detach(), torch.ones(64, device=DEV)))
    h = _randn(5, 64, seed=3).requires_grad_()                              # one tensor on both sides
    y, total = rms_norm(h, w, residual=h)
    gh, = torch.autograd.grad(total.sum(), h)
    assert torch.equal(gh, torch.full_like(h, 2.0))


def test_rms_norm_types_and_layouts():
    x = _randn(4, 6, 80, seed=1)
    w = 1 + 0.1 * _randn(80, seed=2)
    want = rms_norm(x.reshape(24, 80), w).reshape(4, 6, 80)
    assert torch.equal(rms_norm(x, w), want)
    assert torch.equal(rms_norm(x[0, 0], w), want[0, 0])
    wide = torch.zeros(4, 6, 101, device=DEV)
    for off in (0, 1, 2, 4):
        wide[..., off:off + 80] = x
        v = wide[..., off:off + 80]
        assert float((rms_norm(v, w) - want).abs().max()) < 1e-6
        y, t = rms_norm(v, w, residual=v)
        assert torch.equal(t, 2 * x)
    assert torch.equal(rms_norm(x.transpose(0, 1), w), want.transpose(0, 1))
    b = rms_norm(x, w.bfloat16())
    assert torch.equal(b, rms_norm(x, w.bfloat16().float()))
    wb = w.bfloat16().requires_grad_()
    g, = torch.autograd.grad(rms_norm(x, wb).sum(), wb)
    assert g.dtype == BF16
    y, t = rms_norm(x.half(), w, residual=x)
    assert y.dtype == torch.float16 and t.dtype == F32
    y = rms_norm(x.half(), w)
    assert y.dtype == torch.float16


def test_rms_norm_special_values():
    inf, nan = float("inf"), float("nan")
    x = _randn(6, 40, seed=1)
    x[0] = 0.0
    x[1, 3] = nan
    x[2, 5] = inf
    x[3] = 1e-30
    y = rms_norm(x)
    assert not y[0].any()
    assert bool(y[1].isnan().all())
    assert bool(y[2, 5].isnan()) and not y[2, :5].any()
    _within(y[3], x[3].double() / 1e-5 ** 0.5, 27 * U * 1e-27)
    z = rms_norm(torch.zeros(2, 40, device=DEV), eps=0.0)
    assert bool(z.isnan().all())
    y8, scale = rms_norm_fp8(x)
    assert not y8[0].float().any() and float(scale[0]) == pytest.approx(1e-30 / 448, rel=1e-6)
    assert bool(y8[1].float().isnan().all())
    for b in range(4, 6):
        assert float(y8[b].float().abs().max()) == 448.0


# ---- 8 bits --------------------------------------------------------------------------------------------
def _check_rows8(y8, scale, y, err):
    """y8 * scale against y with its float32 error err (relative): half a step of e4m3, or a neighbour where y is that near
    to the border between two."""
    assert y8.dtype == torch.float8_e4m3fn and y8.shape == y.shape and (y8.shape[0] == 1 or y8.stride(0) % 16 == 0)
    top = y.abs().amax(-1)
    want = top.clamp_min(O.TINY) / 448
    _within(scale, want, (err + 2 * U) * want)
    v = y / want[:, None]
    half = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 4)
    _within(y8.double(), v, half * (1 + 1e-9) + (2 * err + 4 * U) * v.abs())


@pytest.mark.parametrize("xd,rd", [(F32, None), (BF16, None), (F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("rows,C", SHAPES)
def test_rms_norm_fp8(rows, C, xd, rd):
    x = _randn(rows, C, seed=1, dtype=xd)
    r = None if rd is None else (2 * _randn(rows, C, seed=2)).to(rd)
    w = 1 + 0.1 * _randn(C, seed=3)
    out = rms_norm_fp8(x, w, residual=r)
    total = x
    if r is not None:
        total = (x.float() + r.float()).to(torch.promote_types(xd, rd))
        assert torch.equal(out[2], total)
    y, _ = O.rms_norm(total.double(), w.double())
    _check_rows8(out[0], out[1], y, 27 * U)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize_fp8(dtype):
    for shape in ((1, 1), (40, 96), (3, 5, 331), (17,)):
        x = _randn(*shape, seed=1, dtype=dtype) * 1e-3
        x8, scale = quantize_fp8(x)
        assert x8.shape == x.shape and scale.shape == x.shape[:-1]
        _check_rows8(x8.reshape(-1, shape[-1]), scale.reshape(-1), x.double().reshape(-1, shape[-1]), 0.0)
    # every e4m3 value times a power of two is kept
    v = torch.arange(127, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    x8, scale = quantize_fp8(torch.stack([v, -v, v * 2.0 ** -40]).to(dtype))
    assert torch.equal(x8[0].float(), v) and torch.equal(x8[1].float(), -v) and torch.equal(x8[2].float(), v)
    assert scale.tolist() == [1.0, 1.0, 2.0 ** -40]


def _rows8(n, K, seed):
    x = _randn(n, K, seed=seed)
    x[:, 0] *= 30
    x8, s = quantize_fp8(x)
    return x8, s


@pytest.mark.parametrize("M,K,N", [(1, 256, 1024), (1, 1, 1), (16, 16, 16), (3, 100, 130), (17, 2560, 300), (33, 640, 128), (64, 2560, 1000),
                                   (65, 33, 257), (128, 5000, 129), (130, 256, 1024), (257, 384, 4000), (1000, 1024, 512), (4099, 300, 700),
                                   (5, 16384, 64), (2, 130, 40000)])
def test_linear_fp8(M, K, N):
    x8, xs = _rows8(M, K, 1)
    w8, ws = _rows8(N, K, 2)
    bias = _randn(N, seed=3)
    for dtype, b, act, res in ((F32, False, None, False), (F32, True, "silu", True), (BF16, True, None, True), (BF16, False, "silu", False)):
        r = _randn(M, N, seed=4, dtype=dtype) if res else None
        y = linear_fp8(x8, xs, w8, ws, bias=bias if b else None, activation=act, residual=r, dtype=dtype)
        assert y.dtype == dtype
        want, size, pre = O.linear(x8, xs, w8, ws, bias if b else None, act == "silu", r)
        bound = 1.1 * (-(-K // 32) + 64) * 2 * U * (size + (bias.abs() if b else 0.0)) + 2.0 ** -20 * pre.abs() + 2 * U * want.abs()
        _within(y, want, bound + HALF[dtype] * want.abs(), (dtype, b, act, res))
        assert torch.equal(y, linear_fp8(x8, xs, w8, ws, bias=bias if b else None, activation=act, residual=r, dtype=dtype))


def test_linear_fp8_exact_values():
    """Small whole numbers: every sum is exact, so every element has to be equal, in every form."""
    for M in (1, 20, 40, 100, 200, 600, 9000):
        for K, N in ((48, 200), (1024, 136)):
            x = torch.randint(-4, 5, (M, K), device=DEV, generator=_gen(M)).float()
            w = torch.randint(-4, 5, (N, K), device=DEV, generator=_gen(K)).float()
            one = torch.ones(1, device=DEV)
            y = linear_fp8(x.to(torch.float8_e4m3fn), one.expand(M), w.to(torch.float8_e4m3fn), one.expand(N), dtype=F32)
            assert torch.equal(y.double(), x.double() @ w.double().T), (M, K, N)


def test_linear_fp8_layouts():
    x8, xs = _rows8(30, 96, 1)
    w8, ws = _rows8(50, 96, 2)
    want = linear_fp8(x8, xs, w8, ws)
    assert want.dtype == BF16
    buf = torch.zeros(61, 200, device=DEV).to(torch.float8_e4m3fn)
    for rows, off in ((slice(0, 60, 2), 0), (slice(1, 61, 2), 16), (slice(0, 30), 7)):      # strided, shifted, unaligned
        buf[rows, off:off + 96] = x8
        assert torch.equal(linear_fp8(buf[rows, off:off + 96], xs, w8, ws), want)
    assert torch.equal(linear_fp8(x8.t().contiguous().t(), xs, w8.t().contiguous().t(), ws), want)
    assert torch.equal(linear_fp8(x8.unflatten(0, (5, 6)), xs.reshape(5, 6), w8, ws), want.reshape(5, 6, 50))
    assert torch.equal(linear_fp8(x8[3], xs[3], w8, ws), linear_fp8(x8[3:4], xs[3:4], w8, ws)[0])
    r = _randn(30, 120, seed=5)[:, 20:70]
    y = linear_fp8(x8, xs, w8, ws, residual=r)
    assert y.dtype == F32
    # the residual is added to the value that is stored without one, and the sum rounded: u of it (values reach 2000 here,
    # where a step is 1.2e-4)
    v = linear_fp8(x8, xs, w8, ws, dtype=F32).double() + r.double()
    _within(y, v, U * v.abs())
    one = linear_fp8(x8[:1], xs[:1], w8, ws)                    # a batch around a row does not reach it
    assert float((one.float() - want[:1].float()).abs().max()) <= 2.0 ** -7 * float(want[:1].float().abs().max())


def test_linear_fp8_non_finite():
    x8, xs = _rows8(20, 64, 1)
    w8, ws = _rows8(30, 64, 2)
    clean = linear_fp8(x8, xs, w8, ws)
    x8 = x8.clone()
    x8.view(torch.uint8)[4, 9] = 0x7f
    ws2 = ws.clone()
    ws2[7] = float("inf")
    y = linear_fp8(x8, xs, w8, ws2)
    assert bool(y[4].isnan().all()) and not bool(y[:4, 7].isfinite().any())
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[4], keep[:, 7] = False, False
    assert torch.equal(y[keep], clean[keep])


# ---- sampling ---------------------------------------------------------------------------------------------
def _sample_rows(logits, u, **kw):
    n = len(u)
    at = {k: v.tolist() if isinstance(v, torch.Tensor) else [v] * n for k, v in kw.items()}
    rows = logits.double()
    return [O.sample(rows[b], float(u[b].double()), **{k: v[b] for k, v in at.items()}) for b in range(n)]


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_p=0.9), dict(top_p=0.3, temperature=1.3),
            dict(min_p=0.1), dict(top_k=20, top_p=0.8, min_p=0.05, temperature=0.9), dict(top_p=1e-9), dict(top_k=10 ** 9), dict(min_p=1.0),
            dict(temperature=1e-6), dict(temperature=1e6, top_p=0.5)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (40, 256), (9, 1000), (7, 5003), (3, 50257), (2, 131072)])
def test_sample_tokens(B, V, dtype):
    logits = (2.5 * _randn(B, V, seed=V)).to(dtype)
    u = torch.rand(B, device=DEV, generator=_gen(B))
    for kw in SETTINGS:
        got = sample_tokens(logits, u, **kw)
        assert got.dtype == torch.int64 and got.tolist() == _sample_rows(logits, u, **kw), kw


def test_sample_settings_by_row():
    B, V = 64, 777
    logits, u = 2 * _randn(B, V, seed=1), torch.rand(B, device=DEV, generator=_gen(2))
    r = torch.rand(4, B, device=DEV, generator=_gen(3))
    kw = dict(temperature=(2 * r[0]).double() * (r[0] > 0.1), top_k=(100 * r[1]).long(), top_p=r[2].double().clamp_min(0.01), min_p=0.2 * r[3].double())
    assert sample_tokens(logits, u, **kw).tolist() == _sample_rows(logits, u, **kw)
    single = dict(kw, temperature=kw["temperature"].float(), top_k=kw["top_k"].int(), min_p=kw["min_p"].float())
    want = {**single, "temperature": single["temperature"].double(), "min_p": single["min_p"].double()}
    assert sample_tokens(logits, u, **single).tolist() == _sample_rows(logits, u, **want)


def test_sample_every_border():
    """Uniform numbers at and next to the borders of equal weights: whole numbers decide."""
    V = 8
    logits = torch.zeros(17, V, device=DEV)
    u = torch.arange(17, device=DEV).float() / 16
    assert sample_tokens(logits, u).tolist() == [min(int(b / 2), V - 1) for b in range(17)]
    assert sample_tokens(logits, u, top_p=0.5).tolist() == [min(b // 4, 3) for b in range(17)]
    assert sample_tokens(logits, u, top_k=4).tolist() == [min(b // 4, 3) for b in range(17)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [300, 60000])
def test_sample_ties_and_masks(V, dtype):
    """Ties by the thousand, masked tokens as -inf and as the type's lowest value, one logit far above."""
    B = 6
    u = torch.rand(B, device=DEV, generator=_gen(1))
    coarse = _randn(B, V, seed=2).mul(2).round().to(dtype)
    masked = (2 * _randn(B, V, seed=3)).to(dtype)
    hide = torch.rand(B, V, device=DEV, generator=_gen(4)) < 0.7
    hide[:, 5] = False
    lowest = masked.masked_fill(hide, torch.finfo(dtype).min)
    inf = masked.masked_fill(hide, float("-inf"))
    peak = masked.clone()
    peak[:, 3] = 1000.0
    for logits in (coarse, torch.zeros_like(coarse), torch.full_like(coarse, torch.finfo(dtype).min), lowest, inf, peak, -coarse * 0.0):
        for kw in (dict(), dict(top_k=17), dict(top_k=V - 10), dict(top_p=0.7), dict(top_k=V // 2, top_p=0.5), dict(top_p=0.999, min_p=0.01)):
            assert sample_tokens(logits, u, **kw).tolist() == _sample_rows(logits, u, **kw), kw


def test_sample_special_rows():
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[-inf, -inf, -inf, -inf], [0.0, nan, 1.0, 2.0], [inf, 0.0, inf, 1.0], [-inf, 3.0, -inf, -inf], [1.0, 2.0, 2.0, 0.0],
                         [nan, nan, nan, nan], [-0.0, 0.0, -0.0, 0.0]], device=DEV)
    u = torch.tensor([0.5, 0.5, 0.6, 0.9, 0.1, 0.5, 0.3], device=DEV)
    assert sample_tokens(rows, u).tolist()[:4] == [-1, -1, 2, 1]
    assert sample_tokens(rows, u, temperature=0.0).tolist() == [-1, -1, 0, 1, 1, -1, 0]
    assert sample_tokens(rows, u, top_k=1).tolist() == [-1, -1, 0, 1, 1, -1, 0]
    assert sample_tokens(rows, u).tolist()[6] == 1
    t = torch.tensor([1.0, 1.0, nan, 1.0, inf, 1.0, 1e-300], device=DEV, dtype=torch.float64)
    got = sample_tokens(rows, u, temperature=t).tolist()
    assert got[2] == -1 and got[4] == 0 and got[6] == 1
    odd = torch.tensor([nan, 2.0, -1.0, 1.0, 0.0, 0.99999994, 0.5], device=DEV)     # numbers outside [0, 1)
    flat = torch.zeros(7, 4, device=DEV)
    assert sample_tokens(flat, odd).tolist() == [0, 3, 0, 3, 0, 3, 2]


@pytest.mark.parametrize("B,V", [(6, 3000), (300, 30000), (6, 400000)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sample_special_rows_of_many_tokens(B, V, dtype):
    """Rows shared by CTAs, by one, and read again instead of kept: infinities, NaN, nothing left, one left, ties, settings at
    their ends."""
    inf = float("inf")
    logits = (2 * _randn(B, V, seed=1)).to(dtype)
    u = torch.rand(B, device=DEV, generator=_gen(2))
    logits[0, [7, V // 2, V - 1]] = inf
    logits[1] = -inf
    logits[2, V - 2] = float("nan")
    logits[3] = -inf
    logits[3, V - 3] = -5.0
    logits[4] = logits[4].round()
    want = None
    for kw in (dict(), dict(top_k=2), dict(top_k=700), dict(top_p=0.9), dict(top_p=0.5, top_k=2000, min_p=0.01), dict(temperature=1e-30, top_p=0.7),
               dict(temperature=1e30, top_p=0.7), dict(temperature=inf, top_k=5), dict(temperature=0.0)):
        got = sample_tokens(logits, u, **kw).tolist()
        rows = list(range(6)) + list(range(6, B, 37))
        want = [_sample_rows(logits[b:b + 1], u[b:b + 1], **kw)[0] for b in rows]
        assert [got[b] for b in rows] == want, kw
    assert want[:4] == [7, -1, -1, V - 3]


def test_sample_layouts():
    wide = _randn(9, 1003, seed=1)
    u = torch.rand(9, device=DEV, generator=_gen(2))
    for v in (wide[:, 1:900], wide[::2, 3:], wide.t()[:9, :9]):
        n = len(v)
        assert sample_tokens(v, u[:n], top_p=0.9).tolist() == sample_tokens(v.contiguous(), u[:n], top_p=0.9).tolist()
    assert sample_tokens(wide.half(), u).tolist() == sample_tokens(wide.half().float(), u).tolist()
    same = sample_tokens(wide, u, top_k=50)                    # a row does not depend on the batch around it
    assert [int(sample_tokens(wide[b:b + 1], u[b:b + 1], top_k=50)) for b in range(9)] == same.tolist()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,V", [(3, 5003), (3, 50257), (3, 131072), (200, 131072), (3, 300001), (2, 1 << 20)])
def test_sample_borders_of_dense_rows(B, V, dtype):
    """The border itself: rows in rising order drawn at 0 give the first token by index, the lowest that is kept; falling ones, just
    below 1, the last.  Borders fall where few tokens are and where thousands share a value.

    A weight is cut down to a whole number of 2^-42 of the largest, the largest itself whole, so a sum of V of them, or the place T
    that is drawn, is short by less than E = V 2^-42 and never long.  With R a running sum, R[want - 1] <= T < R[want], and the same
    of got in whole numbers: what lies between the two tokens weighs less than E; the border of top_p, a place in such sums
    too, adds as much."""
    rows = [0, 1, B - 1]
    for width in (0.3, 1.0, 3.0, 5.0):
        up = (width * _randn(B, V, seed=V)).to(dtype).sort(-1).values
        for logits, at in ((up, 0.0), (up.flip(-1).contiguous(), 1 - 2.0 ** -24)):
            u = torch.full((B,), at, device=DEV)
            for kw in (dict(top_p=0.5), dict(top_p=0.9), dict(top_p=0.95), dict(top_p=0.999), dict(top_k=V // 2), dict(top_k=3000, top_p=0.95),
                       dict(top_p=0.95, temperature=0.6)):
                got = sample_tokens(logits, u, **kw).tolist()
                for b in rows:
                    want = _sample_rows(logits[b:b + 1], u[b:b + 1], **kw)[0]
                    l = logits[b].double()
                    between = torch.exp((l[min(got[b], want) + 1:max(got[b], want)] - l.max()) / kw.get("temperature", 1.0))
                    assert got[b] == want or float(between.sum()) < 2 * V * 2.0 ** -42, (width, at, kw, got[b], want)


def test_sample_the_largest_vocabulary():
    V = 1 << 20
    logits = 3 * _randn(2, V, seed=1)
    u = torch.rand(2, device=DEV, generator=_gen(2))
    for kw in (dict(), dict(top_p=0.95), dict(top_k=1000)):
        assert sample_tokens(logits, u, **kw).tolist() == _sample_rows(logits, u, **kw)
    with pytest.raises(ValueError, match="at most"):
        sample_tokens(torch.zeros(1, V + 1, device=DEV), u[:1])


# ---- streams, graphs, devices -----------------------------------------------------------------------------
def _chain(idx, W, w, p8, ps, u):
    h = embedding(idx, W, 2.0)
    y8, scale, total = rms_norm_fp8(h, w, residual=h)
    logits = linear_fp8(y8, scale, p8, ps, dtype=F32)
    return sample_tokens(logits, u, temperature=0.8, top_k=40, top_p=0.9), total, logits


@pytest.mark.parametrize("tokens", [1, 17, 64, 200])
def test_parameters_written_just_before(tokens):
    """A weight that the kernel right before writes, into the memory of the last one: what is fetched early is not used stale."""
    x8, xs = _rows8(tokens, 640, 1)
    x = _randn(tokens, 640, seed=2)
    tables = [_randn(512, 640, seed=3 + i) * (1 + i) for i in range(4)]
    first = torch.zeros(1, dtype=torch.int64, device=DEV)
    own = [quantize_fp8(t) for t in tables]
    torch.cuda.synchronize()
    products = [linear_fp8(x8, xs, *o) for o in own]
    norms = [rms_norm(x, t[0].clone()) for t in tables]
    places = set()
    for turn in range(40):
        i = turn % 4
        w8, ws = quantize_fp8(tables[i])
        y = linear_fp8(x8, xs, w8, ws)
        places.add(w8.data_ptr())
        z = rms_norm(x, embedding(first, tables[i])[0])
        assert torch.equal(y, products[i]) and torch.equal(z, norms[i]), turn
        del w8, ws
    assert len(places) < 40                                     # the memory did come again


def test_two_streams_at_once():
    """Kernels that are launched early, on two streams: products of every form share the SMs' tensor memory with those that wait."""
    rows = {n: _rows8(n, 640, n) for n in (1, 20, 64, 130, 700, 5000)}
    w8, ws = _rows8(640, 640, 9)
    wide8, wides = _rows8(3000, 640, 10)
    g = 1 + 0.1 * _randn(640, seed=11)
    u = torch.rand(64, device=DEV, generator=_gen(12))

    def run(sizes):
        out = []
        for n in sizes:
            h = linear_fp8(*rows[n], w8, ws, dtype=BF16)
            q, scale = rms_norm_fp8(h, g)
            logits = linear_fp8(q, scale, wide8, wides, dtype=BF16)
            out += [h, logits, sample_tokens(logits[:64], u[:min(n, 64)], top_k=30, top_p=0.9)]
        return out

    orders = [(1, 5000, 64, 20, 700, 130), (700, 1, 130, 5000, 20, 64)]
    want = [run(order) for order in orders]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(orders[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))


def test_graph_and_stream():
    """The operators after one another, captured with two graphs alive, and on a stream of their own."""
    W, w = _randn(500, 96, seed=1), 1 + 0.1 * _randn(96, seed=2)
    p8, ps = _rows8(500, 96, 3)
    idx = [torch.randint(0, 500, (6,), device=DEV, generator=_gen(i)) for i in range(2)]
    u = torch.rand(6, device=DEV, generator=_gen(9))
    want = [[t.clone() for t in _chain(i, W, w, p8, ps, u)] for i in idx]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _chain(idx[0], W, w, p8, ps, u)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graphs, outs = [], []
    for i in idx:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_chain(i, W, w, p8, ps, u))
        graphs.append(g)
    for g in (0, 1, 1, 0):
        graphs[g].replay()
    for o, r in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, r))


def test_training_graph():
    """Forward and backward of embedding and norm captured as one graph."""
    W, w = _randn(60, 64, seed=1).requires_grad_(), torch.ones(64, device=DEV, requires_grad=True)
    idx = torch.randint(0, 60, (200,), device=DEV, generator=_gen(0))

    def step():
        h = embedding(idx, W)
        y, total = rms_norm(h.sin(), w, residual=h)
        return torch.autograd.grad((y * total).sum(), [W, w])

    want = [g.clone() for g in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        g.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_far_offsets():
    """Rows beyond 2^31 elements of a table, of logits and of a normed tensor."""
    big = torch.zeros((1 << 31) // 4096 + 64, 4096, device=DEV, dtype=BF16)
    last = len(big) - 1
    big[last] = _randn(4096, seed=1, dtype=BF16)
    assert torch.equal(embedding(torch.tensor([last], device=DEV), big)[0], big[last])
    y = rms_norm(big, torch.ones(4096, device=DEV))
    want, _ = O.rms_norm(big[last].double())
    _within(y[last], want, (27 * U + HALF[BF16]) * want.abs())
    del y
    u = torch.full((len(big),), 0.37, device=DEV)
    got = sample_tokens(big, u)
    assert int(got[last]) == O.sample(big[last].double(), float(u[0].double()))


# ---- refusals -------------------------------------------------------------------------------------------
def test_what_autograd_does_not_have():
    x = _randn(4, 32, seed=1).requires_grad_()
    for fn in (rms_norm_fp8, quantize_fp8):
        with pytest.raises(RuntimeError, match="no gradient"):
            fn(x)
        with torch.no_grad():
            fn(x)
    W = _randn(9, 8).requires_grad_()
    idx = torch.arange(4, device=DEV)
    with pytest.raises(RuntimeError, match="once"):
        g, = torch.autograd.grad(embedding(idx, W).square().sum(), W, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(rms_norm(x).square().sum(), x, create_graph=True)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = fw.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            rms_norm(dual)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda t: rms_norm(t), x.detach())


def test_two_devices_are_refused():
    x, W = _randn(4, 32), _randn(9, 32)
    cpu = torch.zeros(32)
    for call in (lambda: embedding(torch.zeros(3, dtype=torch.long), W), lambda: rms_norm(x, cpu), lambda: rms_norm(x, residual=x.cpu()),
                 lambda: sample_tokens(x, torch.zeros(4)), lambda: sample_tokens(x, x[:, 0].abs().contiguous(), top_k=torch.ones(4).long())):
        with pytest.raises(ValueError, match="one device"):
            call()
