"""GPU parity of the gated delta rule (ssm_gated_delta_fwd / _bwd / _state_update) against its definition in
float64 (oracle/delta_oracle.py).

Tolerances, on ||difference|| / ||reference|| (2-norms), from the arithmetic:
    F32_TOL   a result passes about six products of at most 128 terms; tensor-core sums truncate at 2^-23 and a
              sum of three-piece products has at most 24 of them: 6 * 24 * 2^-23 = 1.7e-5, taken as 2e-5
    BF16_TOL  one rounding to bf16 (8 bits: at most 2^-8 of each element) over results that are kept to 16 bits:
              2^-8 + 2e-4
"""

import pytest
import torch

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import gated_delta_rule, gated_delta_state_update
from oracle import delta_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32_TOL = 2e-5
BF16_TOL = 2.0 ** -8 + 2e-4
NAMES = ("q", "k", "v", "g", "beta", "h0")


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert nat.read_device_error() == 0


def _inputs(B, L, Hk, Hv, dk, dv, dtype=torch.float32, h0=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    t = {"q": unit(randn(B, L, Hk, dk)).to(dtype), "k": unit(randn(B, L, Hk, dk) + 0.5).to(dtype),
         "v": randn(B, L, Hv, dv).to(dtype), "g": -torch.exp(randn(B, L, Hv) - 2.0),
         "beta": torch.sigmoid(randn(B, L, Hv)), "h0": randn(B, Hv, dk, dv) if h0 else None}
    return t, randn(B, L, Hv, dv).to(dtype), randn(B, Hv, dk, dv)


def _run(fn, t, do, dlast, cast):
    leaves = {n: None if x is None else cast(x).detach().clone().requires_grad_() for n, x in t.items()}
    o, last = fn(**leaves)
    names = [n for n in NAMES if leaves[n] is not None]
    grads = torch.autograd.grad([o, last], [leaves[n] for n in names], [cast(do), cast(dlast)])
    return {"o": o.detach(), "last": last.detach(), **{"d" + n: x for n, x in zip(names, grads)}}


def _err(a, b):
    b = b.double()
    return float((a.cpu().double() - b).norm() / b.norm().clamp_min(1e-300))


def _compare(got, want):
    for n, w in want.items():
        assert got[n].shape == w.shape, n
        tol = BF16_TOL if got[n].dtype == torch.bfloat16 else F32_TOL
        assert _err(got[n], w) <= tol, (n, _err(got[n], w), tol)


SHAPES = [
    (1, 1, 1, 1, 64, 64), (2, 2, 1, 2, 16, 8), (1, 63, 2, 2, 64, 48), (2, 64, 2, 4, 32, 16), (1, 65, 1, 3, 128, 33),
    (2, 130, 2, 2, 17, 80), (1, 200, 2, 4, 65, 17), (3, 129, 1, 1, 1, 1), (1, 96, 2, 2, 128, 160), (1, 320, 1, 1, 100, 7),
    # enough heads to fill the GPU
    (5, 70, 4, 8, 64, 64), (3, 200, 8, 16, 100, 80), (2, 65, 5, 10, 128, 160), (20, 33, 4, 8, 16, 16), (40, 130, 2, 4, 48, 33),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("h0", [True, False])
def test_forward_and_gradients(shape, dtype, h0):
    t, do, dlast = _inputs(*shape, dtype=dtype, h0=h0, seed=sum(shape))
    got = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
    want = _run(O.gated_delta_rule, t, do, dlast, lambda x: x.double())
    assert got["o"].dtype == dtype and got["last"].dtype == torch.float32 and got["dq"].dtype == dtype
    _compare(got, want)
    with torch.no_grad():      # the inference path, which saves nothing
        o, last = gated_delta_rule(**{n: None if x is None else x.to(DEV) for n, x in t.items()})
    assert torch.equal(o, got["o"]) and torch.equal(last, got["last"])


@pytest.mark.parametrize("shape", [(10, 260, 4, 8, 128, 16), (30, 70, 3, 6, 40, 24), (12, 200, 6, 6, 128, 65),
                                   (8, 250, 5, 10, 64, 144)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_several_chunks_per_sm(shape, dtype):
    """More chunks than the GPU has SMs, of one to nine slabs of 16 channels each; the same again, bit by bit."""
    t, do, dlast = _inputs(*shape, dtype=dtype, seed=sum(shape))
    got = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
    _compare(got, _run(O.gated_delta_rule, t, do, dlast, lambda x: x.double()))
    for _ in range(3):
        again = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
        for n, x in got.items():
            assert torch.equal(again[n], x), n


def test_gradients_against_differences():
    """<grad, d> against central differences of the float64 definition along random directions d: with steps of 1e-5
    the difference quotient is exact to about 1e-9 of the terms' size."""
    t, do, dlast = _inputs(1, 70, 1, 2, 24, 12, seed=5)
    got = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
    gen = torch.Generator().manual_seed(9)

    def loss(x):
        o, last = O.gated_delta_rule(**x)
        return float((o * do.double()).sum() + (last * dlast.double()).sum())

    base = {n: x.double() for n, x in t.items()}
    for n in NAMES:
        d = torch.randn(t[n].shape, generator=gen, dtype=torch.float64)
        lo, hi = ({**base, n: base[n] + s * 1e-5 * d} for s in (-1, 1))
        want = (loss(hi) - loss(lo)) / 2e-5
        have = float((got["d" + n].cpu().double() * d).sum())
        size = float(got["d" + n].cpu().double().norm() * d.norm())
        assert abs(have - want) <= F32_TOL * size, n


def test_reset_by_infinite_decay():
    """g = -inf forgets everything before: the same as separate sequences, forward and backward, with no NaN."""
    L1, L2 = 50, 83
    t, do, dlast = _inputs(1, L1 + L2, 1, 2, 32, 24, h0=False, seed=3)
    t["g"][:, L1] = float("-inf")
    got = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
    halves = []
    for sl, dl in ((slice(0, L1), torch.zeros_like(dlast)), (slice(L1, None), dlast)):
        part = {n: None if x is None else x[:, sl].clone() for n, x in t.items()}
        part["g"] = part["g"].masked_fill(torch.isinf(part["g"]), 0.0)
        halves.append(_run(O.gated_delta_rule, part, do[:, sl], dl, lambda x: x.double()))
    for n in ("o", "dq", "dk", "dv", "dbeta"):
        assert _err(got[n], torch.cat([h[n] for h in halves], 1)) <= F32_TOL, n
    dg = torch.cat([h["dg"] for h in halves], 1)
    dg[:, L1] = 0.0
    assert _err(got["dg"], dg) <= F32_TOL
    assert _err(got["last"], halves[1]["last"]) <= F32_TOL


@pytest.mark.parametrize("beta", [0.0, 1.0, 2.0])
def test_constant_beta(beta):
    """beta = 0 writes nothing (and still has a gradient); beta = 2 reflects."""
    t, do, dlast = _inputs(2, 100, 1, 1, 16, 16, seed=4)
    t["beta"] = torch.full_like(t["beta"], beta)
    _compare(_run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV)),
             _run(O.gated_delta_rule, t, do, dlast, lambda x: x.double()))


def test_repeated_keys():
    """One key at every position with beta = 1 and no decay: the triangular system at its worst condition."""
    t, do, dlast = _inputs(1, 128, 1, 1, 64, 32, seed=6)
    t["k"] = t["k"][:, :1].expand_as(t["k"]).contiguous()
    t["g"] = torch.zeros_like(t["g"])
    t["beta"] = torch.ones_like(t["beta"])
    _compare(_run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV)),
             _run(O.gated_delta_rule, t, do, dlast, lambda x: x.double()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    """q, k, v as slices of one projection at an odd offset, (B, H, L, d) storage, gates as columns, a strided
    gradient: bitwise the results of dense copies."""
    B, L, H, d = 2, 90, 2, 40
    t, do, dlast = _inputs(B, L, H, H, d, d, dtype=dtype, seed=8)
    dense = {n: x.to(DEV) for n, x in t.items()}
    pack = torch.zeros(B, L, 3 * H * d + 5, dtype=dtype, device=DEV)
    odd = dict(dense)
    for i, n in enumerate("qkv"):
        view = pack[..., 3 + i * H * d:3 + (i + 1) * H * d].unflatten(-1, (H, d))
        view.copy_(dense[n])
        odd[n] = view
    odd["q"] = dense["q"].transpose(1, 2).contiguous().transpose(1, 2)
    gates = torch.stack([dense["g"], dense["beta"]], -1)
    odd["g"], odd["beta"] = gates[..., 0], gates[..., 1]
    do_t = do.to(DEV).permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
    a = _run(gated_delta_rule, dense, do.to(DEV), dlast.to(DEV), lambda x: x)
    leaves = {n: x.detach().requires_grad_() for n, x in odd.items()}
    assert leaves["v"].data_ptr() % 16 != 0
    o, last = gated_delta_rule(**leaves)
    grads = torch.autograd.grad([o, last], [leaves[n] for n in NAMES], [do_t, dlast.to(DEV)])
    assert torch.equal(o, a["o"]) and torch.equal(last, a["last"])
    for n, x in zip(NAMES, grads):
        assert torch.equal(x, a["d" + n]), n


def test_mixed_types_are_promoted():
    t, *_ = _inputs(1, 40, 1, 1, 16, 16, seed=2)
    t = {n: x.to(DEV) for n, x in t.items()}
    o, last = gated_delta_rule(t["q"].bfloat16(), t["k"], t["v"], t["g"].bfloat16(), t["beta"], t["h0"])
    o2, last2 = gated_delta_rule(t["q"].bfloat16().float(), t["k"], t["v"], t["g"].bfloat16().float(), t["beta"], t["h0"])
    assert o.dtype == torch.float32 and torch.equal(o, o2) and torch.equal(last, last2)


def test_continuation_determinism_and_streams():
    """A sequence in two calls equals one call to rounding; repeated calls and calls on another stream are equal bitwise."""
    t, do, dlast = _inputs(2, 1000, 2, 4, 64, 64, dtype=torch.bfloat16, seed=12)
    d = {n: x.to(DEV) for n, x in t.items()}
    o, last = gated_delta_rule(**d)
    cut = 333
    part = lambda sl, h0: gated_delta_rule(*(d[n][:, sl] for n in NAMES[:5]), h0=h0)
    o1, mid = part(slice(0, cut), d["h0"])
    o2, last2 = part(slice(cut, None), mid)
    assert _err(last2, last.cpu()) <= F32_TOL
    assert _err(torch.cat([o1, o2], 1), o.cpu().double()) <= 2 * BF16_TOL
    a = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(gated_delta_rule, t, do, dlast, lambda x: x.to(DEV))
    torch.cuda.current_stream().wait_stream(side)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_offsets_beyond_32_bits():
    """A batch stride above 2^31 elements."""
    t, do, dlast = _inputs(2, 20, 1, 1, 16, 16, dtype=torch.bfloat16, seed=14)
    big = torch.empty(2 ** 31 + 64 * 1024, dtype=torch.bfloat16, device=DEV)
    v = big.as_strided((2, 20, 1, 16), (2 ** 31 + 8, 16, 16, 1))
    v.copy_(t["v"])
    d = {n: x.to(DEV) for n, x in t.items()}
    want = gated_delta_rule(**d)
    got = gated_delta_rule(**{**d, "v": v})
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("shape", [(1, 1, 1, 16, 16), (3, 2, 4, 64, 64), (2, 1, 3, 128, 33), (2, 2, 2, 17, 130),
                                   (64, 1, 1, 1, 1), (2, 3, 3, 100, 257)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_state_update(shape, dtype):
    B, Hk, Hv, dk, dv = shape
    steps = 3
    t, *_ = _inputs(B, steps, Hk, Hv, dk, dv, dtype=dtype, seed=sum(shape))
    want_o, want_s = O.gated_delta_rule(**{n: x.double() for n, x in t.items()})
    d = {n: x.to(DEV) for n, x in t.items()}
    state = d["h0"].clone()
    for i in range(steps):
        args = [d[n][:, i] for n in NAMES[:5]]
        if i == 1:
            out = torch.empty(B, Hv, dv, dtype=dtype, device=DEV)
            assert gated_delta_state_update(state, *args, out=out) is out
        else:
            out = gated_delta_state_update(state, *args)
        assert out.dtype == dtype
        assert _err(out, want_o[:, i]) <= (BF16_TOL if dtype == torch.bfloat16 else F32_TOL)
    assert _err(state, want_s) <= F32_TOL


def test_state_update_resets_and_replays_in_a_graph():
    t, *_ = _inputs(2, 1, 2, 2, 32, 32, seed=20)
    d = {n: x.to(DEV) for n, x in t.items()}
    args = [d[n][:, 0].clone() for n in NAMES[:5]]
    state = d["h0"].clone()
    gated_delta_state_update(state, *args)                       # warm-up before the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = gated_delta_state_update(state, *args)
    state.copy_(d["h0"])
    args[3].fill_(float("-inf"))                                 # the state is forgotten
    graph.replay()
    want_o, want_s = O.gated_delta_rule(*(x.double().cpu().unsqueeze(1) for x in args[:3]),
                                        torch.zeros(2, 1, 2, dtype=torch.float64), args[4].double().cpu().unsqueeze(1))
    assert _err(o, want_o[:, 0]) <= F32_TOL and _err(state, want_s) <= F32_TOL


def test_partial_gradients():
    """A loss on o alone, or on the last state alone, and inputs that want no gradient."""
    t, do, dlast = _inputs(1, 70, 1, 2, 32, 16, seed=15)
    for which, dout in (("o", do), ("last", dlast)):
        lv = {n: x.to(DEV).requires_grad_(n in ("k", "g")) for n, x in t.items()}
        got = torch.autograd.grad(gated_delta_rule(**lv)[which == "last"], [lv["k"], lv["g"]], dout.to(DEV))
        rv = {n: x.double().requires_grad_() for n, x in t.items()}
        want = torch.autograd.grad(O.gated_delta_rule(**rv)[which == "last"], [rv["k"], rv["g"]], dout.double())
        for a, b in zip(got, want):
            assert _err(a, b) <= F32_TOL, which


def test_second_derivatives_are_refused():
    t, do, _ = _inputs(1, 8, 1, 1, 16, 16, seed=1)
    lv = {n: x.to(DEV).requires_grad_() for n, x in t.items()}
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(gated_delta_rule(**lv)[0], lv["k"], do.to(DEV), create_graph=True)


def test_refusals():
    t, *_ = _inputs(1, 8, 1, 2, 16, 16, seed=1)
    d = {n: x.to(DEV) for n, x in t.items()}
    bad = lambda **kw: gated_delta_rule(**{**d, **kw})
    with pytest.raises(ValueError, match="equal shape"):
        bad(k=d["k"][:, :4])
    with pytest.raises(ValueError, match="multiple"):
        bad(q=d["q"].repeat(1, 1, 3, 1), k=d["k"].repeat(1, 1, 3, 1))
    with pytest.raises(ValueError, match="key width"):
        bad(q=torch.zeros(1, 8, 1, 129, device=DEV), k=torch.zeros(1, 8, 1, 129, device=DEV), h0=None)
    with pytest.raises(ValueError, match="empty"):
        bad(q=d["q"][:, :0], k=d["k"][:, :0], v=d["v"][:, :0], g=d["g"][:, :0], beta=d["beta"][:, :0])
    with pytest.raises(ValueError, match="g and beta must"):
        bad(g=d["g"][..., 0])
    with pytest.raises(ValueError, match="h0 must"):
        bad(h0=d["h0"].transpose(0, 1))
    with pytest.raises(TypeError, match="float64"):
        bad(v=d["v"].double())
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_delta_rule(**t)
    with pytest.raises(ValueError, match="one device"):
        bad(g=t["g"])
    step = lambda state, **kw: gated_delta_state_update(state, *({**d, **kw}[n][:, 0] for n in NAMES[:5]))
    with pytest.raises(ValueError, match="contiguous"):
        step(d["h0"].transpose(2, 3))
    with pytest.raises(ValueError, match="contiguous"):
        step(d["h0"].bfloat16())
    with pytest.raises(ValueError, match="out must"):
        gated_delta_state_update(d["h0"], *(d[n][:, 0] for n in NAMES[:5]), out=torch.empty(1, 2, 15, device=DEV))
