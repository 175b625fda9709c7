"""RMSNorm and TokenEmbedding as modules of any torch program: scripted, traced, exported, compiled, differentiated in forward mode, through
torch.func and more than once, on the CPU and where their kernels run."""

import warnings

import pytest
import torch
import torch.nn.functional as F

from mamba_ssm_benchmark_b200.mixer import RMSNorm, TokenEmbedding

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
pytestmark = [pytest.mark.filterwarnings("ignore"), pytest.mark.parametrize("dev", DEVICES)]


def _cases(dev):
    """(module, its input, the same as torch's own operators)."""
    g = torch.Generator(device=dev).manual_seed(0)
    n, e = RMSNorm(16).to(dev), TokenEmbedding(9, 8).to(dev)
    with torch.no_grad():
        n.weight += 0.1 * torch.randn(16, device=dev, generator=g)
    x, idx = torch.randn(2, 3, 16, device=dev, generator=g), torch.randint(0, 9, (4, 5), device=dev, generator=g)
    return [(n, x, lambda x, w: F.rms_norm(x, (16,), eps=1e-5) * w), (e, idx, lambda i, w: F.embedding(i, w))]


def _near(a, b, tol=1e-6):
    """float32 of at most 20 terms: 2^-24 each, at most 1e-6 of the norm and 1e-5 where squares of them are."""
    return a.shape == b.shape and a.dtype == b.dtype and float((a.double() - b.double()).norm()) <= tol * float(b.double().norm()) + 1e-30


def test_scripts_traces_and_exports(dev):
    for m, x, f in _cases(dev):
        want = f(x, m.weight)
        other = x.flip(0)
        for make in (lambda: torch.jit.script(m), lambda: torch.jit.trace(m, x), lambda: torch.compile(m, fullgraph=True, backend="eager"),
                     lambda: torch.export.export(m, (x,)).module()):
            with warnings.catch_warnings():
                warnings.simplefilter("ignore")
                made = make()
            assert _near(made(x), want) and _near(made(other), f(other, m.weight))
        assert _near(m(x), want)


def test_derivatives_of_any_kind(dev):
    for m, x, f in _cases(dev):
        w, dw = m.weight.detach(), torch.randn_like(m.weight)
        run = lambda w: torch.func.functional_call(m, {"weight": w}, (x,))
        ref = lambda w: f(x, w)
        loss = lambda g: lambda w: g(w).square().sum()
        for a, b in zip(torch.func.jvp(run, (w,), (dw,)), torch.func.jvp(ref, (w,), (dw,))):
            assert _near(a, b)
        assert _near(torch.func.grad(loss(run))(w), torch.func.grad(loss(ref))(w), 1e-5)
        assert _near(torch.func.vmap(m)(x), f(x, w))
        assert _near(torch.func.hessian(loss(run))(w), torch.func.hessian(loss(ref))(w), 1e-5)
    n, x, f = _cases(dev)[0]
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        a, b = fw.unpack_dual(n(dual)), fw.unpack_dual(f(dual, n.weight))
        assert _near(a.primal, b.primal) and _near(a.tangent, b.tangent, 1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_differentiated_three_times(dev, dtype):
    """Gradients of gradients of gradients against torch's own operators in float64: 1e-5 of the norm in float32; in bf16 every
    gradient that comes between is rounded, 2^-8 a step at random, six of them at most."""
    tol = 1e-5 if dtype == torch.float32 else 6 * 2.0 ** -8
    for m, x, f in _cases(dev):
        m = m.to(dtype)
        x = x.to(dtype) if x.is_floating_point() else x
        results = []
        for own in (True, False):
            w = m.weight if own else m.weight.detach().double().requires_grad_()
            xs = x.detach().clone() if own else (x.double() if x.is_floating_point() else x)
            leaves = [w] + ([xs.requires_grad_()] if xs.is_floating_point() else [])
            y = m(xs) if own else f(xs, w)
            out, value = [y], y.double().pow(3).sum()
            for turn in range(3):
                grads = torch.autograd.grad(value, leaves, create_graph=True)
                out += grads
                value = sum(d.double().pow(2).sum() for d in grads)
            results.append(out)
        for k, (a, b) in enumerate(zip(*results)):
            assert a.dtype == dtype and _near(a.double(), b, tol * (1 + k)), (k, type(m).__name__)


def test_subclasses_of_tensors(dev):
    class Tagged(torch.Tensor):
        pass

    for m, x, f in _cases(dev):
        y = m(x.as_subclass(Tagged))
        assert type(y) is Tagged and _near(y.as_subclass(torch.Tensor), f(x, m.weight))


def test_the_sum_and_its_norm_are_differentiated_twice(dev):
    """RMSNorm.add of one and of two types, as of x + residual and the norm of it."""
    if dev == "cpu":
        pytest.skip("the kernels add")
    n, x, f = _cases(dev)[0]
    for rd in (torch.float32, torch.bfloat16):
        r = torch.randn_like(x).to(rd)
        res = []
        for own in (True, False):
            a, b = (t.detach().clone().requires_grad_() for t in (x, r))
            y, total = n.add(a, b) if own else (n(a + b), a + b)
            g = torch.autograd.grad(y.pow(3).sum() + total.pow(2).sum(), [a, b, n.weight], create_graph=True)
            h = torch.autograd.grad(sum(t.float().pow(2).sum() for t in g), [a, b, n.weight])
            only = torch.autograd.grad(n.add(a, b)[1].pow(3).sum(), [a, b], create_graph=True)
            res.append([*g, *h, *torch.autograd.grad(only[0].sum() + only[1].float().sum(), [a, b])])
        for k, (p, q) in enumerate(zip(*res)):
            assert _near(p, q, 1e-5 if rd == torch.float32 else 6 * 2.0 ** -8), (rd, k)


def test_weights_that_broadcast_and_no_eps(dev):
    """What torch's form knows and the kernels do not."""
    x = torch.randn(2, 3, 16, device=dev)
    one, heads, none = RMSNorm(1).to(dev), RMSNorm(16).to(dev), RMSNorm(16, eps=None).to(dev)
    with torch.no_grad():
        one.weight.fill_(3.0)
    heads.weight = torch.nn.Parameter(torch.randn(3, 16, device=dev))
    n = F.rms_norm(x, (16,), eps=1e-5)
    assert _near(one(x), 3 * n) and _near(heads(x), n * heads.weight) and _near(none(x), F.rms_norm(x, (16,)))
    with torch.inference_mode():
        assert _near(RMSNorm(16).to(dev)(x), n)
