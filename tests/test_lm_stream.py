"""What the LM's fused residual stream and 8-bit path leave to the modules that stand in them: replaced and hooked norms and blocks
have their say, types are those of the blocks called one by one, and nothing is skipped without a word."""

import pytest
import torch
import torch.nn as nn

from mamba_ssm_benchmark_b200 import _native as nat
from mamba_ssm_benchmark_b200 import mixer as mix
from mamba_ssm_benchmark_b200.linear import Fp8Linear
from mamba_ssm_benchmark_b200.mixer import MambaLM, RMSNorm

pytestmark = pytest.mark.gpu
DEV = "cuda"
KINDS = [dict(mixer="mamba"), dict(mixer="delta", head_dim=32)]


def _lm(seed=0, **kw):
    torch.manual_seed(seed)
    return MambaLM(n_layers=3, d_model=64, **kw).to(DEV)


def _ids(seed=0):
    return torch.randint(0, 256, (2, 20), device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))


def _one_by_one(lm, idx):
    """The model's definition: every module called, every sum a tensor of its own."""
    x = lm.embed(idx)
    for block in lm.blocks:
        x = block(x)
    return lm.head(lm.norm_f(x))


def _near(a, b, tol):
    assert a.dtype == b.dtype and a.shape == b.shape
    return float((a.double() - b.double()).norm()) <= tol * float(b.double().norm())


class Twice(RMSNorm):
    def forward(self, x):
        return 2 * super().forward(x)


def _patched(block, seen):
    run = block.forward
    block.forward = lambda *a, **k: (seen.append(1), 0.5 * run(*a, **k))[1]


@pytest.mark.parametrize("kw", KINDS)
def test_the_fused_stream_is_taken(kw, monkeypatch):
    """An untouched model adds in its norms: once a block but the first, and in the last norm."""
    calls = []
    add = RMSNorm.add
    monkeypatch.setattr(RMSNorm, "add", lambda self, *a: (calls.append(1), add(self, *a))[1])
    with torch.no_grad():
        _lm(**kw)(_ids())
    assert len(calls) == 3


@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("what", ["norm_f subclass", "norm_f layer norm", "norm_f identity", "norm_f patched", "norm1 subclass", "norm1 patched",
                                  "norm1 add patched", "block patched"])
def test_replaced_modules_have_their_say(kw, what):
    """float32 sums of a few hundred terms in another order at most: 1e-5 of the norm."""
    lm, idx, seen = _lm(**kw), _ids(), []
    place = lm.norm_f if what.startswith("norm_f") else lm.blocks[1].norm1
    if what == "norm_f subclass":
        lm.norm_f = Twice(64).to(DEV)
    elif what == "norm1 subclass":
        lm.blocks[1].norm1 = Twice(64).to(DEV)
    elif what == "norm_f layer norm":
        lm.norm_f = nn.LayerNorm(64).to(DEV)
    elif what == "norm_f identity":
        lm.norm_f = nn.Identity()
    elif what == "block patched":
        _patched(lm.blocks[1], seen)
    elif what == "norm1 add patched":
        place.add = None                                    # not to be called
    else:
        _patched(place, seen)
    with torch.no_grad():
        plain = mix.MambaLM.forward(_lm(**kw), idx)
        got = lm(idx)
        called = len(seen)
        assert _near(got, _one_by_one(lm, idx), 1e-5)
    assert called == (1 if what.endswith("patched") and what != "norm1 add patched" else 0)
    assert what == "norm1 add patched" or not _near(got, plain, 1e-2)


@pytest.mark.parametrize("kw", KINDS)
def test_a_float32_end_of_a_bf16_model(kw):
    """A final norm and a head in float32 behind blocks in bf16: logits in float32, as the norm of a bf16 tensor by a float32 weight."""
    lm, idx = _lm(**kw).bfloat16(), _ids()
    lm.norm_f.float()
    lm.head = nn.Linear(64, 256, bias=False).to(DEV)
    with torch.no_grad():
        got, want = lm(idx), _one_by_one(lm, idx)
    assert got.dtype == torch.float32 and torch.equal(got, want)


def test_a_mixer_of_another_kind():
    """A block around a module that takes (u, state, pos) and has no projections of the mixers' names."""
    class Half(nn.Module):
        def forward(self, u, state=None, pos=0):
            return 0.5 * u

    lm, idx = _lm(), _ids()
    for block in lm.blocks:
        block.mixer = Half()
    with torch.no_grad():
        assert _near(lm(idx), _one_by_one(lm, idx), 1e-5)
        x = torch.randn(2, 3, 64, device=DEV)
        assert torch.equal(lm.blocks[0](x), x + 0.5 * lm.blocks[0].norm1(x))


class Cast(nn.Module):
    """A mixer's result in another type, as one that computes in it gives; looks at what it is given."""

    def __init__(self, mixer, given, to):
        super().__init__()
        self.mixer, self.given, self.to_type = mixer, given, to

    def forward(self, u, state=None, pos=0):
        assert u.dtype == self.given
        return self.mixer(u, state, pos).to(self.to_type)


@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("to", [torch.bfloat16, torch.float16, torch.float64])
def test_mixers_whose_results_have_another_type(kw, to):
    """The stream and its norms are in the wider type, as those of x + mixer(norm(x)).  Where the additions are fused, the mixers
    see the same float32 values but for the order of a norm's sums: 2^-20; a result of a mixer may then round the other way, a step
    of its type (2^-7 of bf16) of few values: 1e-3 of the logits' norm."""
    lm, idx = _lm(**kw), _ids()
    wide = torch.promote_types(torch.float32, to)
    for i, block in enumerate(lm.blocks):
        block.mixer = Cast(block.mixer, wide if i > 0 and to == torch.float64 else torch.float32, to)
    if to == torch.float64:                                 # the kernels' mixers take what the stream's second type gives as float32
        for block in lm.blocks:
            run = block.mixer.mixer.forward
            block.mixer.mixer.forward = lambda u, *a, run=run: run(u.float(), *a)
        lm.head = nn.Linear(64, 256, bias=False, dtype=torch.float64).to(DEV)
    with torch.no_grad():
        assert _near(lm(idx), _one_by_one(lm, idx), 1e-3)
    n = RMSNorm(64).to(DEV)
    x, h = torch.randn(5, 64, device=DEV), torch.randn(5, 64, device=DEV).to(to)
    for a, b in ((x, h), (h, x), (x, h[:1])):
        y, total = n.add(a, b)
        assert torch.equal(total, a + b) and _near(y, n(a + b), 1e-6)


@pytest.mark.parametrize("kw", KINDS)
def test_autocast(kw):
    """Under autocast the mixers give bf16 and the stream stays float32; logits and gradients as block by block, where a product's
    input may round the other way: 2^-8 of few values, 1e-2 of a gradient's norm."""
    lm, idx = _lm(**kw), _ids()

    def run(forward):
        with torch.autocast(DEV, torch.bfloat16):
            logits = forward(idx)
        return [logits, *torch.autograd.grad(logits.float().logsumexp(-1).mean(), list(lm.parameters()), allow_unused=True)]

    for a, b in zip(run(lm), run(lambda i: _one_by_one(lm, i))):
        assert (a is None and b is None) or _near(a, b, 1e-2)


@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("what", ["norm1", "norm_f"])
def test_norms_of_an_8_bit_model_have_their_say(kw, what):
    """Hooks run and their results count, and so do subclasses.  A hook that changes nothing moves an e4m3 value only where the
    norm's rounding to float32 before 8 bits does: one in 10^5 by an eighth, below 2e-3 of the logits' norm."""
    lm, idx, seen = _lm(**kw).quantize_fp8(), _ids(), []
    place = lm.norm_f if what == "norm_f" else lm.blocks[1].norm1
    with torch.no_grad():
        plain = lm(idx)
        handle = place.register_forward_hook(lambda m, i, o: seen.append(o.shape))
        assert _near(lm(idx), plain, 2e-3) and seen == [(2, 20, 64)]
        handle.remove()
        handle = place.register_forward_hook(lambda m, i, o: 2 * o)
        twice = lm(idx)
        handle.remove()
        assert torch.equal(lm(idx), plain)
        other = Twice(64).to(DEV)
        if what == "norm_f":
            lm.norm_f = other
            assert _near(twice, 2 * plain, 2e-3)
        else:
            lm.blocks[1].norm1 = other
        assert torch.equal(lm(idx), twice) and not _near(twice, plain, 1e-2)
        if what == "norm_f":
            lm.norm_f = nn.LayerNorm(64).to(DEV)
        else:
            lm.blocks[1].norm1 = nn.LayerNorm(64).to(DEV)
        assert not _near(lm(idx), plain, 1e-3)


@pytest.mark.parametrize("graph", [False, True])
def test_answers_without_a_token_are_refused(graph):
    """An id outside the vocabulary makes NaN of a row's logits, for which sample_tokens gives -1: no answer, and no id to go on from."""
    lm, prompt = _lm(), _ids()
    u = torch.rand(2, 4, device=DEV)
    want = lm.generate(prompt, 4, uniforms=u, graph=graph)
    bad = prompt.clone()
    bad[0, 3] = 300
    with pytest.raises(RuntimeError, match="without a token"):
        lm.generate(bad, 4, uniforms=u, graph=graph)
    with pytest.raises(RuntimeError, match="without a token"):
        lm.generate(bad, 1, top_p=0.9)
    assert nat.read_device_error() == 2
    assert torch.equal(lm.generate(prompt, 4, uniforms=u, graph=graph), want)
    assert torch.equal(lm.generate(prompt, 0, uniforms=u[:, :0]), prompt)


@pytest.mark.parametrize("eight", [False, True])
def test_norms_with_one_weight_for_all_channels(eight):
    """Such a norm is torch's; 2e-3 as for a hooked norm of an 8-bit model."""
    lm, idx = _lm(), _ids()
    for norm in (lm.blocks[1].norm1, lm.norm_f):
        norm.weight = nn.Parameter(torch.full((1,), 1.5, device=DEV))
    with torch.no_grad():
        want = _one_by_one(lm, idx)
        if not eight:
            assert _near(lm(idx), want, 1e-5)
            return
        lm.quantize_fp8()
        got = lm(idx)
        for norm in (lm.blocks[1].norm1, lm.norm_f):
            norm.weight = nn.Parameter(torch.full((64,), 1.5, device=DEV))
        assert _near(got, lm(idx), 2e-3)


@pytest.mark.parametrize("what", ["bias", "two layers", "hook", "patched"])
def test_a_head_that_is_more_than_a_weight_stays(what):
    """quantize_fp8 leaves it as it is; the logits are those of the head on the norm of the 8-bit blocks' stream, bit by bit."""
    lm, idx, seen = _lm(), _ids(), []
    if what == "bias":
        lm.head = nn.Linear(64, 256).to(DEV)
        with torch.no_grad():
            lm.head.bias += 3.0
    elif what == "two layers":
        lm.head = nn.Sequential(nn.Linear(64, 32), nn.Linear(32, 256)).to(DEV)
    elif what == "hook":
        lm.head.register_forward_hook(lambda m, i, o: o + 3.0)
    else:
        _patched(lm.head, seen)
    head = lm.head
    with torch.no_grad():
        assert lm.quantize_fp8().head is head
        got = lm(idx)
        x = lm.embed(idx)
        for block in lm.blocks:
            assert isinstance(block.mixer.out_proj, Fp8Linear)
            x = block(x)
        assert torch.equal(got, head(lm.norm_f(x)))


def test_mixers_of_another_kind_keep_their_weights():
    """quantize_fp8 knows the projections of this package's mixers; a module that calls its own by the same names goes on as it was."""
    class Own(nn.Module):
        def __init__(self):
            super().__init__()
            self.in_proj, self.out_proj = nn.Linear(64, 32), nn.Linear(32, 64)

        def forward(self, u, state=None, pos=0):
            return self.out_proj(torch.tanh(self.in_proj(u)))

    lm, idx = _lm(), _ids()
    lm.blocks[1].mixer = Own().to(DEV)
    x = torch.randn(2, 5, 64, device=DEV)
    with torch.no_grad():
        want = lm.blocks[1](x)
        lm.quantize_fp8()
        assert torch.equal(lm.blocks[1](x), want) and isinstance(lm.blocks[0].mixer.in_proj, Fp8Linear)
        assert bool(lm(idx).isfinite().all())


class Tagged(torch.Tensor):
    pass


def test_mixers_that_give_a_tensor_of_another_class():
    """A subclass of torch.Tensor goes through the stream as through the blocks one by one."""
    class As(nn.Module):
        def __init__(self, mixer):
            super().__init__()
            self.mixer = mixer

        def forward(self, u, state=None, pos=0):
            return self.mixer(u.as_subclass(torch.Tensor), state, pos).as_subclass(Tagged)

    lm, idx = _lm(), _ids()
    for block in lm.blocks:
        block.mixer = As(block.mixer)
    with torch.no_grad():
        got, want = lm(idx), _one_by_one(lm, idx)
        assert type(want) is Tagged and type(got) is Tagged
        assert _near(got.as_subclass(torch.Tensor), want.as_subclass(torch.Tensor), 1e-5)


@pytest.mark.parametrize("cls", [RMSNorm, mix.MambaBlock])
@pytest.mark.parametrize("eight", [False, True])
def test_a_forward_put_on_the_class_is_called(cls, eight, monkeypatch):
    """As libraries do that exchange a layer's computation for all its instances; 2e-3 as for a hooked norm of an 8-bit model."""
    lm, idx, seen = _lm(), _ids(), []
    run = cls.forward
    with torch.no_grad():
        if eight:
            lm.quantize_fp8()
        plain = lm(idx)
        monkeypatch.setattr(cls, "forward", lambda self, x, *a: (seen.append(1), run(self, x, *a))[1])
        assert _near(lm(idx), plain, 2e-3 if eight else 1e-5)
    assert len(seen) == (4 if cls is RMSNorm else 3)
