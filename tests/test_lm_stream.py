"""What the LM's fused residual stream and 8-bit path leave to the modules that stand in them: replaced and hooked norms and blocks
have their say, types are those of the blocks called one by one, and nothing is skipped without a word."""

import pytest
import torch
import torch.nn as nn

from mamba_ssm_benchmark_b200 import mixer as mix
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
