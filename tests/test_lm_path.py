"""The LM on the operators around its mixers: parameters and refusals (CPU), the fused residual stream against the blocks
one by one, 8-bit weights against the same products in float64, sampling from given numbers (GPU)."""

import copy

import pytest
import torch
import torch.nn.functional as F

from mamba_ssm_benchmark_b200 import linear as lin
from mamba_ssm_benchmark_b200 import mixer as mix
from mamba_ssm_benchmark_b200 import quantize_fp8, rms_norm
from mamba_ssm_benchmark_b200.linear import Fp8Linear
from mamba_ssm_benchmark_b200.mixer import GraphDecoder, MambaLM, RMSNorm, TokenEmbedding

DEV = "cuda"
KINDS = [dict(mixer="mamba"), dict(mixer="delta", head_dim=32)]


def _lm(seed=0, **kw):
    torch.manual_seed(seed)
    return MambaLM(n_layers=3, d_model=64, **kw)


def test_embedding_and_norm_are_what_they_were_on_the_cpu():
    torch.manual_seed(0)
    a = torch.nn.Embedding(9, 4)
    torch.manual_seed(0)
    b = TokenEmbedding(9, 4)
    idx = torch.tensor([[1, 8], [0, 1]])
    assert torch.equal(a.weight, b.weight) and torch.equal(a(idx), b(idx)) and list(b.state_dict()) == ["weight"]
    n, x = RMSNorm(16), torch.randn(3, 16)
    assert torch.equal(n(x), F.rms_norm(x, (16,), eps=1e-5) * n.weight)


@pytest.mark.gpu
def test_embedding_options_keep_torchs_way():
    """padding_idx has no gradient, max_norm shortens rows: the kernels know neither."""
    idx = torch.tensor([0, 1, 1, 3], device=DEV)
    for kw in (dict(padding_idx=1), dict(max_norm=0.5), dict(scale_grad_by_freq=True)):
        torch.manual_seed(0)
        a = torch.nn.Embedding(5, 8, device=DEV, **kw)
        b = TokenEmbedding(5, 8, device=DEV, **kw)
        b.load_state_dict(a.state_dict())
        ya, yb = a(idx), b(idx)
        assert torch.equal(ya, yb)
        ga, gb = (torch.autograd.grad(y.square().sum(), m.weight)[0] for y, m in ((ya, a), (yb, b)))
        assert torch.equal(ga, gb)


def test_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        _lm().quantize_fp8()
    with pytest.raises(ValueError, match="uniforms must be"):
        _lm().generate(torch.zeros(2, 3, dtype=torch.long), 4, uniforms=torch.zeros(2, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", KINDS)
def test_fused_stream_equals_the_blocks(kw):
    """Logits and gradients with every addition in the next norm, and with the blocks called one by one (a hook on each shows
    their results).  float32 throughout: sums of a few hundred terms in other orders, 1e-5 of the norms."""
    lm = _lm(**kw).to(DEV)
    idx = torch.randint(0, 256, (2, 70), device=DEV)

    def run():
        logits = lm(idx)
        return [logits.detach(), *torch.autograd.grad(F.cross_entropy(logits.flatten(0, 1), idx.flatten()), list(lm.parameters()))]

    fused, seen = run(), []
    for b in lm.blocks:
        b.register_forward_hook(lambda m, i, o: seen.append(o))
    plain = run()
    assert len(seen) == 3 and seen[0].shape == (2, 70, 64)
    for a, b in zip(fused, plain):
        assert float((a - b).norm()) <= 1e-5 * float(b.norm())
    with torch.no_grad():
        x = seen[0]
        assert torch.equal(lm.blocks[1].norm1(x), rms_norm(x, lm.blocks[1].norm1.weight))


@pytest.mark.gpu
def test_other_types_keep_their_way():
    """A model in bfloat16, whose norm rounds once instead of twice: 2^-8 a norm, seven of them in a row beside the mixers' own
    roundings.  One in float16 is refused by the mixer's convolution, as it was."""
    lm = _lm().to(DEV)
    idx = torch.randint(0, 256, (2, 40), device=DEV)
    with torch.no_grad():
        want = lm(idx)
        got = copy.deepcopy(lm).bfloat16()(idx)
        assert got.dtype == torch.bfloat16 and float((got.float() - want).norm()) <= 14 * 2.0 ** -8 * float(want.norm())
        with pytest.raises(TypeError, match="float16"):
            copy.deepcopy(lm).half()(idx)


def _reference_linear(x8, x_scale, w8, w_scale, bias=None, activation=None, residual=None, dtype=None):
    y = (x8.double() * x_scale.double()[..., None]) @ (w8.double() * w_scale.double()[:, None]).T
    return (y if residual is None else y + residual.double()).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", KINDS)
def test_8_bit_weights(kw, monkeypatch):
    """The whole path with 8-bit weights against the same with the products in float64.  Both put the same values into 8 bits but
    where a float32 rounding moves one over a border (one value in 10^5, by an eighth: below 2e-3 of a result's norm here);
    against the model before, every value is off by up to 2^-4, at random: 2^-4 sqrt(2) / sqrt(3) a product, seven of them."""
    lm = _lm(**kw).to(DEV)
    idx = torch.randint(0, 256, (2, 50), device=DEV)
    with torch.no_grad():
        before = lm(idx)
        assert lm.quantize_fp8() is lm and isinstance(lm.head, Fp8Linear)
        held = [n for n, _ in lm.named_parameters()]
        assert not any("in_proj" in n or "out_proj" in n or "head" in n for n in held) and "embed.weight" in held
        lm.quantize_fp8()
        got = lm(idx)
        monkeypatch.setattr(lin, "linear_fp8", _reference_linear)
        want = lm(idx)
        monkeypatch.undo()
        assert got.dtype == torch.float32
        assert float((got - want).norm()) <= 2e-3 * float(want.norm())
        assert float((got - before).norm()) <= 7 * 2.0 ** -4 * (2 / 3) ** 0.5 * float(before.norm())
        # decoding: prefill, single tokens, a graph
        states = lm.init_state(2, 50, DEV)
        logits = [lm(idx[:, :40], states)] + [lm(idx[:, i:i + 1], states) for i in range(40, 45)]
        replay = GraphDecoder(lm, states)
        logits += [replay(idx[:, i:i + 1]).clone() for i in range(45, 50)]
        assert float((torch.cat(logits, 1) - got).norm()) <= 2e-3 * float(got.norm())
    with pytest.raises(RuntimeError, match="no gradient"):
        lm(idx)


@pytest.mark.gpu
def test_8_bit_weights_keep_their_form():
    """Casts, copies and state dicts; a width that is no multiple of 16."""
    w = torch.randn(40, 50, device=DEV)
    m = Fp8Linear(w)
    x = torch.randn(3, 7, 50, device=DEV)
    y = m(x)
    assert y.dtype == torch.float32 and float((y - x @ w.T).norm()) <= 2.0 ** -4 * float((x @ w.T).norm())
    for other in (copy.deepcopy(m).bfloat16(), copy.deepcopy(m).half().float()):
        assert other.weight_scale.dtype == torch.float32 and torch.equal(other(x), y)
    fresh = Fp8Linear(torch.zeros_like(w))
    fresh.load_state_dict(m.state_dict())
    assert torch.equal(fresh(x), y)
    assert m(x.bfloat16()).dtype == torch.bfloat16 and m(quantize_fp8(x)).dtype == torch.float32
    r = torch.randn(3, 7, 40, device=DEV)
    assert torch.equal(m(x, residual=r), m(quantize_fp8(x), residual=r))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", KINDS)
def test_generate_from_given_numbers(kw):
    lm = _lm(**kw).to(DEV)
    prompt = torch.randint(0, 256, (3, 9), device=DEV)
    u = torch.rand(3, 6, device=DEV)
    a = lm.generate(prompt, 6, uniforms=u, top_k=50, top_p=0.9, min_p=0.01, temperature=0.8)
    assert torch.equal(a, lm.generate(prompt, 6, uniforms=u, top_k=50, top_p=0.9, min_p=0.01, temperature=0.8, graph=True))
    assert torch.equal(a[:, :9], prompt) and int(a.min()) >= 0
    greedy = lm.generate(prompt, 6, uniforms=u, temperature=0.0)
    assert torch.equal(greedy, lm.generate(prompt, 6, top_k=1))
    t = torch.tensor([0.0, 1.0, 0.5], device=DEV, dtype=torch.float64)
    rows = lm.generate(prompt, 6, uniforms=u, temperature=t, top_p=0.9)
    assert torch.equal(rows[0], greedy[0])
    assert lm.generate(prompt, 6, top_p=0.9).shape == (3, 15)
    assert torch.equal(lm.quantize_fp8().generate(prompt, 6, uniforms=u, top_p=0.9), lm.generate(prompt, 6, uniforms=u, top_p=0.9, graph=True))


@pytest.mark.gpu
def test_training_with_the_fused_stream():
    """Runs, and its gradients are those of the model whose blocks are called one by one; a graph of the whole step too."""
    lm = _lm().to(DEV)
    idx = torch.randint(0, 256, (2, 33), device=DEV)
    grads = lambda: torch.autograd.grad(F.cross_entropy(lm(idx[:, :-1]).flatten(0, 1), idx[:, 1:].flatten()), list(lm.parameters()))
    want = [g.clone() for g in grads()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = grads()
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
