"""The gated delta-rule mixer and the LM built on it: parameters and refusals (CPU), the mixer against its definition
in float64, decoding against a whole pass (GPU).

Tolerances: the mixer adds projections of a few hundred terms in float32 (2^-24 each) to operators held to 2e-5, and
its gradients pass them twice: 1e-4 on ||difference|| / ||reference||."""

import pytest
import torch
import torch.nn.functional as F

from mamba_ssm_benchmark_b200.delta_mixer import GatedDeltaMixer
from mamba_ssm_benchmark_b200.mixer import GraphDecoder, MambaBlock, MambaLM
from oracle import delta_oracle as D
from oracle import scan_oracle as O

DEV = "cuda"
TOL = 1e-4


def test_parameters_and_refusals():
    m = GatedDeltaMixer(128, head_dim=32, key_heads=4)
    shapes = {n: tuple(p.shape) for n, p in m.named_parameters()}
    assert shapes == {"in_proj.weight": (768, 128), "gate_proj.weight": (16, 128), "conv.weight": (512, 1, 4),
                      "conv.bias": (512,), "out_proj.weight": (128, 256), "A_log": (8,), "dt_bias": (8,),
                      "norm_weight": (256,)}
    assert "unit" not in m.state_dict()
    state = m.init_state(3, 100, "cpu")
    assert state.conv.shape == (3, 512, 3) and state.ssm.shape == (3, 8, 32, 32)
    with pytest.raises(ValueError, match="multiple of head_dim"):
        GatedDeltaMixer(100, head_dim=64)
    with pytest.raises(ValueError, match="key heads"):
        GatedDeltaMixer(128, head_dim=64, key_heads=3)
    with pytest.raises(ValueError, match="mixer must"):
        MambaBlock(64, mixer="other")


def test_lm_with_the_mamba_mixer_is_unchanged():
    """The same seed gives the same parameters with and without naming the mixer."""
    torch.manual_seed(0)
    a = MambaLM(n_layers=2, d_model=32)
    torch.manual_seed(0)
    b = MambaLM(n_layers=2, d_model=32, mixer="mamba")
    assert [n for n, _ in a.named_parameters()] == [n for n, _ in b.named_parameters()]
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))


def _definition(m, p, u):
    """GatedDeltaMixer.forward without a state, from the oracles, with parameters p in u's type."""
    B, L, _ = u.shape
    H, d = m.heads, m.head_dim
    xz = u @ p["in_proj.weight"].T
    x, z = xz[..., :m.d_conv_in], xz[..., m.d_conv_in:]
    gate = u @ p["gate_proj.weight"].T
    g = -torch.exp(p["A_log"]) * F.softplus(gate[..., :H] + p["dt_bias"])
    x, _ = O.causal_conv1d(x, p["conv.weight"][:, 0], p["conv.bias"])
    q, k = (x[..., i * m.d_key:(i + 1) * m.d_key].reshape(B, L, m.key_heads, d) for i in range(2))
    q, k = (t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * d ** -0.5 for t in (q, k))
    v = x[..., 2 * m.d_key:].reshape(B, L, H, d)
    o, _ = D.gated_delta_rule(q, k, v, g, torch.sigmoid(gate[..., H:]))
    o = D.group_norm(o.reshape(B * L, -1), H, p["norm_weight"], z=z.reshape(B * L, -1), center=False)
    return o.reshape(B, L, -1) @ p["out_proj.weight"].T


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(head_dim=32, key_heads=2), dict(head_dim=64, expand=1), dict(head_dim=16, d_conv=2)])
def test_mixer_against_its_definition(kw):
    torch.manual_seed(1)
    m = GatedDeltaMixer(64, **kw)
    u, dy = torch.randn(2, 75, 64), torch.randn(2, 75, 64)
    p = {n: t.detach().double().requires_grad_() for n, t in m.named_parameters()}
    ud = u.double().requires_grad_()
    want = _definition(m, p, ud)
    wg = torch.autograd.grad(want, [ud, *p.values()], dy.double())
    m = m.to(DEV)
    ug = u.to(DEV).requires_grad_()
    got = m(ug)
    gg = torch.autograd.grad(got, [ug, *m.parameters()], dy.to(DEV))
    for name, a, b in zip(["out", "u", *p], [got, *gg], [want, *wg]):
        err = float((a.detach().cpu().double() - b).norm() / b.norm())
        assert err <= TOL, (name, err)


@pytest.mark.gpu
def test_decoding_equals_a_whole_pass():
    """Prefill and single tokens, eagerly and as a CUDA graph, give the logits of one pass over the sequence."""
    torch.manual_seed(2)
    lm = MambaLM(n_layers=2, d_model=64, mixer="delta", head_dim=32).to(DEV)
    idx = torch.randint(0, 256, (3, 90), device=DEV)
    with torch.no_grad():
        full = lm(idx)
        states = lm.init_state(3, 90, DEV)
        logits = [lm(idx[:, :70], states)]
        logits += [lm(idx[:, i:i + 1], states) for i in range(70, 80)]
        replay = GraphDecoder(lm, states)
        logits += [replay(idx[:, i:i + 1]).clone() for i in range(80, 90)]
    err = float((torch.cat(logits, 1) - full).norm() / full.norm())
    assert err <= TOL, err
    out = lm.generate(idx[:, :8], 5, graph=True)
    assert out.shape == (3, 13) and torch.equal(out[:, :8], idx[:, :8])


@pytest.mark.gpu
def test_training_lowers_the_loss():
    torch.manual_seed(3)
    lm = MambaLM(n_layers=2, d_model=64, mixer="delta", head_dim=32).to(DEV)
    idx = torch.randint(0, 16, (4, 65), device=DEV)
    opt = torch.optim.AdamW(lm.parameters(), lr=3e-3)
    losses = []
    for _ in range(20):
        loss = F.cross_entropy(lm(idx[:, :-1]).flatten(0, 1), idx[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < 0.8 * losses[0]


@pytest.mark.parametrize("make", [lambda d: GatedDeltaMixer(256, head_dim=d), lambda d: MambaLM(n_layers=1, d_model=256, mixer="delta", head_dim=d)])
def test_head_widths_without_a_kernel_are_refused_at_once(make):
    assert make(128) is not None
    for d in (0, 256):
        with pytest.raises(ValueError, match="head_dim must be"):
            make(d)


def test_a_cast_leaves_the_key_scale():
    """x / rms(x) times head_dim^-1/2: that factor in float32 whatever the model's type."""
    for cast in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.bfloat16().float(), lambda m: m.to("meta").to_empty(device="cpu")):
        m = cast(GatedDeltaMixer(128, head_dim=32))
        assert m.unit.dtype == torch.float32 and torch.equal(m.unit, torch.full((2 * m.d_key,), 32 ** -0.5)), m.unit


@pytest.mark.gpu
def test_bf16_mixer_against_its_definition():
    """A mixer in bfloat16 on its own (rounded) parameters: four operators and two projections in a row each round their
    result (2^-8 of every element, unrelated to one another), the products before the gate pass one of them on twice."""
    torch.manual_seed(5)
    m = GatedDeltaMixer(64, head_dim=32).bfloat16()
    u = torch.randn(2, 75, 64).bfloat16()
    with torch.no_grad():
        want = _definition(m, {n: t.detach().double() for n, t in m.named_parameters()}, u.double())
        got = m.to(DEV)(u.to(DEV))
    assert got.dtype == torch.bfloat16
    assert float((got.cpu().double() - want).norm() / want.norm()) <= 8 * 2.0 ** -8
