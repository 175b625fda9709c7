"""Cases of the gated delta rule and of the channels-last group norm: inputs, plain forms and exact values.

The two operators make up a gated delta-rule mixer layer next to the Mamba mixer:

* ``delta``: per value head a state S (dk x dv), S_t = exp(g_t) S_{t-1} + beta_t k_t (v_t - (exp(g_t) S_{t-1})^T k_t)^T,
  o_t = scale S_t^T q_t.  Directions: "forward" (a sequence, inference), "train" (a sequence and all its
  gradients) and "step" (one token, the state updated in place).
* ``norm``: y = act((x - mean) rstd w + b) silu(z), the statistics over (positions, C / groups) of every sample.
  ``positions == 1`` is the norm of every head of every token, with the gate of the mixer; more positions are the
  norm of a whole sequence.  Directions: "forward" and "train".

With ``own`` false ``run`` uses elementary torch operations in float32, with ``own`` true the package's operators.
"""

import math

import torch

own = False

CHUNK = 64          # positions that the plain form of the delta rule takes together


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _delta(name, what, B, L, Hk, Hv, dk, dv, dtype, h0):
    return {"name": name, "op": "delta", "what": what, "B": B, "L": L, "Hk": Hk, "Hv": Hv, "dk": dk, "dv": dv,
            "dtype": dtype, "h0": h0}


def _norm(name, what, samples, positions, C, groups, dtype, center, act, gate):
    return {"name": name, "op": "norm", "what": what, "samples": samples, "positions": positions, "C": C,
            "groups": groups, "dtype": dtype, "center": center, "act": act, "gate": gate}


def listed():
    return [
        # one token of one sequence through a layer of the 256-wide byte LM (inner width 512: 8 heads of 64)
        _delta("step of one sequence", "step", 1, 1, 8, 8, 64, 64, "float32", True),
        # one token of a serving batch of 64, 16 value heads of 128 over 8 key heads
        _delta("step of a batch", "step", 64, 1, 8, 16, 128, 128, "bfloat16", True),
        # a short ragged prompt that continues from a state
        _delta("short prompt", "forward", 3, 197, 4, 8, 64, 64, "float32", True),
        # a long prompt of one sequence at an inner width of 1024: few heads, many positions
        _delta("long prompt", "forward", 1, 16384, 8, 8, 128, 128, "bfloat16", False),
        # head widths that fill no tile, an odd length
        _delta("odd heads", "train", 2, 333, 3, 6, 48, 80, "bfloat16", True),
        # the byte LM's training batch: 16 sequences of 512, 8 heads of 64
        _delta("training, narrow", "train", 16, 512, 8, 8, 64, 64, "float32", False),
        # training at an inner width of 5120: 40 value heads of 128 that share 20 key heads
        _delta("training, wide", "train", 2, 4096, 20, 40, 128, 128, "bfloat16", False),
        # the head norm and gate behind one decoded token
        _norm("head norm of a token", "forward", 1, 1, 512, 8, "float32", False, "none", True),
        # the head norm and gate in the byte LM's training batch (16 x 512 tokens)
        _norm("head norm, narrow", "train", 16 * 512, 1, 512, 8, "float32", False, "none", True),
        # the head norm and gate in training at an inner width of 5120
        _norm("head norm, wide", "train", 4 * 4096, 1, 5120, 40, "bfloat16", False, "none", True),
        # group norm and SiLU over long sequences, inference
        _norm("sequence norm", "forward", 8, 8192, 512, 32, "bfloat16", True, "silu", False),
        # channels that fill no vector, an odd length, training
        _norm("odd channels", "train", 3, 1021, 330, 11, "float32", True, "silu", False),
    ]


def _spread(rng, lo, hi):
    """A whole number in lo..hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16"])
    if rng.random() < 0.6:
        what = rng.choice(["step", "forward", "train"])
        Hk = _spread(rng, 1, 20)
        Hv = Hk * rng.choice([1, 1, 2])
        dk, dv = (rng.choice([64, 128, rng.randint(16, 128)]) for _ in range(2))
        L = 1 if what == "step" else _spread(rng, 2, 16384 if what == "forward" else 4096)
        most = (64 * 16 if what == "step" else 2 * 4096 * 40 // L) // Hv      # no more than the largest listed case
        B = _spread(rng, 1, max(1, min(64, most)))
        while Hv > 1 and B * L * Hv > 2 * 4096 * 40:
            Hk, Hv = 1, max(1, Hv // 2)
        h0 = what == "step" or rng.random() < 0.5
        return {k: v for k, v in _delta("", what, B, L, Hk, Hv, dk, dv, dtype, h0).items() if k != "name"}
    what = rng.choice(["forward", "train"])
    groups = rng.choice([1, 4, 8, 32, rng.randint(1, 40)])
    C = groups * _spread(rng, 8, max(8, 5120 // groups))
    most = 4 * 4096 * 5120 // C
    if rng.random() < 0.5:
        samples, positions = _spread(rng, 1, min(65536, most)), 1
    else:
        samples = _spread(rng, 1, 16)
        positions = _spread(rng, 2, max(2, min(8192, most // samples)))
    center = positions > 1 or rng.random() < 0.5
    case = _norm("", what, samples, positions, C, groups, dtype, center, rng.choice(["none", "silu"]), positions == 1)
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _inputs(c, seed):
    """The case's tensors by name, made on the GPU from the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, c["dtype"])

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    t = {}
    if c["op"] == "delta":
        B, L, Hk, Hv, dk, dv = (c[k] for k in ("B", "L", "Hk", "Hv", "dk", "dv"))
        for name in ("q", "k"):       # what conv + SiLU leave, every head scaled to length 1
            x = torch.nn.functional.silu(randn(B, L, Hk, dk))
            t[name] = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()).to(dt)
        t["v"] = torch.nn.functional.silu(randn(B, L, Hv, dv)).to(dt)
        # g = -a softplus(dt): decay rates a in [1, 16] by head, step sizes around [1e-3, 1e-1]
        a = 1.0 + 15.0 * rand(Hv)
        dt_bias = math.log(1e-3) + rand(Hv) * math.log(100.0)
        t["g"] = -a * torch.nn.functional.softplus(randn(B, L, Hv) + torch.log(torch.expm1(torch.exp(dt_bias))))
        t["beta"] = torch.sigmoid(randn(B, L, Hv))
        if c["h0"]:
            t["h0"] = 0.1 * randn(B, Hv, dk, dv)
        if c["what"] == "train":
            t["do"] = randn(B, L, Hv, dv).to(dt)
            t["dlast"] = 0.1 * randn(B, Hv, dk, dv)
        return t
    shape = (c["samples"], c["C"]) if c["positions"] == 1 else (c["samples"], c["positions"], c["C"])
    t["x"] = (randn(*shape) * (0.5 + rand(c["C"])) + (0.3 * randn(c["C"]) if c["center"] else 0.0)).to(dt)
    t["weight"] = 1.0 + 0.1 * randn(c["C"])
    if c["center"]:
        t["bias"] = 0.1 * randn(c["C"])
    if c["gate"]:
        t["z"] = randn(*shape).to(dt)
    if c["what"] == "train":
        t["dy"] = randn(*shape).to(dt)
    return t


_LEAVES = {"delta": ("q", "k", "v", "g", "beta", "h0"), "norm": ("x", "weight", "bias", "z")}


def prepare(case, seed):
    return dict(case), _inputs(case, seed)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    c, t = state
    if c["op"] == "delta" and c["what"] == "step":
        return _step(t)
    forward = _delta_forward if c["op"] == "delta" else _norm_forward
    if c["what"] == "forward":
        with torch.no_grad():
            return forward(c, t)
    names = [n for n in _LEAVES[c["op"]] if n in t]
    leaves = {n: t[n].detach().requires_grad_() for n in names}
    out = forward(c, leaves)
    douts = [t["do"], t["dlast"]] if c["op"] == "delta" else [t["dy"]]
    grads = torch.autograd.grad([out[n] for n in (("o", "last") if c["op"] == "delta" else ("y",))],
                                [leaves[n] for n in names], douts)
    return {**{n: x.detach() for n, x in out.items()}, **{"d" + n: x for n, x in zip(names, grads)}}


def _step(t):
    if own:
        from mamba_ssm_benchmark_b200 import gated_delta_state_update
        o = gated_delta_state_update(t["h0"], t["q"][:, 0], t["k"][:, 0], t["v"][:, 0], t["g"][:, 0], t["beta"][:, 0])
        return {"o": o, "state": t["h0"]}
    S, group = t["h0"], t["v"].shape[2] // t["q"].shape[2]
    q, k = (t[n][:, 0].float().repeat_interleave(group, dim=1) for n in ("q", "k"))
    v, beta = t["v"][:, 0].float(), t["beta"][:, 0]
    S.mul_(torch.exp(t["g"][:, 0])[..., None, None])
    e = beta[..., None] * (v - (S * k[..., None]).sum(-2))
    S.add_(k[..., None] * e[..., None, :])
    o = (S * q[..., None]).sum(-2) * q.shape[-1] ** -0.5
    return {"o": o.to(t["v"].dtype), "state": S}


def _delta_forward(c, t):
    if own:
        from mamba_ssm_benchmark_b200 import gated_delta_rule
        o, last = gated_delta_rule(t["q"], t["k"], t["v"], t["g"], t["beta"], h0=t.get("h0"))
    else:
        o, last = _delta_plain(t["q"], t["k"], t["v"], t["g"], t["beta"], t.get("h0"))
    return {"o": o, "last": last}


def _delta_plain(q, k, v, g, beta, h0):
    """The delta rule over chunks of positions, all chunks' own products at once and the state from chunk to chunk.
    Within a chunk, with G the running sum of g:  (I + A) U = beta (V - exp(G) K S),  A = beta exp(G_i - G_j) k_i k_j
    below the diagonal;  O = scale (exp(G) Q S + P U);  S' = exp(G_last) S + (exp(G_last - G) K)^T U."""
    B, L, Hv, dv = v.shape
    dk, n, dtype = q.shape[-1], -(-L // CHUNK), v.dtype

    def chunks(x, group=1):         # (B, L, H, ...) -> (B, Hv, n, CHUNK, ...), positions past L are zero
        x = x.float().repeat_interleave(group, dim=2) if group > 1 else x.float()
        x = torch.cat([x, x.new_zeros(B, n * CHUNK - L, *x.shape[2:])], dim=1)
        return x.unflatten(1, (n, CHUNK)).movedim(3, 1)

    q, k = (chunks(x, Hv // q.shape[2]) for x in (q, k))
    v, G, beta = chunks(v), chunks(g).cumsum(-1), chunks(beta)[..., None]
    row = torch.arange(CHUNK, device=v.device)
    decay = torch.exp((G[..., :, None] - G[..., None, :]).masked_fill(row[:, None] < row, -math.inf))
    kt = k.transpose(-1, -2)
    A = beta * (k @ kt) * decay * (row[:, None] > row)
    P = (q @ kt) * decay
    T = torch.eye(CHUNK, device=v.device).expand_as(A)
    size = 1
    while size < CHUNK:             # inverses of diagonal blocks of twice the size from those of this size
        lower = (row[:, None] // size % 2 == 1) & (row[:, None] // size - 1 == row // size)
        T = T - T @ (A * lower) @ T
        size *= 2
    eG = torch.exp(G)[..., None]
    U0, W = T @ (beta * v), T @ (beta * eG * k)
    Q, K = eG * q, torch.exp(G[..., -1:] - G)[..., None] * k
    keep = torch.exp(G[..., -1])[..., None, None]
    S = v.new_zeros(B, Hv, dk, dv) if h0 is None else h0.float()
    out = []
    for i in range(n):
        U = U0[:, :, i] - W[:, :, i] @ S
        out.append(Q[:, :, i] @ S + P[:, :, i] @ U)
        S = keep[:, :, i] * S + K[:, :, i].transpose(-1, -2) @ U
    o = torch.stack(out, dim=2).movedim(1, 3).flatten(1, 2)[:, :L] * dk ** -0.5
    return o.to(dtype), S


def _norm_forward(c, t):
    act = None if c["act"] == "none" else c["act"]
    if own:
        from mamba_ssm_benchmark_b200 import group_norm
        return {"y": group_norm(t["x"], c["groups"], t["weight"], t.get("bias"), activation=act, z=t.get("z"),
                                center=c["center"])}
    x = t["x"].float()
    x = x.reshape(c["samples"], c["positions"], c["groups"], c["C"] // c["groups"])
    if c["center"]:
        x = x - x.mean(dim=(1, 3), keepdim=True)
    y = x / (x.square().mean(dim=(1, 3), keepdim=True) + 1e-5).sqrt()
    y = y.reshape(t["x"].shape) * t["weight"]
    if c["center"]:
        y = y + t["bias"]
    if act == "silu":
        y = y / (1.0 + torch.exp(-y))
    if c["gate"]:
        z = t["z"].float()
        y = y * (z / (1.0 + torch.exp(-z)))
    return {"y": y.to(t["x"].dtype)}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(c):
    e = 2 if c["dtype"] == "bfloat16" else 4
    train = c["what"] == "train"
    if c["op"] == "delta":
        rows = c["B"] * c["L"]
        qk, vo = 2 * rows * c["Hk"] * c["dk"] * e, 2 * rows * c["Hv"] * c["dv"] * e
        gates, state = 2 * rows * c["Hv"] * 4, c["B"] * c["Hv"] * c["dk"] * c["dv"] * 4
        # q, k, v, g, beta, h0 in, o and the last state out; training: also do and dlast in, all gradients out
        total = qk + vo + gates + state * (2 if c["h0"] else 1)
        if train:
            total += qk + vo + gates + state * (2 if c["h0"] else 1)
        # per position and value head: decay, S^T k, rank-1 update, S^T q; backward the products of each with both factors
        flops = rows * c["Hv"] * c["dk"] * c["dv"] * (7 + (14 if train else 0))
        return {"bytes": total, "flops": flops}
    n = c["samples"] * c["positions"] * c["C"]
    tensors = (3 if c["gate"] else 2) + ((3 if c["gate"] else 2) if train else 0)      # x, z, y; dy, dx, dz
    params = c["C"] * 4 * (2 if c["center"] else 1) * (2 if train else 1)
    return {"bytes": tensors * n * e + params, "flops": n * (10 + (20 if train else 0))}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    t = {n: x.double() for n, x in _inputs(case, seed).items()}
    return (_delta_exact if case["op"] == "delta" else _norm_exact)(case, t)


def _delta_exact(c, t):
    """The recurrence position by position, and its derivative position by position in reverse.  States are kept at
    the start of every 64 positions and computed again from there."""
    B, L, Hv, dv, dk, train = c["B"], c["L"], c["Hv"], c["dv"], c["dk"], c["what"] == "train"
    group, scale = Hv // c["Hk"], c["dk"] ** -0.5
    q, k = (t[n].repeat_interleave(group, dim=2) for n in ("q", "k"))
    v, alpha, beta = t["v"], torch.exp(t["g"])[..., None, None], t["beta"][..., None]
    S = t["h0"] if "h0" in t else v.new_zeros(B, Hv, dk, dv)

    def advance(S, i):
        decayed = alpha[:, i] * S
        miss = v[:, i] - torch.einsum("bhkv,bhk->bhv", decayed, k[:, i])
        return decayed, miss, decayed + k[:, i, :, :, None] * (beta[:, i] * miss)[:, :, None]

    marks, o = [], torch.empty_like(v)
    for i in range(L):
        if train and i % 64 == 0:
            marks.append(S)
        S = advance(S, i)[2]
        o[:, i] = scale * torch.einsum("bhkv,bhk->bhv", S, q[:, i])
    if c["what"] == "step":
        return {"o": o[:, 0], "state": S}
    if not train:
        return {"o": o, "last": S}
    grads = {"dq": torch.empty_like(q), "dk": torch.empty_like(k), "dv": torch.empty_like(v),
             "dg": torch.empty_like(t["g"]), "dbeta": torch.empty_like(t["g"])}
    dS = t["dlast"]
    for m in reversed(range(len(marks))):
        kept, Si = [], marks[m]
        for i in range(64 * m, min(L, 64 * m + 64)):
            kept.append((Si, *advance(Si, i)))
            Si = kept[-1][3]
        for i in reversed(range(64 * m, min(L, 64 * m + 64))):
            before, decayed, miss, after = kept.pop()
            do = t["do"][:, i]
            grads["dq"][:, i] = scale * torch.einsum("bhkv,bhv->bhk", after, do)
            dS = dS + scale * q[:, i, :, :, None] * do[:, :, None]
            dw = torch.einsum("bhkv,bhk->bhv", dS, k[:, i])               # gradient of beta * miss
            dmiss = beta[:, i] * dw
            grads["dk"][:, i] = (torch.einsum("bhkv,bhv->bhk", dS, beta[:, i] * miss)
                                 - torch.einsum("bhkv,bhv->bhk", decayed, dmiss))
            grads["dv"][:, i] = dmiss
            grads["dbeta"][:, i] = (dw * miss).sum(-1)
            dS = dS - k[:, i, :, :, None] * dmiss[:, :, None]
            grads["dg"][:, i] = (dS * decayed).sum((-1, -2))
            dS = alpha[:, i] * dS
    for n in ("dq", "dk"):
        grads[n] = grads[n].unflatten(2, (c["Hk"], group)).sum(3)
    if "h0" in t:
        grads["dh0"] = dS
    return {"o": o, "last": S, **grads}


def _norm_exact(c, t):
    shape, full = t["x"].shape, (c["samples"], c["positions"], c["groups"], c["C"] // c["groups"])
    x = t["x"].reshape(full)
    mean = x.mean(dim=(1, 3), keepdim=True) if c["center"] else torch.zeros_like(x[:, :1, :, :1])
    rstd = ((x - mean).pow(2).mean(dim=(1, 3), keepdim=True) + 1e-5).rsqrt()
    n = ((x - mean) * rstd).reshape(shape)
    pre = n * t["weight"] + (t["bias"] if c["center"] else 0.0)
    sig, z = torch.sigmoid(pre), t.get("z")
    a = pre * sig if c["act"] == "silu" else pre
    gate = z * torch.sigmoid(z) if z is not None else torch.ones_like(pre)
    out = {"y": a * gate}
    if c["what"] == "forward":
        return out
    dpre = t["dy"] * gate * (sig * (1.0 + pre * (1.0 - sig)) if c["act"] == "silu" else 1.0)
    over = tuple(range(len(shape) - 1))
    out["dweight"] = (dpre * n).sum(over)
    if c["center"]:
        out["dbias"] = dpre.sum(over)
    if z is not None:
        s = torch.sigmoid(z)
        out["dz"] = t["dy"] * a * s * (1.0 + z * (1.0 - s))
    dn, n = (dpre * t["weight"]).reshape(full), n.reshape(full)
    dx = dn - n * (dn * n).mean(dim=(1, 3), keepdim=True)
    if c["center"]:
        dx = dx - dn.mean(dim=(1, 3), keepdim=True)
    out["dx"] = (dx * rstd).reshape(shape)
    return out
