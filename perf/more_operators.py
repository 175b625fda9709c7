"""Cases of the operators around a language model's mixers: inputs, plain forms and exact values.

From a token to the next one, outside the mixers:

* ``embedding``: y = scale W[idx], and its gradient dW[v] = scale sum of dy over the places that hold v.
  Directions: "forward" and "train".
* ``norm``: total = x + residual (kept in the wider of their types), y = total / rms(total) weight.  Directions:
  "forward", "train" (all gradients) and "fp8" (y in 8 bits, e4m3, with a scale for every row).
* ``linear``: y = act(x_scale w_scale (x8 W8^T) + bias) + residual, x8 and W8 in e4m3 with a scale for every row.
* ``sample``: the next token of every row of logits from a given uniform number: of softmax(logits / temperature), the
  top_k largest are kept, of these the smallest set that reaches top_p of their sum, of these what has at least min_p of
  the largest one's probability; the token is the first, by index, where the kept weights' running sum passes u times
  their sum.  Ties go to the lowest index, temperature 0 is the largest logit.

With ``own`` false ``run`` uses elementary torch operations, with ``own`` true the package's operators.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
TINY = 1e-30            # rows whose largest value is below it share its scale


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def _embedding(name, what, tokens, vocab, C, dtype, scale):
    return {"name": name, "op": "embedding", "what": what, "tokens": tokens, "vocab": vocab, "C": C, "dtype": dtype,
            "scale": scale}


def _norm(name, what, rows, C, dtype, residual):
    return {"name": name, "op": "norm", "what": what, "rows": rows, "C": C, "dtype": dtype, "residual": residual}


def _linear(name, M, K, N, dtype, bias, act, residual):
    return {"name": name, "op": "linear", "M": M, "K": K, "N": N, "dtype": dtype, "bias": bias, "act": act,
            "residual": residual}


def _sample(name, B, vocab, dtype, spread, temperature, top_k, top_p, min_p, masked, per_row):
    return {"name": name, "op": "sample", "B": B, "vocab": vocab, "dtype": dtype, "spread": spread,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "masked": masked,
            "per_row": per_row}


def listed():
    return [
        # one decoded token of eight sequences of the 256-wide byte LM
        _embedding("embed, decoding", "forward", 8, 256, 256, "float32", 1.0),
        # the byte LM's training batch: 16 sequences of 512
        _embedding("embed, training bytes", "train", 16 * 512, 256, 256, "float32", 1.0),
        # training on words: eight sequences of 8192, a vocabulary of 50257, rows scaled by the root of the width
        _embedding("embed, training words", "train", 8 * 8192, 50257, 2560, "bfloat16", 50.5),
        # the residual stream of one decoded token, normed for an 8-bit projection
        _norm("norm of a token, 8 bits", "fp8", 1, 256, "float32", "float32"),
        # the residual stream of a prompt of 8192 tokens, normed for an 8-bit projection
        _norm("norm of a prompt, 8 bits", "fp8", 8192, 2560, "bfloat16", "bfloat16"),
        # addition and norm in training at a width of 5120
        _norm("norm, training", "train", 4 * 4096, 5120, "bfloat16", "bfloat16"),
        # the input projection of one decoded token of the 256-wide byte LM
        _linear("project a token", 1, 256, 1024, "float32", False, "none", False),
        # the input projection of 64 decoded tokens at a width of 2560 (inner width 5120, x and z)
        _linear("project a batch", 64, 2560, 10240, "bfloat16", False, "none", False),
        # the output projection of a prompt of 16384 tokens, onto the residual stream
        _linear("project a prompt", 16384, 5120, 2560, "bfloat16", True, "none", True),
        # the next byte of one sequence
        _sample("sample a byte", 1, 256, "float32", 2.0, 1.0, 40, 1.0, 0.0, 0.0, False),
        # a serving batch of 64, every sequence with settings of its own
        _sample("sample, serving", 64, 50257, "bfloat16", 3.0, 0.8, 50, 0.95, 0.02, 0.0, True),
        # a large batch over a large vocabulary by top-p alone, some of it masked
        _sample("sample, large", 256, 131072, "float32", 2.0, 1.0, 0, 0.9, 0.0, 0.05, False),
    ]


def _spread(rng, lo, hi):
    """A whole number in lo..hi, even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(["embedding", "norm", "linear", "sample"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "embedding":
        C = _spread(rng, 16, 4096)
        tokens = _spread(rng, 1, min(65536, 8 * 8192 * 2560 // (2 * C)))
        vocab = _spread(rng, 64, min(131072, 50257 * 2560 // (2 * C)))
        case = _embedding("", rng.choice(["forward", "train"]), tokens, vocab, C, dtype, rng.choice([1.0, round(C ** 0.5, 2)]))
    elif op == "norm":
        C = _spread(rng, 16, 8192)
        rows = _spread(rng, 1, min(65536, 4 * 4096 * 5120 // (2 * C)))
        residual = rng.choice(["none", "float32", dtype])
        case = _norm("", rng.choice(["forward", "train", "fp8"]), rows, C, dtype, residual)
    elif op == "linear":
        K, N = _spread(rng, 16, 10240), _spread(rng, 16, 10240)
        M = rng.choice([_spread(rng, 1, 64), _spread(rng, 1, max(1, min(16384, 16384 * 5120 * 2560 // (K * N))))])
        case = _linear("", M, K, N, dtype, rng.random() < 0.5, rng.choice(["none", "silu"]), rng.random() < 0.5)
    else:
        vocab = _spread(rng, 32, 131072)
        B = _spread(rng, 1, min(256, 256 * 131072 // (2 * vocab)))
        case = _sample("", B, vocab, dtype, round(rng.uniform(0.5, 4.0), 2), rng.choice([0.0, 1.0, round(rng.uniform(0.3, 1.5), 2)]),
                       rng.choice([0, _spread(rng, 1, vocab)]), rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)]),
                       rng.choice([0.0, round(rng.uniform(0.001, 0.3), 4)]), rng.choice([0.0, 0.3]), rng.random() < 0.3)
    return {k: v for k, v in case.items() if k != "name"}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _rows8(x):
    """Rows in e4m3 with a scale each; rows start at multiples of 16 bytes, as the framework lays them out."""
    K = x.shape[-1]
    scale = x.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
    buf = torch.zeros(x.shape[0], -(-K // 16) * 16, device=x.device, dtype=torch.float8_e4m3fn)
    buf[:, :K] = (x / scale[:, None]).to(torch.float8_e4m3fn)
    return buf[:, :K], scale


def _inputs(c, seed):
    """The case's tensors by name, made on the GPU from the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, c["dtype"])

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    t = {}
    if c["op"] == "embedding":
        # as in text: the r-th most frequent token has a share of about 1 / r, and the order of ids says nothing
        V, T = c["vocab"], c["tokens"]
        rank = torch.exp(rand(T).double() * math.log(V + 1)).long().sub_(1).clamp_(0, V - 1)
        t["idx"] = torch.randperm(V, device="cuda", generator=gen)[rank]
        t["weight"] = (0.02 * randn(V, c["C"])).to(dt)
        if c["what"] == "train":
            t["dy"] = randn(T, c["C"]).to(dt)
    elif c["op"] == "norm":
        shape = (c["rows"], c["C"])
        t["x"] = (randn(*shape) * (0.5 + rand(c["C"]))).to(dt)
        if c["residual"] != "none":
            t["residual"] = (2.0 * randn(*shape)).to(getattr(torch, c["residual"]))
        t["weight"] = 1.0 + 0.1 * randn(c["C"])
        if c["what"] == "train":
            t["dy"] = randn(*shape).to(dt)
            if c["residual"] != "none":
                t["dtotal"] = randn(*shape).to(_wider(t["x"], t["residual"]))
    elif c["op"] == "linear":
        t["x8"], t["x_scale"] = _rows8(randn(c["M"], c["K"]))
        t["w8"], t["w_scale"] = _rows8(randn(c["N"], c["K"]) * c["K"] ** -0.5)
        if c["bias"]:
            t["bias"] = 0.1 * randn(c["N"])
        if c["residual"]:
            t["residual"] = randn(c["M"], c["N"]).to(dt)
    else:
        B, V = c["B"], c["vocab"]
        logits = c["spread"] * randn(B, V)
        if c["masked"]:
            logits.masked_fill_(rand(V) < c["masked"], -math.inf)
            logits[:, 0] = 0.0
        t["logits"] = logits.to(dt)
        t["u"] = rand(B)
        for name in ("temperature", "top_k", "top_p", "min_p"):
            t[name] = c[name]
        if c["per_row"]:                # around the case's setting, double precision as a program's settings are
            near = 0.5 + rand(3, B).double()
            t["temperature"] = c["temperature"] * near[0]
            if c["top_k"]:
                t["top_k"] = (c["top_k"] * near[1]).ceil().long().clamp_(1, V)
            t["min_p"] = c["min_p"] * near[2]
            t["top_p"] = torch.full((B,), c["top_p"], device="cuda", dtype=torch.float64)
    return t


def _wider(a, b):
    return torch.promote_types(a.dtype, b.dtype)


def prepare(case, seed):
    return dict(case), _inputs(case, seed)


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    c, t = state
    if c["op"] in ("embedding", "norm") and c["what"] == "train":
        return _train(c, t)
    with torch.no_grad():
        return _FORWARD[c["op"]](c, t)


def _train(c, t):
    names = [n for n in ("x", "residual", "weight") if n in t]
    leaves = {**t, **{n: t[n].detach().requires_grad_() for n in names}}
    out = _FORWARD[c["op"]](c, leaves)
    grads = torch.autograd.grad(list(out.values()), [leaves[n] for n in names], [t["d" + n] for n in out])
    return {**{n: x.detach() for n, x in out.items()}, **{"d" + n: x for n, x in zip(names, grads)}}


class _Rows(torch.autograd.Function):
    """W[idx] with its gradient summed in float32 whatever W's type."""

    @staticmethod
    def forward(ctx, weight, idx, scale):
        ctx.save_for_backward(idx)
        ctx.scale, ctx.vocab, ctx.dtype = scale, weight.shape[0], weight.dtype
        return (weight[idx].float() * scale).to(weight.dtype)

    @staticmethod
    def backward(ctx, dy):
        idx, = ctx.saved_tensors
        dw = torch.zeros(ctx.vocab, dy.shape[-1], device=dy.device)
        return (dw.index_add_(0, idx, dy.float()) * ctx.scale).to(ctx.dtype), None, None


def _embedding_forward(c, t):
    if own:
        from mamba_ssm_benchmark_b200 import embedding
        return {"y": embedding(t["idx"], t["weight"], scale=c["scale"])}
    return {"y": _Rows.apply(t["weight"], t["idx"], c["scale"])}


def _norm_forward(c, t):
    x, residual, w = t["x"], t.get("residual"), t["weight"]
    if own:
        from mamba_ssm_benchmark_b200 import rms_norm, rms_norm_fp8
        out = (rms_norm_fp8 if c["what"] == "fp8" else rms_norm)(x, w, residual=residual)
        if c["what"] == "fp8":
            return dict(zip(("y8", "scale", "total"), out))
        return {"y": out} if residual is None else dict(zip(("y", "total"), out))
    out = {}
    total = x.float()
    if residual is not None:
        out["total"] = (total + residual.float()).to(_wider(x, residual))
        total = out["total"].float()
    y = total / (total.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w
    if c["what"] != "fp8":
        return {"y": y.to(x.dtype), **out}
    scale = y.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
    return {"y8": (y / scale[:, None]).to(torch.float8_e4m3fn), "scale": scale, **out}


def _linear_forward(c, t):
    act = None if c["act"] == "none" else c["act"]
    dt = getattr(torch, c["dtype"])
    if own:
        from mamba_ssm_benchmark_b200 import linear_fp8
        return {"y": linear_fp8(t["x8"], t["x_scale"], t["w8"], t["w_scale"], bias=t.get("bias"), activation=act,
                                residual=t.get("residual"), dtype=dt)}
    y = (t["x8"].float() @ t["w8"].float().T) * t["x_scale"][:, None] * t["w_scale"]
    if c["bias"]:
        y = y + t["bias"]
    if act == "silu":
        y = y / (1.0 + torch.exp(-y))
    if c["residual"]:
        y = y + t["residual"].float()
    return {"y": y.to(dt)}


def _sample_forward(c, t):
    if own:
        from mamba_ssm_benchmark_b200 import sample_tokens
        return {"token": sample_tokens(t["logits"], t["u"], temperature=t["temperature"], top_k=t["top_k"], top_p=t["top_p"],
                                       min_p=t["min_p"])}
    B, V = t["logits"].shape

    def setting(name, dtype=torch.float64):
        return torch.as_tensor(t[name], device=t["u"].device, dtype=dtype).expand(B)[:, None]

    # 64 bits: a token next to a border would be another one in 32
    logits, index = torch.sort(t["logits"].double(), dim=-1, descending=True, stable=True)
    gap, temp = logits - logits[:, :1], setting("temperature")
    w = torch.where(temp > 0, torch.exp(gap / temp.clamp_min(1e-300)), (gap == 0).double())
    greedy = (temp <= 0) & (torch.arange(V, device=w.device) > 0)
    k = setting("top_k", torch.long)
    w = w.masked_fill(greedy | ((k > 0) & (torch.arange(V, device=w.device) >= k)), 0.0)
    before = w.cumsum(-1) - w
    top_p = setting("top_p")
    w = w.masked_fill((top_p < 1) & (before >= top_p * w.sum(-1, keepdim=True)), 0.0)
    w = w.masked_fill(w < setting("min_p"), 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)
    run = w.cumsum(-1)
    return {"token": (run <= t["u"].double()[:, None] * run[:, -1:]).sum(-1)}


_FORWARD = {"embedding": _embedding_forward, "norm": _norm_forward, "linear": _linear_forward, "sample": _sample_forward}


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(c):
    e = 2 if c["dtype"] == "bfloat16" else 4
    if c["op"] == "embedding":
        T, V, C = c["tokens"], c["vocab"], c["C"]
        total = 8 * T + (min(T, V) + T) * C * e            # the rows in use, the result
        if c["what"] == "train":
            total += (T + V) * C * e                       # dy, the gradient
        return {"bytes": total, "flops": T * C * (2 if c["what"] == "train" else 1)}
    if c["op"] == "norm":
        n, res = c["rows"] * c["C"], c["residual"]
        r = 4 if res == "float32" else e                   # of the residual; the sum is as wide as the wider
        wide = max(e, r) if res != "none" else 0
        total = n * e + (n * r if res != "none" else 0) + n * wide + n * (1 if c["what"] == "fp8" else e) + 4 * c["C"]
        if c["what"] == "fp8":
            total += 4 * c["rows"]
        if c["what"] == "train":                           # dy, dtotal, the inputs' gradients, the weight's
            total += n * e + n * wide + n * e + (n * r if res not in ("none", c["dtype"]) else 0) + 4 * c["C"]
        return {"bytes": total, "flops": n * (5 + (10 if c["what"] == "train" else 0))}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        total = M * K + N * K + 4 * (M + N) + M * N * e * (2 if c["residual"] else 1) + (4 * N if c["bias"] else 0)
        return {"bytes": total, "flops": 2 * M * N * K}
    return {"bytes": c["B"] * (c["vocab"] * e + 12), "flops": 6 * c["B"] * c["vocab"]}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    return _EXACT[case["op"]](case, _inputs(case, seed))


def _embedding_exact(c, t):
    W = t["weight"].double()
    out = {"y": c["scale"] * W.index_select(0, t["idx"])}
    if c["what"] == "train":
        order = torch.argsort(t["idx"], stable=True)
        count = torch.bincount(t["idx"], minlength=c["vocab"])
        out["dweight"] = c["scale"] * torch.segment_reduce(t["dy"].double()[order], "sum", lengths=count, axis=0, initial=0.0)
    return out


def _norm_exact(c, t):
    x, w, out = t["x"].double(), t["weight"].double(), {}
    if "residual" in t:                 # the sum is a result in its type, and what is normed
        out["total"] = (x + t["residual"].double()).to(_wider(t["x"], t["residual"])).double()
        x = out["total"]
    rstd = (x.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
    n = x * rstd
    if c["what"] == "fp8":
        y = n * w
        scale = y.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
        # the nearest e4m3: three bits behind the leading one, steps of 2^-9 at least
        v = y / scale[:, None]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
        return {"y8": torch.round(v / step) * step, "scale": scale, **out}
    out["y"] = n * w
    if c["what"] == "forward":
        return out
    dn = t["dy"].double() * w
    out["dweight"] = (t["dy"].double() * n).sum(0)
    out["dx"] = rstd * (dn - n * (dn * n).mean(-1, keepdim=True))
    if "residual" in t:
        out["dx"] = out["dresidual"] = out["dx"] + t["dtotal"].double()
    return out


def _linear_exact(c, t):
    x, W = (t[n].double() * t[s].double()[:, None] for n, s in (("x8", "x_scale"), ("w8", "w_scale")))
    y = x @ W.T
    if "bias" in t:
        y = y + t["bias"].double()
    if c["act"] == "silu":
        y = y * torch.sigmoid(y)
    return {"y": y + t["residual"].double() if "residual" in t else y}


def _sample_exact(c, t):
    """Row by row from the definition: what is left after each rule, by rank."""
    logits, u = t["logits"].double(), t["u"].double().tolist()
    B, V = logits.shape
    at = {n: t[n].tolist() if isinstance(t[n], torch.Tensor) else [t[n]] * B for n in ("temperature", "top_k", "top_p", "min_p")}
    tokens = []
    for b in range(B):
        if at["temperature"][b] <= 0:
            tokens.append((logits[b] == logits[b].max()).nonzero()[:1, 0])
            continue
        p = torch.softmax(logits[b] / at["temperature"][b], 0)
        rank = torch.argsort(logits[b], descending=True, stable=True)
        if at["top_k"][b]:
            rank = rank[:at["top_k"][b]]
        q = p[rank]
        run = q.cumsum(0)
        if at["top_p"][b] < 1.0:
            rank = rank[torch.cat([torch.zeros_like(run[:1]), run[:-1]]) < at["top_p"][b] * run[-1]]
        rank = rank[p[rank] >= at["min_p"][b] * p.max()].sort().values
        run = p[rank].cumsum(0)
        tokens.append(rank[torch.searchsorted(run, u[b] * run[-1], right=True).clamp_max(len(rank) - 1)][None])
    return {"token": torch.cat(tokens)}


_EXACT = {"embedding": _embedding_exact, "norm": _norm_exact, "linear": _linear_exact, "sample": _sample_exact}
