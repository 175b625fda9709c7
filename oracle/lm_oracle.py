"""Definitions in float64 of the operators around a language model's mixers (embedding, RMS norm with a residual, 8-bit
rows and their products, sampling), written for the tests: plain torch on the CPU or the GPU, no kernels of this package."""

import torch

E4M3_MAX, TINY = 448.0, 1e-30


def rms_norm(x, weight=None, residual=None, eps=1e-5):
    """(y, total) with total as it is given by the caller's types: x and residual already summed where residual is None."""
    total = x if residual is None else x + residual
    n = total / torch.sqrt(total.square().mean(-1, keepdim=True) + eps)
    return n if weight is None else n * weight, total


def e4m3(v):
    """The nearest e4m3 value, even at ties: four significant bits, steps of 2^-9 at least, at most 448."""
    v = v.double()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def quantize(y):
    """(values, scale) of rows of y."""
    scale = y.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
    return e4m3(y / scale[..., None]), scale


def linear(x8, xs, w8, ws, bias=None, silu=False, residual=None):
    """(y, sum of the absolute terms of every product), in float64."""
    x, w = x8.double() * xs.double()[:, None], w8.double() * ws.double()[:, None]
    pre = x @ w.T
    size = x.abs() @ w.abs().T
    if bias is not None:
        pre = pre + bias.double()
    y = pre * torch.sigmoid(pre) if silu else pre
    return (y if residual is None else y + residual.double()), size, pre


def embedding_grad(idx, dy, vocab, scale):
    """(gradient, sum of absolute terms)."""
    d = dy.double() * scale
    out = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device)
    return out.index_add(0, idx, d), out.index_add(0, idx, d.abs())


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: logits (V), numbers.  The token, or -1."""
    l = logits.double()
    if bool(l.isnan().any()) or float(l.max()) == float("-inf") or temperature != temperature:
        return -1
    if temperature <= 0:
        return int((l == l.max()).nonzero()[0])
    w = torch.where(l == l.max(), 1.0, torch.exp((l - l.max()) / temperature)).nan_to_num(0.0)
    rank = torch.sort(l, descending=True, stable=True).indices
    if top_k > 0:
        rank = rank[:top_k]
    if top_p < 1.0:
        run = w[rank].cumsum(0)
        before = torch.cat([torch.zeros_like(run[:1]), run[:-1]])
        keep = before < top_p * run[-1]
        keep[0] = True
        rank = rank[keep]
    rank = rank[w[rank] >= min_p].sort().values
    run = w[rank].cumsum(0)
    return int(rank[min(int((run <= u * run[-1]).sum()), int((run < run[-1]).sum()))])
