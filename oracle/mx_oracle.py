"""64-bit restatements of microscaled numbers, of the experts over them, of the routing of
logits and of the residual add with RMSNorm (CPU or GPU torch; test infrastructure)."""
from __future__ import annotations

import torch

BLOCK = 32
EMAX = {"e4m3": 8, "e2m1": 2}
TOP = {"e4m3": 448.0, "e2m1": 6.0}
MANT = {"e4m3": 3, "e2m1": 1}
EMIN = {"e4m3": -6, "e2m1": 0}
ACT = {"w4a8": "e4m3", "w4a4": "e2m1"}


def elements(a, fmt):
    """a (64 bits) to the element grid: nearest, ties to even, saturating."""
    e = torch.frexp(a).exponent.double() - 1
    ulp = torch.exp2(e.clamp(min=EMIN[fmt]) - MANT[fmt])
    q = torch.round(a / ulp) * ulp
    return torch.sign(a) * q.abs().clamp(max=TOP[fmt])


def scale_codes(v, fmt):
    """Scale bytes of the blocks of v (.., n*32): floor(log2(amax)) - emax + 127, at least 0;
    255 where a value is not finite."""
    b = v.double().unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(torch.where(amax.isfinite(), amax, 1.0)).exponent.double() - 1, -1000.0)
    code = (e.clamp(min=-127) - EMAX[fmt] + 127).clamp(min=0)
    return torch.where(b.isfinite().all(-1), code, 255.0).to(torch.int64)


def quant(v, fmt):
    """(values, elements, scale bytes) of v (.., K) in blocks along K; a ragged last block is
    filled with zeros."""
    K = v.shape[-1]
    p = torch.nn.functional.pad(v.double(), (0, -K % BLOCK))
    code = scale_codes(p, fmt)
    s = torch.exp2(code.double() - 127).unsqueeze(-1)
    bad = (code == 255).unsqueeze(-1)
    q = torch.where(bad, 0.0, elements(torch.where(bad, 0.0, p.unflatten(-1, (-1, BLOCK))) / s, fmt))
    val = torch.where(bad, float("nan"), q * s)
    return val.flatten(-2)[..., :K], q.flatten(-2)[..., :K], code


def q_cols(w):
    """Values of weights (E, K, N) in e2m1 blocks along K."""
    return quant(w.transpose(1, 2), "e2m1")[0].transpose(1, 2)


class _Through(torch.autograd.Function):
    """Rounded values forward, the gradient unchanged backward."""

    @staticmethod
    def forward(ctx, v, fmt):
        return quant(v, fmt)[0]

    @staticmethod
    def backward(ctx, g):
        return g, None


class _ThroughCols(torch.autograd.Function):
    @staticmethod
    def forward(ctx, w):
        return q_cols(w)

    @staticmethod
    def backward(ctx, g):
        return g


def swiglu_rows(x, w1, w2, w3, fmt):
    """One expert on rows x (n, d), straight-through."""
    xq = _Through.apply(x, fmt)
    w1, w2, w3 = (_ThroughCols.apply(w[None])[0] for w in (w1, w2, w3))
    g, u = xq @ w1, xq @ w2
    return _Through.apply(torch.nn.functional.silu(g) * u, fmt) @ w3


def experts(x, idx, w, w1, w2, w3, mx, slot_on=None):
    """y (T, d) of the token-choice experts; slot_on (T, k) drops assignments."""
    fmt = ACT[mx]
    y = torch.zeros(x.shape[0], w3.shape[2], dtype=torch.float64, device=x.device)
    for e in range(w1.shape[0]):
        on = idx == e
        if slot_on is not None:
            on = on & slot_on
        t, j = on.nonzero(as_tuple=True)
        if len(t):
            y = y.index_add(0, t, swiglu_rows(x[t], w1[e], w2[e], w3[e], fmt) * w[t, j][:, None])
    return y


def scores(logits, kind):
    l = logits.double()
    if kind == "sigmoid":
        return torch.where(l == -float("inf"), 0.0, torch.sigmoid(l))
    empty = (l == -float("inf")).all(-1, keepdim=True)
    return torch.where(empty, 0.0, torch.softmax(torch.where(empty, 0.0, l), -1))


def route(logits, k, kind="softmax", bias=None, groups=1, topk_groups=1, group_top=2, renorm=True, scale=1.0):
    """(idx, w) token by token, in Python numbers."""
    s = scores(logits, kind)
    inf = float("inf")
    T, E = logits.shape
    size = E // groups
    idx = torch.empty(T, k, dtype=torch.int64)
    for t in range(T):
        c = []
        for e in range(E):
            v = float(s[t, e]) + (float(bias[e].double()) if bias is not None else 0.0)
            c.append(-inf if float(logits[t, e]) == -inf else v)
        nan = [v != v for v in c]  # ranks above every number
        key = [(1, 0.0) if nan[e] else (0, c[e]) for e in range(E)]
        allowed = list(range(E))
        if groups > 1:
            val = []
            for g in range(groups):
                m = range(g * size, (g + 1) * size)
                if any(nan[e] for e in m):
                    val.append((1, 0.0))
                    continue
                best = sorted((c[e] for e in m if c[e] > -inf), reverse=True)[:group_top]
                val.append((0, sum(best) if best else -inf))
            keep = sorted(range(groups), key=lambda g: (-val[g][0], -val[g][1], g))[:topk_groups]
            allowed = [e for e in range(E) if e // size in keep]
        order = sorted(allowed, key=lambda e: (-key[e][0], -key[e][1], e))
        idx[t] = torch.tensor(order[:k])
    p = torch.gather(s, 1, idx)
    w = scale * (p / (p.sum(-1, keepdim=True) + 1e-20) if renorm else p)
    return idx, w


def route_weights(logits, idx, kind, renorm, scale):
    """The weights at a fixed choice, differentiable in the logits (64 bits)."""
    s = torch.sigmoid(logits) if kind == "sigmoid" else torch.softmax(logits, -1)
    p = torch.gather(s, 1, idx)
    return scale * (p / (p.sum(-1, keepdim=True) + 1e-20) if renorm else p)


def add_norm(x, delta, g, eps):
    """(h, n) with h rounded to the stream's type (x's), its gradient unchanged."""
    h = x if delta is None else x + delta
    return h, g * h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
