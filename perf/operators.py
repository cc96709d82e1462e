"""Measured cases of the operators around microscaled 4-bit experts: routing of logits with
scores, balance bias and groups; the residual's addition with RMSNorm and 8-bit rows; the
experts' products over 4-bit weights, and the quantisation of those weights.

A case names its operator in `op`:
  route   logits to experts and weights; with `train` also the gradient of the logits
  norm    stream + delta, its RMSNorm, and the norm's rows in e4m3 with a power-of-two scale
          per 32 values; with `train` the gradients of both inputs and of the norm's weight
  experts SwiGLU experts of routed tokens, weights in e2m1 and activations in e4m3 (w4a8) or
          e2m1 (w4a4), all in blocks of 32 with a power-of-two scale; with `train` one
          micro-batch of a gradient accumulation: gradients of x, of the routing weights and,
          straight-through, of the expert weights
  quant   the values that expert weights stand for in 4 bits
"""
import math
import os
import sys

import torch

own = False

BLOCK = 32                       # values that share a scale
EMAX = {"e2m1": 2, "e4m3": 8}    # exponent of the largest power of two of the element type
TOP = {"e2m1": 6.0, "e4m3": 448.0}
ACT = {"w4a8": "e4m3", "w4a4": "e2m1"}
EPS = 1e-5
TINY = 1e-20                     # added to the sum that renormalises the weights


def listed():
    return [
        # one token of one sequence being generated, the default 16 experts
        _route("route_1", T=1, E=16, k=2),
        # a long prompt: sigmoid scores, balance bias, 4 of 8 groups
        _route("route_prompt_16384", T=16384, E=64, k=8, scores="sigmoid", bias=True, groups=8, topk_groups=4, scale=2.5),
        # a training micro-batch of odd length
        _route("route_train_4099", T=4099, E=48, k=6, bias=True, train=True),
        # a batched decode step of 48 sequences
        _norm("norm_48", T=48, d=2048),
        # a long prompt
        _norm("norm_prompt_16384", T=16384, d=2048),
        # a training micro-batch with the residual stream held in 32 bits
        _norm("norm_train_8191", T=8191, d=2048, f32=True, train=True),
        # one token of one sequence being generated
        _experts("experts_1", T=1, mx="w4a4"),
        # a batched decode step of 48 sequences
        _experts("experts_48", T=48, mx="w4a8"),
        # a prompt of odd length
        _experts("experts_777", T=777, mx="w4a4"),
        # a batch of 8 prompts of 2048 tokens
        _experts("experts_16384", T=16384, mx="w4a8"),
        # a training micro-batch of 2 x 1021 tokens
        _experts("experts_train_2042", T=2042, mx="w4a8", train=True),
        # the weights of all experts after an optimizer step
        _quant("quant_weights", E=16, K=2048, N=2816),
    ]


def _route(name, T, E, k, scores="softmax", bias=False, groups=1, topk_groups=1, scale=1.0, train=False):
    return dict(name=name, op="route", T=T, E=E, k=k, scores=scores, bias=bias, groups=groups, topk_groups=topk_groups,
                scale=scale, train=train)


def _norm(name, T, d, f32=False, train=False):
    return dict(name=name, op="norm", T=T, d=d, f32=f32, train=train)


def _experts(name, T, mx, E=16, k=2, d=2048, F=2816, train=False):
    return dict(name=name, op="experts", T=T, E=E, k=k, d=d, F=F, mx=mx, train=train)


def _quant(name, E, K, N):
    return dict(name=name, op="quant", E=E, K=K, N=N)


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("route", "norm", "experts", "experts", "quant"))
    train = rng.random() < 0.35
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        E = groups * rng.randint(2 if groups > 1 else 4, 64 // groups)
        keep = rng.randint(1, groups)
        k = rng.randint(1, min(8, keep * (E // groups)))
        c = _route("", _log(rng, 1, 16384), E, k, rng.choice(("softmax", "sigmoid")), rng.random() < 0.6, groups, keep,
                   rng.choice((1.0, 2.5)), train)
    elif op == "norm":
        d = 64 * _log(rng, 2, 96)
        c = _norm("", _log(rng, 1, max(1, min(16384, 16384 * 2048 // d))), d, rng.random() < 0.4, train)
    elif op == "experts":
        E = rng.randint(1, 16)
        d, F = 64 * _log(rng, 2, 32), _log(rng, 24, 2816)
        T = _log(rng, 1, 2048 if train else 16384)
        c = _experts("", T, rng.choice(tuple(ACT)), E, rng.randint(1, min(2, E)), d, F // 8 * 8 if train else F, train)
    else:
        c = _quant("", rng.randint(1, 16), 32 * _log(rng, 2, 64), _log(rng, 16, 2816))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=g)

    s = dict(case=dict(case))
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        s["logits"] = normal(T, E, std=1.5, dtype=torch.float32)
        s["bias"] = normal(E, std=0.05, dtype=torch.float32) if case["bias"] else None
        s["dw"] = normal(T, k, dtype=torch.float32)
    elif case["op"] == "norm":
        T, d = case["T"], case["d"]
        stream = torch.float32 if case["f32"] else torch.bfloat16
        s["x"], s["delta"] = normal(T, d, std=2.0, dtype=stream), normal(T, d)
        s["g"] = (1.0 + 0.1 * normal(d, dtype=torch.float32)).to(torch.bfloat16)
        if case["train"]:
            s["dh"], s["dn"] = normal(T, d, dtype=stream), normal(T, d)
    elif case["op"] == "experts":
        T, E, k, d, F = case["T"], case["E"], case["k"], case["d"], case["F"]
        s["x"] = normal(T, d)
        lg = normal(T, E, dtype=torch.float32) + 0.3 * normal(E, dtype=torch.float32)
        v, s["idx"] = torch.topk(lg, k, dim=-1)
        s["w"] = torch.softmax(v, -1).to(torch.bfloat16)
        s["cap"] = int(torch.bincount(s["idx"].reshape(-1), minlength=E).max())
        # the values that 4-bit weights stand for
        for name, shape in (("w1", (E, d, F)), ("w2", (E, d, F)), ("w3", (E, F, d))):
            s[name] = _values(normal(*shape, std=0.02))
        if case["train"]:
            s["dy"] = normal(T, d)
    else:
        s["w"] = normal(case["E"], case["K"], case["N"], std=0.02)
    return s


# ---------------------------------------------------------------- plain forms

def _blocks(v, fmt):
    """Values of v (.., K) rounded to blocks of 32 along K (ragged ends as if zeros followed):
    scale 2^(floor(log2(largest)) - emax), elements to nearest even, saturating.  Returns
    (elements, scales)."""
    K = v.shape[-1]
    b = torch.nn.functional.pad(v.float(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = b.abs().amax(-1, keepdim=True)
    # the power of two below a positive float: its exponent bits
    power = (amax.view(torch.int32) & 0x7F800000).view(torch.float32)
    scale = (power * 2.0 ** -EMAX[fmt]).clamp(min=2.0 ** -126)
    a = b / scale
    if fmt == "e2m1":
        m = a.abs()
        step = torch.where(m < 2.0, 0.5, torch.where(m < 4.0, 1.0, 2.0))
    else:
        low = (a.view(torch.int32) & 0x7F800000).view(torch.float32)
        step = low.clamp(min=2.0 ** -6) * 0.125
    q = (torch.round(a / step) * step).clamp(-TOP[fmt], TOP[fmt])
    return q.flatten(-2)[..., :K], scale.squeeze(-1)


def _q(v, fmt):
    q, scale = _blocks(v, fmt)
    return q * scale.repeat_interleave(BLOCK, -1)[..., : v.shape[-1]]


def _values(w):
    """The values of weights (E, K, N) in 4-bit blocks along K."""
    return _q(w.transpose(1, 2), "e2m1").transpose(1, 2).contiguous().to(w.dtype)


def _plain_route(s):
    c = s["case"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    lg = s["logits"].double()  # 64 bits: two choices may be closer than 32 bits tell apart
    if c["scores"] == "sigmoid":
        p = 1.0 / (1.0 + torch.exp(-lg))
    else:
        p = torch.exp(lg - lg.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    choice = p + s["bias"].double() if s["bias"] is not None else p
    if G > 1:
        grouped = choice.view(T, G, E // G)
        best = torch.sort(grouped, dim=-1, descending=True).values[..., :2].sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, : c["topk_groups"]]
        on = torch.zeros(T, G, dtype=torch.bool, device=lg.device).scatter_(1, kept, True)
        choice = torch.where(on[:, :, None], grouped, -math.inf).view(T, E)
    idx = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
    chosen = torch.gather(p, 1, idx)
    total = chosen.sum(-1, keepdim=True) + TINY
    w = c["scale"] * chosen / total
    out = {"idx": idx, "w": w.float()}
    if c["train"]:
        dw = s["dw"].double()
        ds = c["scale"] / total * (dw - (dw * chosen).sum(-1, keepdim=True) / total)
        if c["scores"] == "sigmoid":
            dl = torch.zeros_like(p).scatter_(1, idx, ds * chosen * (1.0 - chosen))
        else:
            dl = p * (torch.zeros_like(p).scatter_(1, idx, ds) - (ds * chosen).sum(-1, keepdim=True))
        out["dlogits"] = dl.float()
    return out


def _plain_norm(s):
    c = s["case"]
    h = (s["x"].float() + s["delta"].float()).to(s["x"].dtype)
    hf, g = h.float(), s["g"].float()
    r = 1.0 / torch.sqrt((hf * hf).mean(-1, keepdim=True) + EPS)
    n = (hf * r * g).to(torch.bfloat16)
    if not c["train"]:
        q, scale = _blocks(n, "e4m3")
        return {"h": h, "n": n, "q": q.to(torch.float8_e4m3fn), "scale": scale.to(torch.float8_e8m0fnu)}
    dn = s["dn"].float()
    gd = g * dn
    dx = s["dh"].float() + r * gd - r ** 3 * hf * (gd * hf).mean(-1, keepdim=True)
    return {"h": h, "n": n, "dx": dx.to(h.dtype), "ddelta": dx.to(s["delta"].dtype),
            "dg": (dn * hf * r).sum(0).to(s["g"].dtype)}


def _plain_experts(s):
    c = s["case"]
    T, E, k, d = c["T"], c["E"], c["k"], c["d"]
    fmt, cap = ACT[c["mx"]], s["cap"]
    w = s["w"].float()
    w1, w2, w3 = s["w1"].float(), s["w2"].float(), s["w3"].float()
    # each expert's rows one below the other, in blocks of `cap`
    flat = s["idx"].reshape(-1)
    chosen = flat[:, None] == torch.arange(E, device=flat.device)
    at = torch.gather(chosen.cumsum(0) - 1, 1, flat[:, None]).squeeze(1)
    slot = flat * cap + at
    token = torch.arange(T * k, device=flat.device) // k

    def rows(v):
        return torch.zeros(E * cap, d, device=v.device).index_copy_(0, slot, v).view(E, cap, d)

    x = rows(_q(s["x"], fmt)[token])
    gate, up = torch.bmm(x, w1), torch.bmm(x, w2)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    h = _q(gate * sig * up, fmt)
    yr = torch.bmm(h, w3).view(-1, d)[slot]
    y = (yr.view(T, k, d) * w[:, :, None]).sum(1)
    if not c["train"]:
        return {"y": y.to(torch.bfloat16)}
    dyt = s["dy"].float()[token]
    dy = rows(dyt * w.reshape(-1, 1))
    dh = torch.bmm(dy, w3.transpose(1, 2).contiguous())
    dgate, dup = dh * up * sig * (1.0 + gate * (1.0 - sig)), dh * gate * sig
    dx = torch.bmm(dgate, w1.transpose(1, 2).contiguous()) + torch.bmm(dup, w2.transpose(1, 2).contiguous())
    xt = x.transpose(1, 2).contiguous()
    bf = torch.bfloat16
    return {"y": y.to(bf), "dx": dx.view(-1, d)[slot].view(T, k, d).sum(1).to(bf),
            "dw": (yr * dyt).sum(-1).view(T, k).to(bf), "dw1": torch.bmm(xt, dgate).to(bf),
            "dw2": torch.bmm(xt, dup).to(bf), "dw3": torch.bmm(h.transpose(1, 2).contiguous(), dy).to(bf)}


# ---------------------------------------------------------------- the framework's calls

def _kmoe():
    path = os.path.join(os.getcwd(), "kolmogorov-moe-architecture_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kmoe
    return kmoe


def _own_route(s):
    kmoe, c = _kmoe(), s["case"]
    how = dict(scores=c["scores"], bias=s["bias"], groups=c["groups"], topk_groups=c["topk_groups"], scale=c["scale"])
    if not c["train"]:
        r = kmoe.ops.route_topk(s["logits"], c["k"], **how)
        return {"idx": r.idx, "w": r.w}
    logits = s["logits"].detach().requires_grad_(True)
    w, idx = kmoe.route_topk(logits, c["k"], **how)
    (dl,) = torch.autograd.grad(w, logits, s["dw"])
    return {"idx": idx, "w": w.detach(), "dlogits": dl}


def _own_norm(s):
    kmoe, c = _kmoe(), s["case"]
    if not c["train"]:
        r = kmoe.ops.add_rmsnorm(s["x"], s["delta"], s["g"], EPS, quant="e4m3")
        d = c["d"]
        # codes and scale exponents as the values they stand for
        return {"h": r.h, "n": r.n, "q": r.q[:, :d].view(torch.float8_e4m3fn),
                "scale": r.scale[:, : d // BLOCK].view(torch.float8_e8m0fnu)}
    x, delta, g = (s[n].detach().requires_grad_(True) for n in ("x", "delta", "g"))
    h, n = kmoe.add_rms_norm(x, delta, g, EPS)
    dx, ddelta, dg = torch.autograd.grad((h, n), (x, delta, g), (s["dh"], s["dn"]))
    return {"h": h.detach(), "n": n.detach(), "dx": dx, "ddelta": ddelta, "dg": dg}


def _own_experts(s):
    kmoe, c = _kmoe(), s["case"]
    experts = s.get("experts")
    if experts is None:  # the module that a program keeps
        with torch.device("meta"):
            experts = kmoe.GroupedExperts(c["E"], c["d"], c["F"])
        experts.mx = c["mx"]
        for n in ("w1", "w2", "w3"):
            setattr(experts, n, torch.nn.Parameter(s[n], requires_grad=c["train"]))
        s["experts"] = experts
    if not c["train"]:
        with torch.no_grad():
            return {"y": experts(s["x"], s["idx"], s["w"])}
    x, w = s["x"].detach().requires_grad_(True), s["w"].detach().requires_grad_(True)
    y = experts(x, s["idx"], w)
    g = torch.autograd.grad(y, (x, w, experts.w1, experts.w2, experts.w3), s["dy"])
    return dict(zip(("y", "dx", "dw", "dw1", "dw2", "dw3"), (y.detach(), *g)))


def run(state):
    op = state["case"]["op"]
    if op == "route":
        return _own_route(state) if own else _plain_route(state)
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    if op == "experts":
        return _own_experts(state) if own else _plain_experts(state)
    return {"w": _kmoe().ops.fake_quant_mx_cols(state["w"]) if own else _values(state["w"])}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        # logits in, experts and weights out; their gradient in and the logits' out
        bytes_ = T * (4 * E + 12 * k) + (T * (4 * k + 4 * E) if case["train"] else 0)
        return {"bytes": bytes_, "flops": T * E * (10 if case["train"] else 5)}
    if case["op"] == "norm":
        T, d = case["T"], case["d"]
        es = 4 if case["f32"] else 2
        # stream and delta in, stream and norm out; codes and scales, or the gradients
        per = es + 2 + es + 2 + ((es + 2 + es + 2) if case["train"] else 1 + 1 / BLOCK)
        return {"bytes": T * d * per + 2 * d, "flops": T * d * (20 if case["train"] else 8)}
    if case["op"] == "experts":
        T, E, k, d, F = case["T"], case["E"], case["k"], case["d"], case["F"]
        met = E * (1.0 - (1.0 - k / E) ** T)  # experts with a token
        weights = 3 * d * F
        bytes_ = 4 * T * d + T * k * 10 + met * weights * (0.5 + 1 / BLOCK)
        flops = 2.0 * T * k * weights
        if case["train"]:
            # dy in, dx out, the weights' gradients out
            bytes_ += 4 * T * d + T * k * 2 + E * weights * 2
            flops *= 3
        return {"bytes": bytes_, "flops": flops}
    n = case["E"] * case["K"] * case["N"]
    return {"bytes": 4 * n, "flops": 4 * n}


# ---------------------------------------------------------------- the same in 64 bits

def _round64(v, fmt):
    """_blocks() in 64 bits, from the numbers' exponents."""
    K = v.shape[-1]
    b = torch.nn.functional.pad(v.double(), (0, -K % BLOCK)).unflatten(-1, (-1, BLOCK))
    e = torch.frexp(b.abs().amax(-1, keepdim=True)).exponent.double() - 1 - EMAX[fmt]
    scale = torch.pow(torch.full_like(e, 2.0), e.clamp(min=-126))
    a = b / scale
    bits, low = (1, 0) if fmt == "e2m1" else (3, -6)  # mantissa bits, smallest normal exponent
    ulp = torch.pow(torch.full_like(a, 2.0), (torch.frexp(a).exponent.double() - 1).clamp(min=low) - bits)
    q = (a / ulp).round() * ulp
    q = torch.minimum(q.abs(), torch.full_like(q, TOP[fmt])) * torch.sign(q)
    return (q * scale).flatten(-2)[..., :K], q.flatten(-2)[..., :K], scale.squeeze(-1)


def _exact_route(s):
    c = s["case"]
    lg = s["logits"].double()
    p = torch.sigmoid(lg) if c["scores"] == "sigmoid" else torch.softmax(lg, -1)
    choice = p if s["bias"] is None else p + s["bias"].double()
    if c["groups"] > 1:
        size = c["E"] // c["groups"]
        value = torch.stack([choice[:, i * size:(i + 1) * size].topk(min(2, size)).values.sum(-1)
                             for i in range(c["groups"])], 1)
        off = torch.ones_like(value, dtype=torch.bool)
        off.scatter_(1, value.topk(c["topk_groups"]).indices, False)
        choice = choice.masked_fill(off.repeat_interleave(size, 1), -math.inf)
    idx = choice.topk(c["k"]).indices
    p = p.detach().requires_grad_(True)
    lp = lg.detach().requires_grad_(True)
    p = torch.sigmoid(lp) if c["scores"] == "sigmoid" else torch.softmax(lp, -1)
    v = p.gather(1, idx)
    w = c["scale"] * v / (v.sum(-1, keepdim=True) + TINY)
    out = {"idx": None, "w": w.detach()}
    if c["train"]:
        out["dlogits"] = torch.autograd.grad(w, lp, s["dw"].double())[0]
    return out


def _exact_norm(s):
    c = s["case"]
    h = (s["x"].double() + s["delta"].double()).to(s["x"].dtype).double().requires_grad_(True)
    g = s["g"].double().requires_grad_(True)
    n = g * h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    if not c["train"]:
        _, q, scale = _round64(n.detach().to(torch.bfloat16), "e4m3")
        return {"h": h.detach(), "n": n.detach(), "q": q, "scale": scale}
    dh, dg = torch.autograd.grad(n, (h, g), s["dn"].double())
    dx = s["dh"].double() + dh
    return {"h": h.detach(), "n": n.detach(), "dx": dx, "ddelta": dx, "dg": dg}


def _exact_experts(s):
    c = s["case"]
    fmt, k, d = ACT[c["mx"]], c["k"], c["d"]
    x, w = s["x"].double(), s["w"].double().reshape(-1)
    flat = s["idx"].reshape(-1)
    y = torch.zeros(c["T"], d, device=x.device, dtype=x.dtype)
    dx, dw = torch.zeros_like(y), torch.zeros_like(w)
    grads = {n: [] for n in ("dw1", "dw2", "dw3")}
    for e in range(c["E"]):
        a = (flat == e).nonzero().squeeze(1)
        t = a // k
        w1, w2, w3 = (s[n][e].double() for n in ("w1", "w2", "w3"))
        xq = _round64(x[t], fmt)[0]
        gate, up = xq @ w1, xq @ w2
        sig = torch.sigmoid(gate)
        h = _round64(gate * sig * up, fmt)[0]
        yr = h @ w3
        y.index_add_(0, t, yr * w[a, None])
        if c["train"]:
            dyt = s["dy"].double()[t]
            dyr = dyt * w[a, None]
            dw[a] = (dyt * yr).sum(-1)
            dh = dyr @ w3.t()
            dgate, dup = dh * up * (sig + gate * sig * (1.0 - sig)), dh * gate * sig
            dx.index_add_(0, t, dgate @ w1.t() + dup @ w2.t())
            for n, v in (("dw1", xq.t() @ dgate), ("dw2", xq.t() @ dup), ("dw3", h.t() @ dyr)):
                grads[n].append(v)
    if not c["train"]:
        return {"y": y}
    return {"y": y, "dx": dx, "dw": dw.view(c["T"], k), **{n: torch.stack(v) for n, v in grads.items()}}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        return {"w": _round64(s["w"].transpose(1, 2), "e2m1")[0].transpose(1, 2)}
    return {"route": _exact_route, "norm": _exact_norm, "experts": _exact_experts}[case["op"]](s)
