"""Routing of logits (scores, balance bias, groups, renormalisation) and its backward against
64-bit restatements."""
import pytest
import torch

import kmoe
from kmoe import ops
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
F32 = torch.float32
HALF_F32 = torch.finfo(F32).eps / 2
INF = float("inf")
# weights: scores in f32 (the logit's difference to the largest, at most 16 here, is rounded:
# 16 half steps of the exponential; exp, six sums of a pair and the quotient: 9 half steps more);
# the sum they are divided by has the same error and those of four additions, the quotient
# and the scale round once each
W_ERR = (2 * 25 + 6) * HALF_F32


def logits_of(dev, T, E, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(T, E, generator=g)).to(dev)


def bias_of(dev, E, seed=1):
    return (0.1 * torch.randn(E, generator=torch.Generator().manual_seed(seed))).to(dev)


CASES = [
    # T, E, k, scores, bias, groups, topk_groups, group_top, renorm, scale
    (1, 1, 1, "softmax", False, 1, 1, 2, True, 1.0),
    (1, 16, 2, "softmax", False, 1, 1, 2, True, 1.0),
    (3, 5, 5, "sigmoid", True, 1, 1, 2, False, 0.5),
    (33, 13, 3, "softmax", True, 1, 1, 2, True, 2.5),
    (129, 64, 8, "sigmoid", True, 8, 4, 2, True, 2.5),
    (70, 63, 7, "softmax", True, 7, 1, 1, False, 1.0),
    (65, 24, 4, "sigmoid", False, 12, 2, 2, True, 1.0),
    (40, 32, 2, "softmax", False, 32, 3, 2, True, 1.0),   # groups of one expert
    (513, 48, 6, "softmax", True, 2, 1, 2, True, 1.0),
]


def kwargs(dev, c):
    _, E, _, scores, bias, groups, keep, top, renorm, scale = c
    return dict(scores=scores, bias=bias_of(dev, E) if bias else None, groups=groups, topk_groups=keep, group_top=top,
                renorm=renorm, scale=scale)


@pytest.mark.parametrize("c", CASES)
def test_forward(dev, c):
    T, E, k = c[:3]
    lg = logits_of(dev, T, E, seed=T + E)
    kw = kwargs(dev, c)
    r = ops.route_topk(lg, k, hist=True, **kw)
    cpu = {**kw, "bias": None if kw["bias"] is None else kw["bias"].cpu()}
    idx, w = M.route(lg.cpu(), k, kind=cpu.pop("scores"), **cpu)
    assert torch.equal(r.idx.cpu(), idx)
    assert bool(((r.w.double().cpu() - w).abs() <= W_ERR * w.abs()).all())
    hb = ops.router_block_tokens(T)
    want = torch.stack([torch.bincount(b.reshape(-1), minlength=E) for b in r.idx.cpu().split(hb)])
    assert torch.equal(r.block_counts.cpu().long(), want)


def test_near_ties_are_told_apart(dev):
    """Choices that differ by less than 32 bits resolve, and equal ones: lowest index first."""
    T, E = 64, 16
    base = torch.zeros(T, E, dtype=F32)
    base[:, 5] = 2.0
    base[:, 9] = 2.0                      # tie of 5 and 9
    base[:, 3] = 2.0 + 2.0 ** -22         # one step of a float above
    bias = torch.zeros(E)
    r = ops.route_topk(base.to(dev), 3, scores="sigmoid", bias=bias.to(dev))
    assert r.idx.cpu().tolist() == [[3, 5, 9]] * T
    # a bias that closes the gap of two scores but for 1e-12
    s = torch.sigmoid(torch.tensor([0.3, -0.7], dtype=F32).double())
    b = float((s[0] - s[1]).float())
    lg = torch.full((T, E), -5.0)
    lg[:, 2], lg[:, 11] = 0.3, -0.7
    bias[11] = b
    exact = float(s[1]) + float(bias[11].double()) > float(s[0])
    r = ops.route_topk(lg.to(dev), 1, scores="sigmoid", bias=bias.to(dev))
    assert r.idx.cpu().flatten().tolist() == [11 if exact else 2] * T


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_masked_rows_infinities_and_nan(dev, scores, groups, keep):
    E, k = 16, 3
    lg = logits_of(dev, 8, E).cpu()
    lg[0] = -INF                       # nothing left
    lg[1, 2:] = -INF                   # fewer experts than k
    lg[2, 4:12] = torch.finfo(F32).min
    lg[3] = torch.finfo(F32).min
    lg[4, 3] = INF
    lg[5, 7] = float("nan")
    lg[6, ::2] = -INF
    bias = bias_of("cpu", E)
    bias[:] += 1.0
    kw = dict(groups=groups, topk_groups=keep)
    r = ops.route_topk(lg.to(dev), k, scores=scores, bias=bias.to(dev), **kw)
    idx, w = M.route(lg, k, kind=scores, bias=bias, **kw)
    got = r.idx.cpu()
    assert int(got.min()) >= 0 and int(got.max()) < E
    assert all(len(set(row)) == k for row in got.tolist())
    assert torch.equal(got, idx)
    wd = r.w.double().cpu()
    assert torch.equal(wd.isnan(), w.isnan())
    assert bool(((wd - w).abs().nan_to_num() <= W_ERR * w.abs().nan_to_num() + 1e-45).all())
    assert not wd[0].any()
    dl = ops.route_topk_bwd(lg.to(dev), r.idx, torch.ones(8, k, device=dev), scores=scores)
    assert bool(dl[:4].isfinite().all()) and not dl[0].any()


@pytest.mark.parametrize("c", CASES)
def test_backward(dev, c):
    T, E, k, scores, _, _, _, _, renorm, scale = c
    lg = logits_of(dev, T, E, seed=T)
    kw = kwargs(dev, c)
    x = lg.clone().requires_grad_(True)
    w, idx = kmoe.route_topk(x, k, **kw)
    dw = logits_of(dev, T, k, seed=7)
    (dl,) = torch.autograd.grad(w, x, dw)
    x64 = lg.double().cpu().requires_grad_(True)
    w64 = M.route_weights(x64, idx.cpu(), scores, renorm, scale)
    (want,) = torch.autograd.grad(w64, x64, dw.double().cpu())
    # f32 sums over the token's experts and k weights: exp and quotient (8 steps of 2^-24), sums
    # of E and of k terms; the terms of a row, before they cancel, are at most scale max|dw|
    # (without renorm times s <= 1)
    bound = (16 + E + 3 * k) * 2.0 ** -24 * 4 * abs(scale) * dw.double().cpu().abs().amax(1, keepdim=True)
    assert bool(((dl.double().cpu() - want).abs() <= bound).all())
    add = torch.ones(T, E, device=dev)
    ops.route_topk_bwd(lg, idx, dw, scores, renorm, scale, dlogits=add)
    assert bool(((add - 1) - dl).abs().max() <= 2.0 ** -22 * (1 + float(dl.abs().max())))


@pytest.mark.parametrize("scores,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_backward_against_differences(dev, scores, renorm):
    T, E, k, h = 6, 12, 3, 2.0 ** -7
    lg = logits_of(dev, T, E, std=1.0)
    _, idx = kmoe.route_topk(lg, k, scores=scores, renorm=renorm)
    dw = logits_of(dev, T, k, seed=3)
    dl = ops.route_topk_bwd(lg, idx, dw, scores, renorm).double().cpu()
    f = lambda l: (M.route_weights(l, idx.cpu(), scores, renorm, 1.0) * dw.double().cpu()).sum()  # noqa: E731
    x = lg.double().cpu()
    for t in range(T):
        for e in range(E):
            d = torch.zeros_like(x)
            d[t, e] = h
            num = float(f(x + d) - f(x - d)) / (2 * h)
            # central difference: h^2 / 6 of the third derivative, below 8 max|dw| k here
            assert abs(num - float(dl[t, e])) <= h * h / 6 * 8 * k * float(dw.abs().max()) + 1e-5


def test_strides_types_streams_and_graph(dev):
    lg = logits_of(dev, 100, 32)
    want = ops.route_topk(lg, 4, scores="sigmoid", groups=4, topk_groups=2)
    wide = torch.randn(100, 64, device=dev)
    wide[:, 16:48] = lg
    got = ops.route_topk(wide[:, 16:48], 4, scores="sigmoid", groups=4, topk_groups=2)
    assert torch.equal(got.idx, want.idx) and torch.equal(got.w, want.w)
    lb = lg.to(torch.bfloat16)
    a, b = ops.route_topk(lb, 4), ops.route_topk(lb.float(), 4)
    assert torch.equal(a.idx, b.idx) and torch.equal(a.w, b.w)
    buf = lg.clone()
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=s):
        r = ops.route_topk(buf, 4, scores="sigmoid", groups=4, topk_groups=2, hist=True)
    for seed in (1, 2, 3):
        new = logits_of(dev, 100, 32, seed=seed)
        eager = ops.route_topk(new, 4, scores="sigmoid", groups=4, topk_groups=2, hist=True)
        buf.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(r.idx, eager.idx) and torch.equal(r.w, eager.w)
        assert torch.equal(r.block_counts, eager.block_counts)


def test_order_of_close_choices(dev):
    """Rows whose neighbours differ by parts of an f32 step of the scores, among ordinary rows:
    the order is that of 64 bits."""
    T, E, k = 257, 24, 6
    lg = logits_of("cpu", T, E, seed=5)
    g = torch.Generator().manual_seed(6)
    for t in range(0, T, 3):
        i, j = torch.randperm(E, generator=g)[:2].tolist()
        lg[t, i] = lg[t].max()
        lg[t, j] = torch.nextafter(lg[t, i], torch.tensor(INF))
    # a bias that equals the difference of two scores to f32: 64 bits tell them apart
    bias = torch.zeros(E)
    s = torch.sigmoid(lg.double())
    bias[3] = (s[1, 4] - s[1, 3]).float()
    for kind in ("softmax", "sigmoid"):
        for kw in (dict(), dict(bias=bias), dict(groups=4, topk_groups=2), dict(groups=8, topk_groups=3, group_top=1, bias=bias)):
            dkw = {n: v.to(dev) if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
            r = ops.route_topk(lg.to(dev), k, scores=kind, **dkw)
            assert torch.equal(r.idx.cpu(), M.route(lg, k, kind=kind, **kw)[0])


def test_large_and_empty(dev):
    lg = logits_of(dev, 20001, 64)
    bias = bias_of(dev, 64)
    r = ops.route_topk(lg, 8, scores="sigmoid", bias=bias, groups=8, topk_groups=4, hist=True)
    s = torch.sigmoid(lg.double())
    c = (s + bias.double()).view(-1, 8, 8)
    keep = c.topk(2, -1).values.sum(-1).topk(4, -1).indices
    on = torch.zeros(20001, 8, dtype=torch.bool, device=dev).scatter_(1, keep, True)
    idx = torch.where(on[:, :, None], c, -INF).view(-1, 64).topk(8, -1).indices
    assert torch.equal(r.idx, idx)
    assert int(r.block_counts.sum()) == 20001 * 8
    e = ops.route_topk(lg[:0], 4, hist=True)
    assert e.idx.shape == (0, 4) and e.block_counts is None
    assert ops.route_topk_bwd(lg[:0], e.idx, e.w).shape == (0, 64)


def test_router_module(dev):
    """The layer's router with grouped sigmoid scores and a balance bias: forward and gradients
    against 64-bit autograd at the kernel's choice."""
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=16, moe_top_k=4, d_ff_expert=64, moe_router_scores="sigmoid",
                                 moe_router_groups=4, moe_router_topk_groups=2, moe_router_scale=2.5, moe_balance_bias=True)
    router = kmoe.Router(cfg).to(dev).to(torch.bfloat16)
    assert router.balance_bias.dtype == F32 and router.balance_bias.is_cuda
    assert "balance_bias" in router.state_dict()
    with torch.no_grad():
        router.balance_bias.copy_(bias_of("cpu", 16))
    x = torch.randn(2, 30, 128, device=dev, dtype=torch.bfloat16)
    with torch.no_grad():
        w0, idx0, lg0 = router(x)
    xg = x.clone().requires_grad_(True)
    w, idx, lg = router(xg)
    assert torch.equal(idx, idx0) and torch.equal(w, w0)
    dw = torch.randn_like(w)
    got = torch.autograd.grad(w, (xg, router.router[0].weight, router.router[2].weight), dw)
    d64 = lambda t: t.detach().double().cpu().requires_grad_(True)  # noqa: E731
    leaves = [d64(x), d64(router.router[0].weight), d64(router.router[2].weight)]
    l64 = torch.nn.functional.silu(leaves[0].reshape(60, 128) @ leaves[1].t()) @ leaves[2].t()
    w64 = M.route_weights(l64, idx.reshape(60, 4).cpu(), "sigmoid", True, 2.5)
    want = torch.autograd.grad(w64, leaves, dw.reshape(60, 4).double().cpu())
    for a, b in zip(got, want):
        # bf16 roundings: the hidden gradient and the result
        assert float((a.double().cpu() - b).norm() / b.norm()) <= 4 * torch.finfo(torch.bfloat16).eps / 2
    plain = kmoe.Router(kmoe.AdvancedMoEConfig(d_model=128, n_experts=16, d_ff_expert=64))
    assert plain.spec is None and "balance_bias" not in plain.state_dict()


def test_layer_with_aux_losses(dev):
    """Aux losses and routed gradients meet in the logit gradient: the sum of both parts."""
    kw = dict(d_model=128, n_experts=8, moe_top_k=2, d_ff_expert=64, moe_router_scores="sigmoid", moe_router_groups=2)
    layer = kmoe.MoELayer(kmoe.AdvancedMoEConfig(**kw)).to(dev).to(torch.bfloat16).train()
    x = torch.randn(1, 70, 128, device=dev, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    w_out = layer.router.router[2].weight

    def grad(with_y, with_aux):
        y = layer(x)
        loss = (y * dy).sum().float() * with_y + layer.aux_loss * with_aux
        return torch.autograd.grad(loss, w_out)[0].double()
    both, a, b = grad(1.0, 1.0), grad(1.0, 0.0), grad(0.0, 1.0)
    assert float(a.norm()) > 0 and float(b.norm()) > 0
    assert float((both - a - b).norm()) <= 4 * torch.finfo(torch.bfloat16).eps / 2 * float(a.norm() + b.norm())


def test_refusals(dev):
    lg = logits_of(dev, 4, 16)
    for kw, err in ((dict(k=0), kmoe.KmoeError), (dict(k=9), kmoe.KmoeError), (dict(k=2, groups=3), kmoe.KmoeError),
                    (dict(k=5, groups=4, topk_groups=1), kmoe.KmoeError), (dict(k=2, groups=4, topk_groups=5), kmoe.KmoeError),
                    (dict(k=2, groups=2, group_top=3), kmoe.KmoeError), (dict(k=2, scores="tanh"), ValueError),
                    (dict(k=2, bias=torch.zeros(3, device=dev)), ValueError), (dict(k=2, bias=torch.zeros(16)), ValueError)):
        with pytest.raises(err):
            ops.route_topk(lg, **kw)
    with pytest.raises(kmoe.KmoeError):
        ops.route_topk(logits_of(dev, 2, 65), 2)
    with pytest.raises(ValueError):
        ops.route_topk(lg[0], 2)
    with pytest.raises(ValueError):
        ops.route_topk_bwd(lg, torch.zeros(4, 2, dtype=torch.int64, device=dev), torch.zeros(4, 3, device=dev))


@pytest.mark.parametrize("scores,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("k,same,std", [(1, False, 1.5), (4, True, 1.5), (4, False, 6.0), (8, False, 1.5)])
def test_gradients_that_nearly_vanish(dev, scores, renorm, k, same, std):
    """One expert, or equal gradients of the weights, renormalised: only the 1e-20 is left of the
    gradient.  Confident scores: 1 - s is small.  Held against the terms that remain when the sums
    that cancel are taken exactly, not against the largest gradient."""
    T, E, scale, tiny = 2000, 16, 2.5, 1e-20
    lg = logits_of(dev, T, E, seed=k, std=std)
    idx = ops.route_topk(lg, k, scores=scores, renorm=renorm).idx
    dw = logits_of(dev, T, 1 if same else k, seed=9).expand(T, k).contiguous()
    got = ops.route_topk_bwd(lg, idx, dw, scores, renorm, scale).double().cpu()
    l, i, g = lg.double().cpu(), idx.cpu(), dw.double().cpu()
    s = torch.sigmoid(l) if scores == "sigmoid" else torch.softmax(l, -1)
    on = torch.zeros(T, E, dtype=torch.bool).scatter_(1, i, True)
    ge = torch.zeros(T, E, dtype=torch.float64).scatter_(1, i, g)
    sc = s.gather(1, i)
    S = sc.sum(1, keepdim=True) + tiny
    diff = ge[:, :, None] - g[:, None, :]                  # (T, E, k)
    D, Dabs = (diff * sc[:, None, :]).sum(-1), (diff.abs() * sc[:, None, :]).sum(-1)
    slope = s * torch.sigmoid(-l)
    if renorm:
        c, cabs = torch.where(on, (D + tiny * ge) / S, 0.0), torch.where(on, (Dabs + tiny * ge.abs()) / S, 0.0)
        m, mabs = (sc * g).sum(1, keepdim=True) / S, (sc * g.abs()).sum(1, keepdim=True) / S
        want, terms = (slope / S * c, slope / S * cabs) if scores == "sigmoid" else (
            s / S * (c - tiny * m), s / S * (cabs + tiny * mabs))
    elif scores == "sigmoid":
        want = terms = torch.where(on, ge * slope, 0.0)
    else:
        U = torch.where(on, 0.0, s).sum(1, keepdim=True)
        want, terms = s * (D + ge * U), s * (Dabs + ge.abs() * U)
    # scores: the logit's difference to the largest (below 32 at std 1.5, 64 at 6, asserted) is rounded, the
    # exponential off by 2 half steps of f32, the sum of E and the quotient: far + E + 4 half steps;
    # a term has at most three of them (s, S, s_i, or S twice), a difference, sums of E + k and eight products
    far = 64 if std > 2 else 32
    assert float((l.amax(1, keepdim=True) - l).max()) < far
    steps = 3 * (far + E + 4) + E + k + 10
    assert bool(((got - scale * want).abs() <= steps * HALF_F32 * scale * terms.abs() + 1e-37).all())


ROUTED = [
    dict(moe_router_scores="sigmoid", moe_router_groups=4, moe_router_topk_groups=2, moe_router_scale=2.5, moe_balance_bias=True),
    dict(moe_router_scores="softmax", moe_router_renorm=False, moe_router_scale=1.5),
    dict(moe_router_scores="sigmoid", moe_router_renorm=False, moe_balance_bias=True),
]


def layer64(x, w_in, w_out, w1, w2, w3, idx, cfg, mx):
    """(y, aux) of the layer in 64 bits at the choice idx, differentiable."""
    T, k = idx.shape
    E = w1.shape[0]
    lg = torch.nn.functional.silu(x @ w_in.t()) @ w_out.t()
    w = M.route_weights(lg, idx, cfg.moe_router_scores, cfg.moe_router_renorm, cfg.moe_router_scale)
    if mx:
        y = M.experts(x, idx, w, w1, w2, w3, mx)
    else:
        y = torch.zeros(T, x.shape[1], dtype=torch.float64)
        for e in range(E):
            t, j = (idx == e).nonzero(as_tuple=True)
            y = y.index_add(0, t, (torch.nn.functional.silu(x[t] @ w1[e]) * (x[t] @ w2[e])) @ w3[e] * w[t, j][:, None])
    f = torch.bincount(idx.reshape(-1), minlength=E).double() / (T * k)
    aux = (cfg.moe_load_balance_loss_weight * E * (f * torch.softmax(lg, -1).mean(0)).sum()
           + cfg.moe_router_z_loss_weight * torch.logsumexp(lg, -1).square().mean())
    return y, aux


# Gradients through the experts have the bf16 roundings of their backward: w dy, the two
# pre-activations, dh, dgate / dup, a row's dx, the sum (seven); through the router those of the expert rows (the
# weights' gradient is their product with dy), of the hidden gradient and the result (three); 4-bit
# experts: elements of h on the other side of a border, 2e-3 of the norm.
ROUTED_TOL = 10 * torch.finfo(torch.bfloat16).eps / 2


@pytest.mark.parametrize("case", ROUTED)
@pytest.mark.parametrize("mx", [None, "w4a8"])
@pytest.mark.parametrize("with_y,with_aux", [(1.0, 0.0), (0.0, 1.0), (1.0, 1.0)])
def test_layer_gradients_against_64_bits(dev, case, mx, with_y, with_aux):
    """Every gradient of a layer with its own routing, of its output, of its aux losses, and of both (scaled
    so that both count), at the kernel's choice of experts."""
    torch.manual_seed(3)
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=16, moe_top_k=4, d_ff_expert=64, moe_mx=mx, **case)
    layer = kmoe.MoELayer(cfg).to(dev).to(torch.bfloat16).train()
    with torch.no_grad():
        layer.router.router[2].weight.mul_(4.0)  # logits that differ
        if layer.router.balance_bias is not None:
            layer.router.balance_bias.copy_(bias_of("cpu", 16))
    x = torch.randn(1, 150, 128, device=dev, dtype=torch.bfloat16)
    dy = torch.randn_like(x)
    with torch.no_grad():
        idx = layer.router.route(x[0]).idx.cpu()
    ge = layer.grouped_experts
    xg = x.clone().requires_grad_(True)
    leaves = [xg, layer.router.router[0].weight, layer.router.router[2].weight, ge.w1, ge.w2, ge.w3]
    l64 = [v.detach().double().cpu().requires_grad_(True) for v in leaves]
    y64, aux64 = layer64(l64[0][0], *l64[1:], idx, cfg, mx)
    dy64 = dy.double().cpu()[0]
    # the aux losses' share of the router's gradient is made as large as the output's
    ga, = torch.autograd.grad(aux64, l64[2], retain_graph=True)
    gy, = torch.autograd.grad((y64 * dy64).sum(), l64[2], retain_graph=True)
    c = with_aux * float(gy.norm() / ga.norm())
    want = torch.autograd.grad(with_y * (y64 * dy64).sum() + c * aux64, l64, allow_unused=True)
    y = layer(xg)
    assert abs(float(layer.aux_loss.detach()) - float(aux64)) <= 1e-4 * float(aux64)
    assert float((y.detach().double().cpu()[0] - y64).norm() / y64.norm()) <= 4 * torch.finfo(torch.bfloat16).eps / 2
    got = torch.autograd.grad((y.float() * dy.float()).sum() * with_y + c * layer.aux_loss, leaves)
    for name, a, b in zip(("dx", "dw_in", "dw_out", "dw1", "dw2", "dw3"), got, want):
        if not with_y and name[:3] in ("dw1", "dw2", "dw3"):
            assert not a.any()
            continue
        err = float((a.double().cpu() - b).norm() / b.norm())
        assert err <= ROUTED_TOL + (2e-3 if mx else 0.0), (name, err)


@pytest.mark.parametrize("case", ROUTED)
def test_block_gradients_against_64_bits(dev, case):
    """The block of an f32 stream and a delta not yet added: h and delta get the same gradient, that of the
    formula, next to the norm's, the router's and the experts'."""
    torch.manual_seed(4)
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=16, moe_top_k=4, d_ff_expert=64, mod_enabled=False,
                                 residual_dropout=0.0, **case)
    blk = kmoe.MoEFFNBlock(cfg).to(dev).train()
    r = blk.ffn.router
    with torch.no_grad():
        r.router[2].weight.mul_(4.0)
        blk.ffn_norm.weight.add_(0.1 * torch.randn_like(blk.ffn_norm.weight))
        if r.balance_bias is not None:
            r.balance_bias.copy_(bias_of("cpu", 16))
        for p in blk.parameters():  # values that bf16 holds: the kernels cast them
            p.copy_(p.to(torch.bfloat16))
    h, delta, dout = (torch.randn(1, 150, 128, device=dev) for _ in range(3))
    with torch.no_grad():
        idx = r.route(ops.rmsnorm((h + delta)[0], blk.ffn_norm.weight, cfg.norm_eps).n).idx.cpu()
    ge = blk.ffn.grouped_experts
    hg, dg = h.clone().requires_grad_(True), delta.clone().requires_grad_(True)
    leaves = [hg, blk.ffn_norm.weight, r.router[0].weight, r.router[2].weight, ge.w1, ge.w2, ge.w3]
    l64 = [v.detach().double().cpu().requires_grad_(True) for v in leaves]
    s64 = l64[0][0] + delta.double().cpu()[0]
    n64 = M.add_norm(s64, None, l64[1], cfg.norm_eps)[1]
    y64, aux64 = layer64(n64, *l64[2:], idx, cfg, None)
    d64 = dout.double().cpu()[0]
    ga, = torch.autograd.grad(aux64, l64[3], retain_graph=True)
    gy, = torch.autograd.grad((y64 * d64).sum(), l64[3], retain_graph=True)
    c = float(gy.norm() / ga.norm())
    want = list(torch.autograd.grad((y64 * d64).sum() + c * aux64, l64))  # without the residual's dout
    out = blk(hg, dg)
    assert blk.last_path == "fused_train"
    g = torch.autograd.grad((out * dout).sum() + c * blk.aux_loss, leaves + [dg])
    assert torch.equal(g[0], g[-1])
    got = [(g[0] - dout).double().cpu()] + [v.double().cpu() for v in g[1:-1]]
    for name, a, b in zip(("dh", "dg", "dw_in", "dw_out", "dw1", "dw2", "dw3"), got, want):
        # (and the normalised rows are rounded to bf16 first, their gradient too: two more)
        err = float((a - b).norm() / b.norm())
        assert err <= ROUTED_TOL * 1.2, (name, err)
