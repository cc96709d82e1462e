"""Microscaled rows, weights and experts (4-bit weights, e4m3 or e2m1 activations) against
64-bit restatements: codes bit for bit, products within the rounding of their sums, the
layer, its straight-through gradients, and the calls that are refused."""
import pytest
import torch

import kmoe
from kmoe import ops
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HALF_BF16 = torch.finfo(BF).eps / 2


def rnd(dev, *shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(*shape, generator=g)).to(dtype).to(dev)


def used(r: ops.MXRows):
    """The scale bytes of the padded row (those behind are not written)."""
    return r.scale[:, :(r.K + 127) // 128 * 4]


def decode(r: ops.MXRows):
    """(elements, scale bytes) of coded rows on the CPU, K padded to 128 included."""
    s = used(r).cpu().long()
    if r.fmt == "e4m3":
        return r.q.cpu().view(torch.float8_e4m3fn).double(), s
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
    q = r.q.cpu().long()
    return grid[torch.stack([q & 15, q >> 4], -1).flatten(-2)], s


def special_rows():
    """One block of 32 a row: midpoints, saturation, zeros, subnormal and huge values, NaN, inf."""
    rows = [torch.zeros(32), torch.full((32,), -0.0)]
    mids = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5., 6., 7., 7.9, .5, 1., 1.5, 2., 3., 4.])
    for e in (-130, -126, -100, -3, 0, 5, 100, 124):
        rows.append(torch.cat([mids, -mids]) * 2.0 ** e)
    m8 = torch.tensor([448., 449., 464., 480., 500., 511., 256., 17., 18., 19., 1.0625, 0.015625, 0.0078125, 0.001953125,
                       0.0009765625, 0.0029296875])
    for e in (-120, -8, 0, 100):
        rows.append(torch.cat([m8, -m8]) * 2.0 ** e)
    for bad in (float("nan"), float("inf"), -float("inf")):
        r = torch.linspace(-1, 1, 32)
        r[7] = bad
        rows.append(r)
    return torch.stack(rows).to(BF)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_quant_special_values(dev, fmt):
    x = special_rows()
    r = ops.quant_rows_mx(x.to(dev), fmt)
    q, s = decode(r)
    _, eq, es = M.quant(x, fmt)
    assert torch.equal(s[:, :1], es)
    assert torch.equal(q[:, :32], eq)
    assert not q[:, 32:].any() and not s[:, 1:].any()  # padding to 128
    val = ops.dequant_rows_mx(r).double().cpu()
    want = M.quant(x, fmt)[0].to(BF).double()
    assert torch.equal(val.isnan(), want.isnan()) and torch.equal(val.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 64), (7, 192), (130, 2048), (33, 4096)])
def test_quant_rows(dev, fmt, rows, K):
    x = rnd(dev, rows, K, seed=rows + K)
    x[0, :32] *= 2.0 ** -30  # blocks of very different sizes
    q, s = decode(ops.quant_rows_mx(x, fmt))
    _, eq, es = M.quant(x.cpu(), fmt)
    assert torch.equal(s[:, :K // 32], es) and torch.equal(q[:, :K], eq)
    assert not q[:, K:].any() and not s[:, K // 32:].any()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_quant_gathered_rows_and_row_count(dev, fmt):
    x = rnd(dev, 50, 128, seed=1)
    index = torch.tensor([49, 0, 0, 7, 31], dtype=torch.int32, device=dev)
    got = ops.quant_rows_mx(x, fmt, row_index=index)
    want = ops.quant_rows_mx(x[index.long()], fmt)
    assert torch.equal(got.q, want.q) and torch.equal(used(got), used(want))
    # a strided view, as a slice of a wider activation
    wide = rnd(dev, 50, 256, seed=2)
    assert torch.equal(ops.quant_rows_mx(wide[:, 64:192], fmt).q, ops.quant_rows_mx(wide[:, 64:192].contiguous(), fmt).q)
    # rows past the count are left as they were
    from kmoe._lib import call, ptr
    q, s = torch.full_like(want.q, 7), torch.full_like(want.scale, 9)
    n = torch.tensor([3], dtype=torch.int32, device=dev)
    call("kmoe_quant_rows_mx", ptr(x), ptr(index), 5, ptr(n), 128, ops.MX_FORMATS[fmt], ptr(q), ptr(s), ops._stream(x))
    assert torch.equal(q[:3], want.q[:3]) and bool((q[3:] == 7).all()) and bool((s[3:] == 9).all())
    # -1 decodes to zeros
    back = ops.dequant_rows_mx(want, torch.tensor([2, -1, 4], dtype=torch.int32, device=dev))
    full = ops.dequant_rows_mx(want)
    assert torch.equal(back[0], full[2]) and torch.equal(back[2], full[4]) and not back[1].any()


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("E,K,N", [(1, 1, 1), (2, 33, 5), (3, 64, 352), (2, 100, 131), (2, 100, 132), (4, 256, 40), (1, 31, 4)])
def test_fake_quant_weights(dev, dtype, E, K, N):
    w = rnd(dev, E, K, N, seed=K, std=0.02, dtype=dtype)
    if K > 1:
        w[0, 1, 0] = 0.0
    got = ops.fake_quant_mx_cols(w)
    assert torch.equal(got.double().cpu(), M.q_cols(w.cpu()))
    t = rnd(dev, E, N, K, seed=K, std=0.02, dtype=dtype).transpose(1, 2)  # a transposed view
    assert torch.equal(ops.fake_quant_mx_cols(t), ops.fake_quant_mx_cols(t.contiguous()))


def weights(dev, E, d, F, seed=0, dtype=BF):
    return tuple(rnd(dev, *s, seed=seed + i, std=0.05, dtype=dtype) for i, s in enumerate([(E, d, F), (E, d, F), (E, F, d)]))


def dropped(x, w, fmt):
    """What the matrix instruction may drop of a sum x (n, K) @ w (K, N) besides f32 rounding.  With
    an 8-bit operand it aligns products (eight consecutive K at a time, as measured) to the
    largest of them and keeps 13 bits below it: a product of 2^-13 of the largest still counts,
    one of 2^-14 does not.  So each product is off by less than 2^-13 of the largest of its group,
    and 64 of them, in whatever groups, by less than 64 times that of the largest of the 64.
    Products of e2m1 pairs are multiples of 1/4 up to 36: nothing is dropped."""
    out = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64)
    if fmt == "e4m3":
        for k in range(0, x.shape[1], 64):
            out += 64 * 2.0 ** -13 * (x[:, k:k + 64, None].abs() * w[None, k:k + 64].abs()).amax(1)
    return out


# rows of each expert: none, one, a whole tile, several tiles, one more than a tile
PRODUCTS = [
    (1, 64, 8, [1]),
    (2, 64, 40, [0, 3]),
    (3, 192, 100, [5, 0, 70]),
    (4, 256, 352, [64, 65, 1, 200]),
    (2, 128, 128, [257, 600]),
    (5, 320, 264, [300, 0, 256, 12, 513]),
    (64, 64, 64, [3] * 63 + [0]),
]


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("case", range(len(PRODUCTS)))
def test_products(dev, fmt, case):
    """Gate/up and down rows.  The sums are exact products in f32: K additions, each off by at
    most 2^-24 of the sum of magnitudes so far, and what dropped() says.  h passes a quantiser: the coded value lies
    between the codes of the two ends of that interval, where both ends have the block's scale."""
    E, d, F, counts = PRODUCTS[case]
    print(f"products E={E} d={d} F={F} rows={counts} {fmt}", flush=True)
    A = sum(counts)
    w = weights(dev, E, d, F, seed=case)
    pw = ops.pack_weights_mx(*w)
    offsets = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    tokens = torch.randperm(A + 3, generator=torch.Generator().manual_seed(case))[:A].to(torch.int32).to(dev)
    x = rnd(dev, A + 3, d, seed=100 + case)
    xq = ops.quant_rows_mx(x, fmt)
    h, gu = ops.gemm_gate_up_mx(xq, tokens, offsets, pw, A, save_gu=True)
    # permuted rows give the same bits, and so does the call without the saved values
    perm = ops.MXRows(xq.q[tokens.long()], xq.scale[tokens.long()], d, fmt)
    h2 = ops.gemm_gate_up_mx(perm, None, offsets, pw, A)
    assert torch.equal(h.q, h2.q) and torch.equal(used(h), used(h2))
    y = ops.gemm_down_mx(h, offsets, pw, A)
    xv = M.quant(x.cpu(), fmt)[0][tokens.cpu().long()]
    wv = [M.q_cols(t.cpu()) for t in w]
    hq, hs = decode(h)
    Fp = (F + 127) // 128 * 128
    assert not hq[:, F:].any()
    guc = gu.double().cpu().view(A, Fp // 128, 2, 128)
    gate_s, up_s = guc[:, :, 0].reshape(A, Fp)[:, :F], guc[:, :, 1].reshape(A, Fp)[:, :F]
    lo = 0
    for e, n in enumerate(counts):
        r = slice(lo, lo + n)
        lo += n
        if not n:
            continue
        w1, w2, w3 = (t[e] for t in wv)
        g, u = xv[r] @ w1, xv[r] @ w2
        mag1, mag2 = xv[r].abs() @ w1.abs(), xv[r].abs() @ w2.abs()
        eg = d * 2.0 ** -24 * mag1 + dropped(xv[r], w1, fmt)
        eu = d * 2.0 ** -24 * mag2 + dropped(xv[r], w2, fmt)
        assert bool(((gate_s[r] - g).abs() <= eg + HALF_BF16 * (g.abs() + eg)).all())
        assert bool(((up_s[r] - u).abs() <= eu + HALF_BF16 * (u.abs() + eu)).all())
        hv = torch.nn.functional.silu(g) * u
        # |silu'| < 1.1; exp, reciprocal and three products: 8 steps of 2^-23 each
        eh = 1.1 * eg * (u.abs() + eu) + (torch.nn.functional.silu(g).abs() + 1.1 * eg) * eu + 2.0 ** -20 * hv.abs()
        pad = -F % 32
        P = lambda v: torch.nn.functional.pad(v, (0, pad)).unflatten(-1, (-1, 32))  # noqa: E731
        amax = P(hv).abs().amax(-1)
        slack = P(eh).amax(-1)
        low, high = (torch.frexp((amax - slack).clamp(min=1e-300)).exponent, torch.frexp(amax + slack).exponent)
        code = hs[r][:, :amax.shape[1]]
        want_low = (low.long() - 1 - M.EMAX[fmt] + 127).clamp(min=0)
        want_high = (high.long() - 1 - M.EMAX[fmt] + 127).clamp(min=0)
        assert bool(((code >= want_low) & (code <= want_high)).all())
        s = torch.exp2(code.double() - 127).unsqueeze(-1)
        a = M.elements((P(hv) - P(eh)) / s, fmt)
        b = M.elements((P(hv) + P(eh)) / s, fmt)
        q = P(hq[r][:, :F])
        assert bool(((q >= a) & (q <= b)).all())
        # down, from the coded h
        hval = (q * s).flatten(-2)[:, :F]
        yv, mag = hval @ w3, hval.abs() @ w3.abs()
        ey = Fp * 2.0 ** -24 * mag + dropped(hval, w3, fmt)
        assert bool(((y[r].double().cpu() - yv).abs() <= ey + HALF_BF16 * (yv.abs() + ey)).all())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_products_leave_rows_past_the_last(dev, fmt):
    """max_rows may exceed the routed rows (a capacity drop): the rows behind stay."""
    E, d, F = 2, 128, 96
    from kmoe._lib import call, ptr
    pw = ops.pack_weights_mx(*weights(dev, E, d, F))
    offsets = torch.tensor([0, 5, 37], dtype=torch.int32, device=dev)
    xq = ops.quant_rows_mx(rnd(dev, 100, d), fmt)
    fresh = ops.gemm_gate_up_mx(xq, None, offsets, pw, 100)
    q, s = torch.full_like(fresh.q, 3), torch.full_like(fresh.scale, 5)
    call("kmoe_gemm_gate_up_mx", ptr(xq.q), ptr(xq.scale), ops.MX_FORMATS[fmt], 100, None, ptr(offsets), E, d, F, 100,
         ptr(pw.w13), ptr(pw.s13), ptr(q), ptr(s), None, ops._stream(q))
    assert bool((q[37:] == 3).all()) and bool((s[37:] == 5).all()) and torch.equal(q[:37], fresh.q[:37])
    y = torch.full((100, d), 2.0, device=dev, dtype=BF)
    call("kmoe_gemm_down_mx", ptr(q), ptr(s), ops.MX_FORMATS[fmt], ptr(offsets), E, d, F, 100, ptr(pw.w3), ptr(pw.s3),
         ptr(y), ops._stream(y))
    assert bool((y[37:] == 2.0).all()) and bool(y[:37].isfinite().all())


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_nan_rows_and_missing_rows(dev, fmt):
    """A NaN or infinity in a row makes that row NaN and no other; row_token -1 is a zero row."""
    E, d, F = 1, 128, 64
    pw = ops.pack_weights_mx(*weights(dev, E, d, F))
    x = rnd(dev, 70, d)
    clean = ops.quant_rows_mx(x, fmt)
    offsets = torch.tensor([0, 70], dtype=torch.int32, device=dev)
    y0 = ops.gemm_down_mx(ops.gemm_gate_up_mx(clean, None, offsets, pw, 70), offsets, pw, 70)
    x[3, 5] = float("nan")
    x[66, 127] = float("inf")
    y = ops.gemm_down_mx(ops.gemm_gate_up_mx(ops.quant_rows_mx(x, fmt), None, offsets, pw, 70), offsets, pw, 70)
    bad = torch.zeros(70, dtype=torch.bool, device=dev)
    bad[[3, 66]] = True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], y0[~bad])
    tok = torch.arange(70, dtype=torch.int32, device=dev)
    tok[10] = -1
    yt = ops.gemm_down_mx(ops.gemm_gate_up_mx(clean, tok, offsets, pw, 70), offsets, pw, 70)
    assert not yt[10].any() and torch.equal(yt[11:], y0[11:])


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("A", [3, 200])
def test_rows_past_the_last_are_zeros(dev, fmt, A):
    """row_token entries outside of the gathered rows, in the small-row kernel and in a tile."""
    pw = ops.pack_weights_mx(*weights(dev, 1, 128, 64))
    x = ops.quant_rows_mx(rnd(dev, 5, 128), fmt)
    token = torch.arange(A, dtype=torch.int32) % 5
    bad = [1, 2] if A == 3 else [1, 64, 130, 199]
    token[bad] = torch.tensor([5, 5000, -1, 77777], dtype=torch.int32)[:len(bad)]
    off = torch.tensor([0, A], dtype=torch.int32, device=dev)
    h = ops.gemm_gate_up_mx(x, token.to(dev), off, pw, A)
    good = [i for i in range(A) if i not in bad]
    assert not h.q[bad].any() and bool(h.q[good].any(1).all())
    one = ops.gemm_gate_up_mx(x, torch.tensor([0], dtype=torch.int32, device=dev), off.clamp(max=1), pw, 1)
    assert torch.equal(h.q[0], one.q[0])


def test_products_do_not_depend_on_the_run(dev):
    E, d, F, T, k = 4, 256, 352, 300, 2
    ex = kmoe.GroupedExperts(E, d, F).to(dev).to(BF)
    ex.mx = "w4a8"
    x = rnd(dev, T, d)
    idx = torch.topk(rnd(dev, T, E, seed=3, dtype=torch.float32), k, 1).indices
    w = torch.softmax(rnd(dev, T, k, seed=4, dtype=torch.float32), 1)
    with torch.no_grad():
        first = ex(x, idx, w)
        for _ in range(3):
            assert torch.equal(ex(x, idx, w), first)


def config(E=4, d=128, F=96, k=2, **kw):
    base = dict(d_model=d, n_experts=E, d_ff_expert=F, moe_top_k=k, residual_dropout=0.0, mod_enabled=False)
    return kmoe.AdvancedMoEConfig(**{**base, **kw})


def f64(t):
    return t.detach().double().cpu()


# y: two roundings to bf16 (the expert rows, the sum) of at most half a step each, and single
# elements of h that land on the other side of a quantiser's border (one step of it, 2^-3 for
# e4m3 and 2^-1 for e2m1, for at most one element in 10^4: 2e-3 of the norm)
TOL_Y = 2 * HALF_BF16 + 2e-3


@pytest.mark.parametrize("mx", ["w4a8", "w4a4"])
@pytest.mark.parametrize("E,T,k,d,F", [(1, 1, 1, 64, 8), (4, 1, 2, 128, 96), (4, 37, 2, 192, 100), (8, 500, 3, 256, 352)])
def test_experts_forward(dev, mx, E, T, k, d, F):
    ex = kmoe.GroupedExperts(E, d, F).to(dev).to(BF)
    ex.mx = mx
    x = rnd(dev, T, d, seed=T)
    idx = torch.topk(rnd(dev, T, E, seed=3, dtype=torch.float32), k, 1).indices
    w = torch.softmax(rnd(dev, T, k, seed=4, dtype=torch.float32), 1)
    with torch.no_grad():
        y = ex(x, idx, w)
    want = M.experts(f64(x), idx.cpu(), f64(w), f64(ex.w1), f64(ex.w2), f64(ex.w3), mx)
    assert float((f64(y) - want).norm() / want.norm()) <= TOL_Y


@pytest.mark.parametrize("mx", ["w4a8", "w4a4"])
@pytest.mark.parametrize("E,T,k,d,F", [(1, 3, 1, 64, 8), (4, 61, 2, 128, 96), (4, 300, 2, 256, 256)])
def test_experts_gradients(dev, mx, E, T, k, d, F):
    """Straight-through gradients against the same formula in 64 bits.  bf16 roundings on the way
    to the last gradient: w dy, the two pre-activations, dh, dgate / dup, the row's dx, the sum."""
    ex = kmoe.GroupedExperts(E, d, F).to(dev).to(BF)
    ex.mx = mx
    x = rnd(dev, T, d, seed=T).requires_grad_(True)
    idx = torch.topk(rnd(dev, T, E, seed=3, dtype=torch.float32), k, 1).indices
    w = torch.softmax(rnd(dev, T, k, seed=4, dtype=torch.float32), 1).requires_grad_(True)
    dy = rnd(dev, T, d, seed=9)
    got = torch.autograd.grad(ex(x, idx, w), (x, w, ex.w1, ex.w2, ex.w3), dy)
    leaves = [f64(t).requires_grad_(True) for t in (x, w, ex.w1, ex.w2, ex.w3)]
    want = torch.autograd.grad(M.experts(leaves[0], idx.cpu(), *leaves[1:], mx), leaves, f64(dy))
    for name, a, b in zip(("dx", "dw", "dw1", "dw2", "dw3"), got, want):
        assert a.shape == b.shape
        err = float((f64(a) - b).norm() / b.norm())
        assert err <= 7 * HALF_BF16 + 2e-3, (name, err)


def test_experts_gradient_against_differences(dev):
    """y is linear in the routing weights and, over representable changes, in w3."""
    E, T, k, d, F = 2, 24, 1, 64, 64
    ex = kmoe.GroupedExperts(E, d, F).to(dev).to(torch.float32)
    ex.mx = "w4a8"
    with torch.no_grad():
        for p in (ex.w1, ex.w2, ex.w3):
            p.copy_(ops.fake_quant_mx_cols(p).float())
    x = rnd(dev, T, d, dtype=torch.float32).requires_grad_(True)
    idx = torch.randint(0, E, (T, k), device=dev)
    w = torch.rand(T, k, device=dev).add_(0.5).requires_grad_(True)
    dy = rnd(dev, T, d, seed=2, dtype=torch.float32)
    y = ex(x, idx, w)
    gw, g3 = torch.autograd.grad(y, (w, ex.w3), dy)
    with torch.no_grad():
        up = ex(x, idx, w + 1.0)
        diff = ((up - y) * dy).sum(1, keepdim=True)
        scale = (y.abs() * dy.abs()).sum(1, keepdim=True) / w
        # the expert rows are rounded to bf16 once, and so is dy in the backward
        assert bool(((diff - gw).abs() <= 3 * HALF_BF16 * scale).all())
        # the sign of one column of each expert's w3 flips: codes and scales stay representable
        col = 5
        old = ex.w3[:, :, col].clone()
        ex.w3[:, :, col] = -old
        diff3 = ((ex(x, idx, w) - y) * dy).sum()
        want = (g3[:, :, col] * (-2 * old)).sum()
        # y's rows are rounded to bf16; w dy, dW3 too
        bound = 6 * HALF_BF16 * float((g3[:, :, col].abs() * 2 * old.abs()).sum() + 2 * (y[:, col].abs() * dy[:, col].abs()).sum())
        assert abs(float(diff3 - want)) <= bound


@pytest.mark.parametrize("mx", ["w4a8", "w4a4"])
@pytest.mark.parametrize("routing", ["token_choice", "expert_choice"])
def test_layer_forward_and_training(dev, mx, routing):
    cfg = config(moe_mx=mx, moe_routing=routing, moe_drop_overflow=routing == "token_choice")
    layer = kmoe.MoELayer(cfg).to(dev).to(BF).train()
    x = rnd(dev, 2, 90, cfg.d_model)
    with torch.no_grad():
        y0 = layer(x)
        aux0 = layer.aux_loss
    xg = x.clone().requires_grad_(True)
    y1 = layer(xg)
    assert torch.equal(y0, y1) and float(aux0) == float(layer.aux_loss.detach())
    (y1.float().square().sum() + layer.aux_loss).backward()
    for n, p in layer.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()) and float(p.grad.abs().sum()) > 0, n
    assert bool(xg.grad.isfinite().all())
    # new weights are packed again
    with torch.no_grad():
        ge = layer.grouped_experts if layer.grouped_experts is not None else layer.grouped_experts_ec
        ge.w3.mul_(2.0)
        err = (layer(x).float() - 2 * y0.float()).norm() / y0.float().norm()
        assert float(err) <= 4 * HALF_BF16


def test_layer_against_oracle(dev):
    cfg = config(E=8, d=256, F=352, moe_mx="w4a8")
    layer = kmoe.MoELayer(cfg).to(dev).to(BF).eval()
    x = rnd(dev, 1, 257, 256)
    with torch.no_grad():
        y = layer(x)[0]
        r = layer.router.route(x[0])
    ge = layer.grouped_experts
    want = M.experts(f64(x[0]), r.idx.cpu(), f64(r.w), f64(ge.w1), f64(ge.w2), f64(ge.w3), "w4a8")
    assert float((f64(y) - want).norm() / want.norm()) <= TOL_Y


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("with_delta", [False, True])
@pytest.mark.parametrize("training", [False, True])
def test_block_runs_norm_routing_and_experts_together(dev, dtype, with_delta, training):
    """Residual add, norm with coded rows, grouped sigmoid routing, 4-bit experts and the
    residual in one block: the same values as the pieces one after the other."""
    cfg = config(E=8, d=256, F=96, moe_mx="w4a8", moe_router_scores="sigmoid", moe_router_groups=4,
                 moe_router_topk_groups=2, moe_router_scale=2.5, moe_balance_bias=True)
    blk = kmoe.MoEFFNBlock(cfg).to(dev).to(dtype).train(training)
    with torch.no_grad():
        blk.ffn.router.balance_bias.copy_(0.05 * torch.randn(8))
        blk.ffn_norm.weight.add_(0.1 * torch.randn_like(blk.ffn_norm.weight))
    x, delta = rnd(dev, 2, 41, 256, dtype=dtype), rnd(dev, 2, 41, 256, seed=5, dtype=dtype)
    with torch.no_grad():
        out = blk(x, delta) if with_delta else blk(x)
        assert blk.last_path == "fused_mx"
        h = x + delta if with_delta else x
        n = ops.rmsnorm(h.reshape(-1, 256), blk.ffn_norm.weight, cfg.norm_eps).n
        r = blk.ffn.router.route(n)
        y, _ = blk.ffn.grouped_experts.run(n, r.idx, r.w, out_dtype=dtype, residual=h.reshape(-1, 256))
    assert torch.equal(out.reshape(-1, 256), y)
    if training:
        hg, dg = x.clone().requires_grad_(True), delta.clone().requires_grad_(True)
        o2 = blk(hg, dg) if with_delta else blk(hg)
        assert blk.last_path == "fused_train" and torch.equal(o2, out)
        (o2.float().square().mean() + blk.aux_loss).backward()
        assert bool(hg.grad.isfinite().all())
        if with_delta:
            assert torch.equal(hg.grad, dg.grad)
        for p in blk.parameters():
            assert p.grad is not None and bool(p.grad.isfinite().all())


def test_mod_composition(dev):
    cfg = config(moe_mx="w4a4", mod_enabled=True)
    mod = kmoe.MoDMoE(cfg).to(dev).to(BF).train()
    x = rnd(dev, 2, 64, cfg.d_model)
    with torch.no_grad():
        y0 = mod(x)
    xg = x.clone().requires_grad_(True)
    y1 = mod(xg)
    assert torch.equal(y0, y1)
    (y1.float().sum() + mod.aux_loss).backward()
    assert bool(xg.grad.isfinite().all())


def test_other_stream_and_graph(dev):
    """A captured layer forward replayed on new inputs, between eager passes, and a call on
    another stream."""
    cfg = config(E=8, d=256, F=352, moe_mx="w4a8", moe_router_scores="sigmoid", moe_router_groups=2)
    layer = kmoe.MoELayer(cfg).to(dev).to(BF).eval()
    xs = [rnd(dev, 1, 50, 256, seed=i) for i in range(4)]
    with torch.no_grad():
        eager = [layer(x) for x in xs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = layer(xs[1])
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(y, eager[1])
        buf = xs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(buf)
        for i in (1, 2, 3, 0):
            buf.copy_(xs[i])
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[i])
            assert torch.equal(layer(xs[(i + 1) % 4]), eager[(i + 1) % 4])


@pytest.mark.parametrize("mx", ["w4a8", "w4a4"])
@pytest.mark.parametrize("T,k,E,cap", [(1, 1, 1, 0), (1, 8, 16, 0), (48, 2, 16, 5), (341, 3, 64, 0), (342, 3, 5, 100), (700, 2, 8, 0), (2048, 2, 16, 200),
                                       (2049, 2, 16, 0), (600, 2, 64, 0)])
def test_one_call_is_the_calls_it_makes(dev, mx, T, k, E, cap):
    """The native pass against its pieces, bit for bit: up to 4096 assignments (fewer over
    many experts) go through the one-workgroup dispatch.  Ids out of range and one expert twice included."""
    d, F = 192, 100
    ex = kmoe.GroupedExperts(E, d, F).to(dev).to(BF)
    ex.mx = mx
    x, res = rnd(dev, T + 9, d), rnd(dev, T, d, seed=8)
    rows = torch.randperm(T + 9, generator=torch.Generator().manual_seed(1))[:T].to(torch.int32).to(dev)
    idx = torch.randint(0, E, (T, k), generator=torch.Generator().manual_seed(2)).to(dev)
    if T > 1:
        idx[1, 0] = -1
        idx[0, :] = E - 1
    for w in (torch.rand(T, k, device=dev), torch.rand(T, k, device=dev).to(BF)):
        for kw in (dict(), dict(row_index=rows), dict(residual=res), dict(out_dtype=torch.float32),
                   dict(coded=ops.quant_rows_mx(x[:T], ex.mx_act))):
            xin = x if "row_index" in kw else x[:T]
            one, d1 = ex.run(xin, idx, w, capacity=cap, **kw)
            ops.set_stage_timing([])
            try:
                many, d2 = ex.run(xin, idx, w, capacity=cap, **kw)
            finally:
                ops.set_stage_timing(None)
            assert torch.equal(one, many) and torch.equal(d1.counts, d2.counts)


def test_empty_calls(dev):
    assert ops.quant_rows_mx(rnd(dev, 0, 64)).q.shape == (0, 128)
    assert ops.dequant_rows_mx(ops.quant_rows_mx(rnd(dev, 0, 64))).shape == (0, 64)
    ex = kmoe.GroupedExperts(2, 64, 64).to(dev).to(BF)
    ex.mx = "w4a8"
    with torch.no_grad():
        y = ex(rnd(dev, 0, 64), torch.zeros(0, 2, dtype=torch.int64, device=dev), torch.zeros(0, 2, device=dev))
    assert y.shape == (0, 64)
    r = rnd(dev, 0, 64)
    layer = kmoe.GroupedExperts(2, 64, 64).to(dev).to(BF)
    layer.mx = "w4a4"
    got, info = layer.run(r, torch.zeros(0, 2, dtype=torch.int64, device=dev), torch.zeros(0, 2, device=dev), residual=r)
    assert got.shape == (0, 64) and not info.counts.any()


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_missing_rows_are_zeros(dev, fmt):
    """row_index -1 in the quantisation and in the one-call pass."""
    x = rnd(dev, 5, 96)
    rows = torch.tensor([3, -1, 0, -1], dtype=torch.int32, device=dev)
    q = ops.quant_rows_mx(x, fmt, row_index=rows)
    want = ops.quant_rows_mx(torch.stack([x[3], torch.zeros_like(x[0]), x[0], torch.zeros_like(x[0])]), fmt)
    assert torch.equal(q.q, want.q) and torch.equal(used(q), used(want))
    pw = ops.pack_weights_mx(*weights(dev, 2, 128, 64))
    x = rnd(dev, 5, 128)
    idx, w = torch.tensor([[0], [1], [1], [0]], device=dev), torch.ones(4, 1, device=dev)
    y = ops.mx_experts(x, idx, w, pw, fmt, row_index=rows)[0]
    assert not y[1].any() and not y[3].any()
    assert torch.equal(y[[0, 2]], ops.mx_experts(x[[3, 0]], idx[[0, 2]], w[[0, 2]], pw, fmt)[0])


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("d,F", [(128, 2816), (2816, 128)])
def test_offsets_past_32_bits(dev, fmt, d, F):
    """The last tokens of a batch whose expert rows (h, or y) hold over 2^31 values: those of
    the same tokens alone."""
    E, k, T = 3, 2, 400_003
    pw = ops.pack_weights_mx(*weights(dev, E, d, F))
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.empty(T, d, device=dev, dtype=BF).normal_(generator=g)
    idx = torch.randint(0, E, (T, k), device=dev, generator=g)
    w = torch.ones(T, k, device=dev)
    y = ops.mx_experts(x, idx, w, pw, fmt)[0]
    few = [0, 1, T // 2, T - 3, T - 2, T - 1]
    assert torch.equal(y[few], ops.mx_experts(x[few], idx[few], w[few], pw, fmt)[0])


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_tile_sizes_agree(dev, fmt):
    """The first tokens of batches that take the different tile sizes of both products (64 x 128,
    64 x 256, 128 x 256 on 256 CUs), with and without the kept gate / up values: each K sum has one
    order in all of them, so the same bits."""
    E, d, F, k = 4, 1024, 2048, 2
    pw = ops.pack_weights_mx(*weights(dev, E, d, F))
    T = 8001
    x = rnd(dev, T, d)
    idx = torch.rand(T, E, generator=torch.Generator().manual_seed(4)).topk(k, 1).indices.to(dev)
    w = torch.ones(T, k, device=dev)
    want = None
    for t in (100, 1203, T):
        y = ops.mx_experts(x[:t], idx[:t], w[:t], pw, fmt)[0]
        disp = ops.dispatch(x[:t], idx[:t], w[:t], E, materialize=False)
        h, gu = ops.gemm_gate_up_mx(ops.quant_rows_mx(x[:t], fmt), disp.row_token, disp.offsets, pw, t * k, save_gu=True)
        rows = disp.slot_row.view(t, k)[:100].long().flatten()
        got = (y[:100], ops.gemm_down_mx(h, disp.offsets, pw, t * k)[rows], h.q[rows], used(h)[rows], gu[rows])
        want = got if want is None else want
        assert all(torch.equal(u, v) for u, v in zip(got, want))


def test_weights_past_32_bits(dev):
    """Experts whose weights and packed codes hold over 2^31 values and bytes: the last ones
    alone give the same values, packs and products."""
    E, d, F = 64, 4096, 9216
    w = [torch.empty(*s, device=dev, dtype=BF) for s in ((E, d, F), (E, d, F), (E, F, d))]
    for i, v in enumerate(w):
        v.zero_()
        v[-1].normal_(std=0.02, generator=torch.Generator(device=dev).manual_seed(i))
    last = [v[-1:].contiguous() for v in w]
    assert torch.equal(ops.fake_quant_mx_cols(w[0])[-1:], ops.fake_quant_mx_cols(last[0]))
    pw, p1 = ops.pack_weights_mx(*w), ops.pack_weights_mx(*last)
    for u, v in zip(pw[:4], p1[:4]):
        assert torch.equal(u[-v.numel():], v)
    x, one = rnd(dev, 40, d), torch.ones(40, 1, device=dev)
    idx = torch.full((40, 1), E - 1, device=dev)
    for fmt in ("e4m3", "e2m1"):
        assert torch.equal(ops.mx_experts(x, idx, one, pw, fmt)[0], ops.mx_experts(x, 0 * idx, one, p1, fmt)[0])


@pytest.mark.parametrize("mx", ["w4a8", "w4a4"])
def test_capacity_in_training(dev, mx):
    """Dropped assignments: the training forward gives the inference one's values, a token whose
    every assignment was dropped gets no output, and no gradient through the experts."""
    cfg = config(E=4, d=128, F=96, moe_mx=mx, moe_drop_overflow=True, moe_capacity_factor=0.25)
    layer = kmoe.MoELayer(cfg).to(dev).to(BF).train()
    x = rnd(dev, 1, 300, 128)
    with torch.no_grad():
        want = layer(x)
    xg = x.clone().requires_grad_(True)
    y = layer(xg)
    assert torch.equal(y, want)
    empty = ~want[0].any(1)
    assert bool(empty.any()) and not bool(empty.all())
    ex = layer.grouped_experts
    dw = torch.autograd.grad(y, [ex.w1, ex.w2, ex.w3], rnd(dev, 1, 300, 128, seed=1), retain_graph=False)
    assert all(bool(g.isfinite().all()) and bool(g.any()) for g in dw)
    y2 = layer(xg)
    dy = rnd(dev, 1, 300, 128, seed=1)
    dy[0, empty] = 100.0  # (what a token without output gets does not reach the experts)
    assert all(torch.equal(u, v) for u, v in zip(torch.autograd.grad(y2, [ex.w1, ex.w2, ex.w3], dy), dw))


def test_two_streams_at_once(dev):
    """Two passes of one layer on two streams at once, several times: each its own result."""
    layer = kmoe.MoELayer(config(E=8, d=256, F=352, moe_mx="w4a4")).to(dev).to(BF).eval()
    xs = [rnd(dev, 1, T, 256, seed=T) for T in (33, 700)]
    with torch.no_grad():
        want = [layer(x) for x in xs]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(8):
            for s, x in zip(streams, xs):
                with torch.cuda.stream(s):
                    got.append(layer(x))
        torch.cuda.synchronize()
        for i, y in enumerate(got):
            assert torch.equal(y, want[i % 2])


def test_training_step_in_a_graph(dev):
    """Forward and gradients of norm, routing and experts captured together and replayed on new
    inputs, eager passes of other leaves in between."""
    d, E, k, T = 128, 8, 2, 40
    ex = kmoe.GroupedExperts(E, d, 96).to(dev).to(BF)
    ex.mx = "w4a8"
    wr = rnd(dev, E, d, std=0.1, dtype=torch.float32)
    dy, dh = rnd(dev, T, d, seed=5), rnd(dev, T, d, seed=6)

    def step(x, delta, gain):
        leaves = [v.detach().requires_grad_(True) for v in (x, delta, gain)]
        params = list(ex.parameters())
        h, n = kmoe.add_rms_norm(*leaves)
        w, idx = kmoe.route_topk(torch.nn.functional.linear(n.float(), wr), k, scores="sigmoid", groups=2)
        y = ex(n, idx, w)
        return [y.detach(), h.detach()] + list(torch.autograd.grad([y, h], leaves + params, [dy, dh]))

    sets = [(rnd(dev, T, d, seed=i), rnd(dev, T, d, seed=10 + i), 1 + rnd(dev, d, seed=20 + i, std=0.1)) for i in range(4)]
    buf = [v.clone() for v in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*buf)
    torch.cuda.current_stream().wait_stream(side)
    eager = [step(*s) for s in sets]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*buf)
    for i in (1, 2, 3, 0):
        for b, v in zip(buf, sets[i]):
            b.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        for u, v in zip(out, eager[i]):
            assert torch.equal(u, v)
        assert all(torch.equal(u, v) for u, v in zip(step(*sets[(i + 1) % 4]), eager[(i + 1) % 4]))


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_beside_an_eager_graph(dev):
    """Refused before anything is recorded, for each operator; captured once that graph is gone."""
    ex = kmoe.GroupedExperts(4, 64, 64).to(dev).to(BF)
    ex.mx = "w4a4"
    x, gain = rnd(dev, 8, 64), torch.ones(64, device=dev, dtype=BF).requires_grad_(True)
    logits = rnd(dev, 8, 4, dtype=torch.float32).requires_grad_(True)
    idx, w = torch.zeros(8, 1, dtype=torch.int64, device=dev), torch.ones(8, 1, device=dev)
    dy = rnd(dev, 8, 64, seed=1)
    calls = [(lambda: kmoe.route_topk(logits, 2)[0], logits, torch.ones(8, 2, device=dev)),
             (lambda: kmoe.add_rms_norm(x, x, gain)[1], gain, dy), (lambda: ex(x, idx, w), ex.w1, dy)]
    for call, leaf, dout in calls:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(call(), leaf, dout)
        torch.cuda.current_stream().wait_stream(side)
        alive = call()
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        want = torch.autograd.grad(alive, leaf, dout)[0]
        del alive
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = torch.autograd.grad(call(), leaf, dout)[0]
        for _ in range(3):
            got.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@pytest.mark.parametrize("training", [False, True])
@pytest.mark.parametrize("dtype", [BF, torch.float32, torch.float16])
def test_block_edge_calls(dev, training, dtype):
    """One token, and streams and deltas of other types than the weights'; an empty batch is
    refused by the router, as in the bf16 block."""
    cfg = config(E=4, d=128, F=96, moe_mx="w4a8")
    blk = kmoe.MoEFFNBlock(cfg).to(dev).to(BF).train(training)
    with torch.no_grad():
        h = rnd(dev, 1, 1, 128, dtype=dtype)
        for empty in ((h[:, :0],), (h[:, :0], h[:, :0])):
            with pytest.raises(kmoe.KmoeError, match="kmoe_router"):
                blk(*empty)
        for dd in (BF, torch.float32, torch.float16, torch.float64):
            delta = rnd(dev, 1, 1, 128, seed=1, dtype=dd)
            y = blk(h, delta)
            want = blk(h + delta)
            assert y.dtype == want.dtype and torch.equal(y, want)


def test_refusals(dev):
    with pytest.raises(ValueError, match="element type"):
        ops.quant_rows_mx(rnd(dev, 2, 64), "e5m2")
    with pytest.raises(kmoe.KmoeError, match="multiple of 32"):
        ops.quant_rows_mx(rnd(dev, 2, 40))
    with pytest.raises(ValueError):
        ops.fake_quant_mx_cols(rnd(dev, 2, 40))
    with pytest.raises(ValueError):
        ops.fake_quant_mx_cols(rnd(dev, 1, 2, 40, dtype=torch.float16))
    w = weights(dev, 2, 64, 64)
    with pytest.raises(ValueError, match="w1/w2"):
        ops.pack_weights_mx(w[0], w[1][:, :, :32], w[2])
    pw = ops.pack_weights_mx(*w)
    off = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="d=64"):
        ops.gemm_gate_up_mx(ops.quant_rows_mx(rnd(dev, 2, 128)), None, off, pw, 2)
    with pytest.raises(ValueError, match="permuted rows"):
        ops.gemm_gate_up_mx(ops.quant_rows_mx(rnd(dev, 2, 64)), None, off, pw, 3)
    with pytest.raises(ValueError):
        ops.gemm_down_mx(ops.quant_rows_mx(rnd(dev, 2, 128)), off, pw, 2)
    ex = kmoe.GroupedExperts(2, 64, 64).to(dev).to(BF)
    ex.mx = "w4a16"
    with pytest.raises(ValueError, match="w4a16"):
        ex(rnd(dev, 2, 64), torch.zeros(2, 1, dtype=torch.int64, device=dev), torch.ones(2, 1, device=dev))
    ex.mx, ex.use_fp8 = "w4a8", True
    with pytest.raises(ValueError, match="not both"):
        ex(rnd(dev, 2, 64), torch.zeros(2, 1, dtype=torch.int64, device=dev), torch.ones(2, 1, device=dev))
    i1, w1 = torch.zeros(2, 1, dtype=torch.int64, device=dev), torch.ones(2, 1, device=dev)
    x64 = rnd(dev, 2, 64)
    for bad in (dict(coded=ops.quant_rows_mx(x64, "e2m1")), dict(coded=ops.quant_rows_mx(rnd(dev, 3, 64))),
                dict(residual=x64[:1]), dict(row_index=torch.zeros(3, dtype=torch.int32, device=dev)),
                dict(block_counts=torch.zeros(3, dtype=torch.int32, device=dev))):
        with pytest.raises(ValueError):
            ops.mx_experts(x64, i1, w1, pw, "e4m3", **bad)
    with pytest.raises(ValueError):
        ops.mx_experts(rnd(dev, 3, 64), i1, w1, pw, "e4m3")
    with pytest.raises(ValueError, match="packed-weight files"):
        ex.use_fp8 = False
        kmoe.checkpoint.save_packed(ex, "unused.safetensors")


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
@pytest.mark.parametrize("A", [5, 200])
def test_rows_far_past_the_last_are_zeros(dev, fmt, A):
    """row_token entries whose byte offset is a multiple of 2^32 (of the codes: 2^25 and 2^26 rows of
    128 and 64 bytes; of the scales: 2^28 of 16), and the largest entry, in the small-row kernel and a
    tile."""
    pw = ops.pack_weights_mx(*weights(dev, 1, 128, 64))
    x = ops.quant_rows_mx(rnd(dev, 5, 128), fmt)
    far = [1 << 25, (1 << 26) + 1, 1 << 28, 2**31 - 1]
    token = torch.arange(A, dtype=torch.int32) % 5
    bad = [1, 2, 3, 4] if A == 5 else [1, 64, 130, 199]
    token[bad] = torch.tensor(far, dtype=torch.int32)
    off = torch.tensor([0, A], dtype=torch.int32, device=dev)
    h = ops.gemm_gate_up_mx(x, token.to(dev), off, pw, A)
    good = [i for i in range(A) if i not in bad]
    assert not h.q[bad].any() and bool(h.q[good].any(1).all())


@pytest.mark.parametrize("mx", ["w4a8", "w4a4"])
def test_more_rows_than_a_grid_of_small_slots(dev, mx):
    """400000 tokens of top-8 at F 2816: 3.2 M routed rows, of which 32-row slots of 32 columns would be more
    workgroups than a launch takes; the kernel that runs needs a sixteenth of them.  Tokens among
    them are those of a call of their own."""
    T, k, E, d, F = 400_000, 8, 8, 64, 2816
    pw = ops.pack_weights_mx(*weights(dev, E, d, F))
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.empty(T, d, device=dev, dtype=BF).normal_(generator=g)
    idx = torch.argsort(torch.rand(T, E, device=dev, generator=g), 1)
    w = torch.rand(T, k, device=dev, generator=g)
    y, counts, _ = ops.mx_experts(x, idx, w, pw, ops.MX_EXPERTS[mx])
    assert int(counts.sum()) == T * k
    few = torch.tensor(list(range(0, T, T // 300)) + [T - 1], device=dev)
    want, _, _ = ops.mx_experts(x[few], idx[few], w[few], pw, ops.MX_EXPERTS[mx])
    assert torch.equal(y[few], want)


@pytest.mark.parametrize("mx", [None, "w4a8"])
@pytest.mark.parametrize("how", ["parameter", "data", "written"])
def test_outputs_follow_the_weights(dev, mx, how):
    """Weights that are replaced (the new ones in the freed ones' memory), assigned through .data, or written
    there and told of: the layer's output, and its gradients, are those of a layer that never had others."""
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=4, moe_top_k=2, d_ff_expert=64, moe_mx=mx)
    torch.manual_seed(1)
    layer, other = kmoe.MoELayer(cfg).to(dev), kmoe.MoELayer(cfg).to(dev)
    x, dy = rnd(dev, 1, 30, 128, dtype=torch.float32), rnd(dev, 1, 30, 128, seed=1, dtype=torch.float32)

    def run(m):
        xg = x.clone().requires_grad_(True)
        y = m(xg)
        with torch.no_grad():
            return [m(x), y.detach()] + list(torch.autograd.grad(y, [xg] + list(m.parameters()), dy))
    run(layer)
    for (name, p), q in zip(layer.named_parameters(), other.parameters()):
        if how == "written":
            p.data.copy_(q)
            continue
        shape = p.shape
        p.data = torch.empty(0, device=dev)  # its memory is the next one's
        new = torch.empty(shape, device=dev)
        new.data.copy_(q)
        if how == "data":
            p.data = new
        else:
            owner, _, leaf = name.rpartition(".")
            setattr(layer.get_submodule(owner), leaf, torch.nn.Parameter(new))
    if how == "written":
        kmoe.weights_changed(layer)
    for u, v in zip(run(layer), run(other)):
        assert torch.equal(u, v)


@pytest.mark.parametrize("mx", [None, "w4a8"])
def test_a_captured_forward_packs_nothing_for_others(dev, mx):
    """The first call of a layer is captured: an eager call before any replay does not take the packed weights
    that the capture recorded and nothing has written yet.  Replays follow."""
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=4, moe_top_k=2, d_ff_expert=64, moe_mx=mx)
    layer, x = kmoe.MoELayer(cfg).to(dev), rnd(dev, 1, 30, 128, dtype=torch.float32)
    want = None
    with torch.no_grad():
        other = kmoe.MoELayer(cfg).to(dev)
        other.load_state_dict(layer.state_dict())
        want = other(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(x)
        assert torch.equal(layer(x), want)
        for _ in range(3):
            y.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(layer(x), want)


@pytest.mark.parametrize("mx", [None, "w4a8"])
def test_a_captured_forward_keeps_its_weights(dev, mx):
    """Weights packed before the capture, then moved: the replays give what the weights at the capture
    gave, whatever the memory of packed weights that nobody else needs is used for."""
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=4, moe_top_k=2, d_ff_expert=64, moe_mx=mx)
    layer, x = kmoe.MoELayer(cfg).to(dev), rnd(dev, 1, 30, 128, dtype=torch.float32)
    with torch.no_grad():
        want = layer(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer(x)
        for i in range(3):
            for p in layer.parameters():
                p.mul_(1.5)
            now = layer(x)
            junk = [torch.full((n << 8,), 0x7f, dtype=torch.uint8, device=dev) for n in range(1, 600)]
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(layer(x), now) and not torch.equal(now, want)
            del junk


@pytest.mark.parametrize("mx", [None, "w4a8"])
def test_a_captured_training_step_follows_its_weights(dev, mx):
    """Forward and gradients captured after an eager pass has packed the weights, which then move between the
    replays: each replay is the eager pass at the weights of its time."""
    cfg = kmoe.AdvancedMoEConfig(d_model=128, n_experts=4, moe_top_k=2, d_ff_expert=64, moe_mx=mx)
    layer, other = kmoe.MoELayer(cfg).to(dev), kmoe.MoELayer(cfg).to(dev)
    x, dy = rnd(dev, 1, 30, 128, dtype=torch.float32), rnd(dev, 1, 30, 128, seed=1, dtype=torch.float32)

    def step(m):
        xg = x.detach().requires_grad_(True)
        y = m(xg)
        return [y.detach()] + list(torch.autograd.grad(y, [xg] + list(m.parameters()), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(layer)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(layer)
    for i in range(4):
        if i:
            with torch.no_grad():
                for p in layer.parameters():
                    p.add_(rnd(dev, *p.shape, seed=i, std=0.02, dtype=p.dtype))
        g.replay()
        torch.cuda.synchronize()
        other.load_state_dict(layer.state_dict())
        for u, v in zip(out, step(other)):
            assert torch.equal(u, v)


def test_misplaced_arguments_are_refused(dev):
    """Tables and outputs in host memory, histograms of another type: refused before a launch."""
    E, d, F, T, k = 4, 64, 64, 3000, 2
    pw = ops.pack_weights_mx(*weights(dev, E, d, F))
    x, w = rnd(dev, T, d), torch.ones(T, k, device=dev)
    lg = rnd(dev, T, E, dtype=torch.float32)
    r = ops.route_topk(lg, k, hist=True)
    ops.mx_experts(x, r.idx, w, pw, "e4m3", block_counts=r.block_counts)
    bad = [dict(block_counts=r.block_counts.long()), dict(block_counts=r.block_counts.float()),
           dict(block_counts=r.block_counts.cpu()), dict(block_counts=r.block_counts.t()),
           dict(out_map=torch.arange(T, dtype=torch.int32), T_out=T), dict(scale=torch.ones(T)), dict(residual=x.cpu())]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.mx_experts(x, r.idx, w, pw, "e4m3", **kw)
    cpu = pw._replace(w13=pw.w13.cpu(), w3=pw.w3.cpu())
    off = torch.zeros(E + 1, device=dev, dtype=torch.int32)
    rows = ops.quant_rows_mx(x)
    for call in (lambda: ops.mx_experts(x, r.idx, w, cpu, "e4m3"), lambda: ops.gemm_gate_up_mx(rows, None, off, cpu, T),
                 lambda: ops.gemm_down_mx(rows, off, cpu, T),
                 lambda: ops.route_topk_bwd(lg, r.idx, w, dlogits=torch.zeros(T, E))):
        with pytest.raises(ValueError, match="one GPU"):
            call()


def test_captured_forward_beside_an_eager_graph(dev):
    """Without gradients a capture takes the same leaves while an eager graph of them lives, and that
    graph's backward is as it was."""
    x = rnd(dev, 8, 64)
    gain = torch.ones(64, device=dev, dtype=BF).requires_grad_(True)
    logits = rnd(dev, 8, 4, dtype=torch.float32).requires_grad_(True)
    for call, leaf in ((lambda: kmoe.add_rms_norm(x, x, gain), gain), (lambda: kmoe.route_topk(logits, 2), logits)):
        alive, again = call(), call()
        i = 0 if alive[0].requires_grad and alive[0].dtype == torch.float32 else 1
        g = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(g):
            out = call()
        assert not any(o.requires_grad for o in out)
        for _ in range(3):
            for o in out:
                o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(u, v) for u, v in zip(out, alive))
        a, b = (torch.autograd.grad(v[i].float().square().sum(), leaf)[0] for v in (alive, again))
        assert torch.equal(a, b) and bool(a.any())
