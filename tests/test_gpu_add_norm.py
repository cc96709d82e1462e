"""Residual add with RMSNorm and coded rows (ops.add_rmsnorm, kmoe.add_rms_norm)."""
import pytest
import torch

import kmoe
from kmoe import ops
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5


def rnd(dev, *shape, seed=0, std=1.0, dtype=BF):
    g = torch.Generator().manual_seed(seed)
    return (std * torch.randn(*shape, generator=g)).to(dtype).to(dev)


@pytest.mark.parametrize("quant", [None, "e4m3", "e2m1"])
@pytest.mark.parametrize("xd,dd,wd", [(BF, BF, BF), (F32, BF, F32), (BF, F32, BF), (F32, F32, BF)])
@pytest.mark.parametrize("T,d", [(1, 32), (5, 64), (3, 96), (70, 2048), (9, 4160), (2, 8192)])
def test_forward(dev, quant, xd, dd, wd, T, d):
    x, delta = rnd(dev, T, d, seed=1, std=2.0, dtype=xd), rnd(dev, T, d, seed=2, dtype=dd)
    w = (1 + 0.1 * rnd(dev, d, seed=3, dtype=F32)).to(wd)
    r = ops.add_rmsnorm(x, delta, w, EPS, quant=quant)
    stream = F32 if F32 in (xd, dd) else BF
    h = (x.float() + delta.float()).to(stream)
    assert r.h.dtype == stream and torch.equal(r.h, h)
    # the framework's own norm of the sum, bit for bit
    base = ops.rmsnorm(h, w, EPS)
    assert torch.equal(r.n, base.n) and torch.equal(r.rrms, base.rrms)
    _, n64 = M.add_norm(h.double(), None, w.double(), EPS)
    # f32 sum of d squares and one rounding to bf16
    tol = torch.finfo(BF).eps / 2 * (1 + 1e-3) + (d + 8) * 2.0 ** -24
    assert bool(((r.n.double() - n64).abs() <= tol * n64.abs()).all())
    if quant:
        want = ops.quant_rows_mx(base.n, quant)
        n = (d + 127) // 128 * 4  # scale bytes behind are not written
        assert torch.equal(r.q, want.q) and torch.equal(r.scale[:, :n], want.scale[:, :n])
    else:
        assert r.q is None and r.scale is None


def test_without_delta_zero_rows_and_bad_values(dev):
    x = rnd(dev, 6, 128)
    x[1] = 0.0
    x[2, 3] = float("nan")
    x[3, 100] = float("inf")
    w = torch.ones(128, device=dev)
    r = ops.add_rmsnorm(x, None, w, EPS, quant="e4m3")
    assert r.h.data_ptr() == x.data_ptr()
    assert not r.n[1].any() and not r.q[1].any()
    assert bool(r.n[2].isnan().all()) and bool((r.scale[2, :4] == 255).all())
    good = [0, 1, 4, 5]
    clean = ops.add_rmsnorm(x[good], None, w, EPS, quant="e4m3")
    assert torch.equal(r.q[good], clean.q) and torch.equal(r.n[good], clean.n)
    e = ops.add_rmsnorm(x[:0], x[:0], w, EPS, quant="e4m3")
    assert e.h.shape == (0, 128) and e.q.shape == (0, 128)


@pytest.mark.parametrize("xd,dd", [(BF, BF), (F32, BF), (F32, F32)])
@pytest.mark.parametrize("T,d", [(1, 64), (37, 256), (1000, 2048)])
def test_backward(dev, xd, dd, T, d):
    x, delta = rnd(dev, T, d, seed=1, dtype=xd).requires_grad_(True), rnd(dev, T, d, seed=2, dtype=dd).requires_grad_(True)
    w = (1 + 0.1 * rnd(dev, d, seed=3, dtype=F32)).requires_grad_(True)
    h, n = kmoe.add_rms_norm(x, delta, w, EPS)
    dh, dn = rnd(dev, T, d, seed=4, dtype=h.dtype), rnd(dev, T, d, seed=5)
    dx, dd_, dg = torch.autograd.grad((h, n), (x, delta, w), (dh, dn))
    h64, w64 = h.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    _, n64 = M.add_norm(h64, None, w64, EPS)
    gh, gw = torch.autograd.grad(n64, (h64, w64), dn.double())
    gh = gh + dh.double()
    for got, dt in ((dx, xd), (dd_, dd)):
        # the f32 sums over d, and a rounding to the stream's and to the input's type
        tol = (torch.finfo(h.dtype).eps / 2 + torch.finfo(dt).eps / 2) + 2.0 ** -20
        assert got.dtype == dt and float((got.double() - gh).norm() / gh.norm()) <= tol
    assert float((dg.double() - gw).norm() / gw.norm()) <= 2.0 ** -18


def test_backward_of_one_output(dev):
    """Only n, or only h, goes on: the other's gradient is nothing."""
    x, delta = rnd(dev, 30, 128, dtype=F32).requires_grad_(True), rnd(dev, 30, 128, seed=1).requires_grad_(True)
    w = torch.ones(128, device=dev).requires_grad_(True)
    dn, dh = rnd(dev, 30, 128, seed=2), rnd(dev, 30, 128, seed=3, dtype=F32)
    h, n = kmoe.add_rms_norm(x, delta, w, EPS)
    a = torch.autograd.grad(n, (x, delta, w), dn, retain_graph=True)
    b = torch.autograd.grad((h, n), (x, delta, w), (torch.zeros_like(h), dn), retain_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    c = torch.autograd.grad(h, (x, delta), dh, retain_graph=True)
    assert torch.equal(c[0], dh) and torch.equal(c[1], dh.to(BF))
    with pytest.raises(RuntimeError):  # no second derivative
        (g,) = torch.autograd.grad(n.float().square().sum(), x, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("xd,dd", [(BF, BF), (F32, F32), (F32, BF), (BF, F32)])
@pytest.mark.parametrize("both", [False, True])
def test_gradients_are_not_shared(dev, xd, dd, both):
    """x and delta leaves of one sum: writing to one's gradient leaves the other's as it was; one
    tensor as both gets twice the gradient."""
    x, delta = (rnd(dev, 3, 64, seed=i, dtype=t).requires_grad_(True) for i, t in enumerate((xd, dd)))
    w = torch.ones(64, device=dev)
    h, n = kmoe.add_rms_norm(x, delta, w, EPS)
    torch.autograd.backward([n, h] if both else [h], [torch.ones_like(t) for t in ([n, h] if both else [h])])
    want = delta.grad.clone()
    x.grad.mul_(2.0)
    assert torch.equal(delta.grad, want)
    y = rnd(dev, 3, 64, dtype=xd).requires_grad_(True)
    z = y.detach().clone().requires_grad_(True)
    u = y.detach().clone().requires_grad_(True)
    for a, b in ((y, y), (z, u)):
        h, n = kmoe.add_rms_norm(a, b, w, EPS)
        torch.autograd.backward([n, h], [torch.ones_like(n), torch.ones_like(h)])
    assert torch.equal(y.grad, z.grad + u.grad)


def test_backward_against_differences(dev):
    T, d, h = 3, 64, 2.0 ** -6
    x, delta = rnd(dev, T, d, dtype=F32).requires_grad_(True), rnd(dev, T, d, seed=1, dtype=F32)
    w = rnd(dev, d, seed=2, dtype=F32).abs().add_(0.5)
    hh, n = kmoe.add_rms_norm(x, delta, w, EPS)
    dh, dn = rnd(dev, T, d, seed=3, dtype=F32), rnd(dev, T, d, seed=4)
    (dx,) = torch.autograd.grad((hh, n), x, (dh, dn))

    def f(v):
        s, m = M.add_norm(v, delta.double(), w.double(), EPS)
        return (s * dh.double()).sum() + (m * dn.double()).sum()
    v = x.detach().double()
    for t in range(T):
        for c in range(0, d, 7):
            e = torch.zeros_like(v)
            e[t, c] = h
            num = float(f(v + e) - f(v - e)) / (2 * h)
            # h^2 / 6 of the third derivative, which r^3 sum|g dn| bounds a few times over
            r3 = float(v[t].square().mean() ** -1.5)
            bound = h * h / 6 * 16 * max(r3, 1.0) * float((w.double() * dn[t].double().abs()).sum()) / d ** 0.5
            assert abs(num - float(dx[t, c])) <= bound + 1e-4


def test_offsets_past_32_bits(dev):
    """The last rows of 2^31 values, forward and backward: those of the same rows alone."""
    T, d = 525_003, 4096
    g = torch.Generator(device=dev).manual_seed(1)
    x, delta, dn = (torch.empty(T, d, device=dev, dtype=BF).normal_(generator=g) for _ in range(3))
    w = 1 + rnd(dev, d, std=0.1)
    few = [0, T // 2, T - 2, T - 1]
    r, f = ops.add_rmsnorm(x, delta, w, EPS, quant="e4m3"), ops.add_rmsnorm(x[few], delta[few], w, EPS, quant="e4m3")
    assert all(torch.equal(u[few], v) for u, v in zip(r, f))
    dx = ops.add_rmsnorm_bwd(dn, r.h, w, r.rrms, dh=delta)[0]
    assert torch.equal(dx[few], ops.add_rmsnorm_bwd(dn[few], f.h, w, f.rrms, dh=delta[few])[0])


def test_views_streams_and_graph(dev):
    x, delta = rnd(dev, 40, 512), rnd(dev, 40, 512, seed=1)
    w = torch.ones(256, device=dev, dtype=BF)
    a = ops.add_rmsnorm(x[:, 128:384], delta[:, :256], w, EPS, quant="e4m3")
    b = ops.add_rmsnorm(x[:, 128:384].contiguous(), delta[:, :256].contiguous(), w, EPS, quant="e4m3")
    def same(a, b):
        return all(torch.equal(u, v) for u, v in zip((*a[:4], a.scale[:, :8]), (*b[:4], b.scale[:, :8])))
    assert same(a, b)
    bx, bd = x[:, :256].contiguous(), delta[:, :256].contiguous()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = ops.add_rmsnorm(bx, bd, w, EPS, quant="e4m3")
    for seed in (5, 6, 7):
        nx = rnd(dev, 40, 256, seed=seed)
        want = ops.add_rmsnorm(nx, bd, w, EPS, quant="e4m3")
        bx.copy_(nx)
        g.replay()
        torch.cuda.synchronize()
        assert same(r, want)


def test_refusals(dev):
    x, w = rnd(dev, 2, 64), torch.ones(64, device=dev)
    with pytest.raises(ValueError):
        ops.add_rmsnorm(x, x[:, :32], w, EPS)
    with pytest.raises(ValueError):
        ops.add_rmsnorm(x, x, w[:32], EPS)
    with pytest.raises(ValueError, match="element type"):
        ops.add_rmsnorm(x, x, w, EPS, quant="int8")
    with pytest.raises(ValueError):
        kmoe.add_rms_norm(x, x[:1], w, EPS)
    r = ops.add_rmsnorm(x, x, w, EPS)
    with pytest.raises(ValueError):
        ops.add_rmsnorm_bwd(x[:1], r.h, w, r.rrms)
    y = rnd(dev, 2, 40)
    with pytest.raises(kmoe.KmoeError, match="multiple of 32"):
        ops.add_rmsnorm(y, y, torch.ones(40, device=dev), EPS, quant="e4m3")
    with pytest.raises(kmoe.KmoeError):
        ops.add_rmsnorm(y, y, torch.ones(40, device=dev), -1.0)


@pytest.mark.parametrize("xd,dd", [(BF, BF), (F32, BF), (F32, F32), (BF, F32)])
@pytest.mark.parametrize("T,d", [(3, 2112), (300, 4160), (33, 6144), (301, 8192)])
def test_backward_of_wide_rows(dev, xd, dd, T, d):
    """Rows of more than 2048 values, in each pair of types, with a bf16 gradient next to an f32
    one: against the formula in 64 bits."""
    x, delta = rnd(dev, T, d, seed=1, dtype=xd).requires_grad_(True), rnd(dev, T, d, seed=2, dtype=dd).requires_grad_(True)
    w = (1 + 0.1 * rnd(dev, d, seed=3, dtype=F32)).requires_grad_(True)
    h, n = kmoe.add_rms_norm(x, delta, w, EPS)
    dh, dn = rnd(dev, T, d, seed=4, dtype=h.dtype), rnd(dev, T, d, seed=5)
    dx, dd_, dg = torch.autograd.grad((h, n), (x, delta, w), (dh, dn))
    h64, w64, dn64 = h.detach().double(), w.detach().double(), dn.double()
    r = (h64.square().mean(1, keepdim=True) + EPS).rsqrt()
    dot = w64 * dn64 * h64
    want = dh.double() + r * w64 * dn64 - r ** 3 * h64 * dot.mean(1, keepdim=True)
    terms = dh.double().abs() + r * (w64 * dn64).abs() + r ** 3 * h64.abs() * dot.abs().mean(1, keepdim=True)
    # f32: a lane's sum of d / 64 terms and six additions over the wave, in r and in the dot product; a
    # dozen operations; the stream's and the input's rounding
    steps = (2 * (d // 64 + 6) + 12) * 2.0 ** -24
    for got, dt in ((dx, xd), (dd_, dd)):
        rounding = (torch.finfo(h.dtype).eps / 2 + torch.finfo(dt).eps / 2) * (1 + steps)
        assert got.dtype == dt
        assert bool(((got.double() - want).abs() <= rounding * want.abs() + (1 + rounding) * steps * terms).all())
    gt = dn64 * h64 * r
    assert bool(((dg.double() - gt.sum(0)).abs() <= (T + d // 64 + 16) * 2.0 ** -24 * gt.abs().sum(0)).all())
