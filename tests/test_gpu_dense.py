"""The gated block and adapted projections on the GPU against their formulas in 64 bits, within
bounds that carry every rounding (dense_bounds.py)."""
import ctypes
import os
import sys

import pytest
import torch

import kmoe
from kmoe import _lib

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import dense_bounds as B  # noqa: E402

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
ACTS = ("silu", "gelu", "gelu_tanh", "relu")


def rnd(dev, *shape, std=1.0, dtype=BF, seed=[0]):
    seed[0] += 1
    g = torch.Generator().manual_seed(seed[0])
    return torch.randn(*shape, generator=g).mul(std).to(dtype).to(dev)


def make_ffn(dev, T, d, F):
    return rnd(dev, T, d), rnd(dev, F, d, std=d ** -0.5), rnd(dev, F, d, std=d ** -0.5), rnd(dev, d, F, std=F ** -0.5)


def make_ad(dev, n, r, K, N, scale=True):
    return kmoe.Adapters(rnd(dev, n, r, K, std=K ** -0.5), rnd(dev, n, N, r, std=0.3),
                         torch.linspace(0.5, 2.0, n).to(dev) if scale else None)


# rows from one to many (the kernel of few rows up to 16, runs of K, the tiles), widths of odd eighths
SIZES = [(1, 64, 72), (2, 8, 8), (5, 136, 128), (16, 200, 24), (17, 72, 264), (33, 256, 136), (64, 520, 200), (65, 64, 72),
         (127, 200, 136), (130, 136, 392), (300, 520, 264), (777, 64, 1032), (2042, 72, 1544), (16379, 136, 1096)]
# sizes that take each of the large tiles in each kind of product
LARGE = [(10001, 1032, 2056), (8195, 1032, 1096), (1030, 2056, 5640)]


@pytest.mark.parametrize("T,d,F", SIZES)
def test_ffn(dev, T, d, F):
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    for act in ACTS if T in (5, 130) else ("silu",):
        with torch.no_grad():
            y = kmoe.gated_ffn(x, wg, wu, wd, act)
        B.check(act, y, B.ffn(x, wg, wu, wd, act)[0])


@pytest.mark.parametrize("T,d,F", SIZES + LARGE)
def test_ffn_backward(dev, T, d, F):
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    dy = rnd(dev, T, d)
    for act in ACTS if T in (5, 130) else ("silu",):
        leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = kmoe.gated_ffn(*leaves, act)
        grads = torch.autograd.grad(y, leaves, dy)
        want, h, p, q = B.ffn(x, wg, wu, wd, act)
        B.check(act, y.detach(), want)
        for name, g, w in zip(("dx", "dwg", "dwu", "dwd"), grads, B.ffn_grads(x, wg, wu, wd, dy, h, p, q)):
            B.check((act, name), g, w)


@pytest.mark.parametrize("T,d,F", [(1, 64, 72), (8, 136, 200), (9, 200, 136), (17, 72, 1096), (32, 1032, 264)])
def test_few_rows_are_rounded_once(dev, T, d, F):
    """Of up to 32 rows h, dgate, dup and the adapters' inner products are two bf16 each."""
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    dy, ids = rnd(dev, T, d), make_ids(dev, T, 3, "mixed")
    ads = [make_ad(dev, 3, r, *kn) for kn, r in (((d, F), 16), ((d, F), 16), ((F, d), 8))]
    with torch.no_grad():
        B.check("y", kmoe.gated_ffn(x, wg, wu, wd), B.ffn(x, wg, wu, wd, "silu", to=B.V.twice)[0])
        B.check("adapters", kmoe.gated_ffn(x, wg, wu, wd, "silu", kmoe.FFNAdapters(*ads), ids),
                B.ffn(x, wg, wu, wd, "silu", ads, ids, B.V.twice)[0])
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves)
    want, h, p, q = B.ffn(x, wg, wu, wd, "silu", to=B.V.twice)
    B.check("train", y.detach(), want)
    for name, g, w in zip(("dx", "dwg", "dwu", "dwd"), torch.autograd.grad(y, leaves, dy),
                          B.ffn_grads(x, wg, wu, wd, dy, h, p, q, B.V.twice)):
        B.check(name, g, w)


def test_overflowing_rows(dev):
    """Values that bf16 holds no more become infinite, as of one rounding, and reach their own rows only."""
    x, wg, wu, wd = make_ffn(dev, 8, 64, 72)
    x[3] *= 1e20
    good = torch.arange(8, device=dev) != 3
    with torch.no_grad():
        y, z = kmoe.gated_ffn(x, wg, wu, wd), kmoe.gated_ffn(x[good], wg, wu, wd)
    assert torch.equal(y[good], z) and not bool(torch.isfinite(y[3]).any())


def test_ffn_gradient_is_the_difference(dev):
    """The gradients against differences of the block itself, in a direction of every input."""
    x, wg, wu, wd = make_ffn(dev, 40, 64, 72)
    dy = rnd(dev, 40, 64)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    grads = torch.autograd.grad(kmoe.gated_ffn(*leaves, "gelu"), leaves, dy)

    def f(ts):  # the block in f64, so that the difference quotient is exact to about 1e-9
        x, wg, wu, wd = ts
        return float(((torch.nn.functional.gelu(x @ wg.t()) * (x @ wu.t())) @ wd.t() * dy.double()).sum())
    base = [t.double() for t in (x, wg, wu, wd)]
    for i, g in enumerate(grads):
        way = torch.randn_like(base[i])
        eps = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + eps * way, base[i] - eps * way
        slope = (f(up) - f(down)) / (2 * eps)
        # each element is off by a few roundings of bf16 of its terms, of either sign: their sum in
        # a random direction stays within 8 of the root of their squares
        bound = 8 * 4 * 2.0 ** -8 * float((g.double() * way).norm())
        assert abs(float((g.double() * way).sum()) - slope) <= bound


@pytest.mark.parametrize("need", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 1)])
def test_ffn_some_gradients(dev, need):
    x, wg, wu, wd = make_ffn(dev, 70, 64, 136)
    dy = rnd(dev, 70, 64)
    full = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    all_g = torch.autograd.grad(kmoe.gated_ffn(*full), full, dy)
    part = [t.clone().requires_grad_(bool(k)) for t, k in zip((x, wg, wu, wd), need)]
    kmoe.gated_ffn(*part).backward(dy)
    for t, g, k in zip(part, all_g, need):
        assert (t.grad is None) if not k else torch.equal(t.grad, g)


def test_ffn_f32_weights_and_rows(dev):
    """f32 masters: products of their bf16 casts, gradients of the weights in f32, of x in x's type."""
    x, wg, wu, wd = (t.float() for t in make_ffn(dev, 100, 64, 72))
    wg = wg + 1e-4
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves)
    dy = rnd(dev, 100, 64, dtype=torch.float32)
    grads = torch.autograd.grad(y, leaves, dy)
    cast = [t.to(BF) for t in (x, wg, wu, wd)]
    want, h, p, q = B.ffn(*cast, "silu")
    assert y.dtype == torch.float32
    B.check("y", y.detach().to(BF), want)
    assert torch.equal(y.detach().to(BF).float(), y.detach())
    bw = B.ffn_grads(*cast, dy.to(BF), h, p, q)
    B.check("dx", grads[0].to(BF), bw[0])
    for g, w in zip(grads[1:], bw[1:]):
        B.check("dw", g, w, torch.float32)


def test_ffn_layouts(dev):
    """Leading dimensions, strided and misaligned inputs, no rows."""
    x, wg, wu, wd = make_ffn(dev, 96, 64, 72)
    y = kmoe.gated_ffn(x, wg, wu, wd)
    assert torch.equal(kmoe.gated_ffn(x.view(2, 4, 12, 64), wg, wu, wd), y.view(2, 4, 12, 64))
    wide = torch.randn(96, 128, device=dev).to(BF)
    wide[:, :64] = x
    assert torch.equal(kmoe.gated_ffn(wide[:, :64], wg, wu, wd), y)
    buf = torch.empty(96 * 64 + 1, device=dev, dtype=BF)
    buf[1:] = x.view(-1)
    assert torch.equal(kmoe.gated_ffn(buf[1:].view(96, 64), wg, wu, wd), y)
    assert torch.equal(kmoe.gated_ffn(x, wg.t().contiguous().t(), wu, wd), y)
    assert torch.equal(kmoe.gated_ffn(x[5], wg, wu, wd), kmoe.gated_ffn(x[5:6], wg, wu, wd)[0])
    e = x[:0].clone().requires_grad_(True)
    w = wg.clone().requires_grad_(True)
    out = kmoe.gated_ffn(e, w, wu, wd)
    out.sum().backward()
    assert out.shape == (0, 64) and e.grad.shape == (0, 64) and bool((w.grad == 0).all())


def test_rows_stay_apart(dev):
    """A row of NaN or infinities leaves the others as they were, and what lies past the rows too."""
    for T in (33, 200, 700):
        x, wg, wu, wd = make_ffn(dev, T, 136, 200)
        y = kmoe.gated_ffn(x, wg, wu, wd)
        z = x.clone()
        z[7] = float("nan")
        z[20, 3] = float("inf")
        got = kmoe.gated_ffn(z, wg, wu, wd)
        keep = torch.ones(T, dtype=torch.bool, device=dev)
        keep[[7, 20]] = False
        assert torch.equal(got[keep], y[keep]) and bool(got[7].isnan().all())


# ---------------------------------------------------------------- adapters
LINEAR = [(1, 64, 72, 3, 8), (3, 8, 8, 1, 8), (16, 72, 200, 5, 16), (48, 136, 136, 48, 16), (64, 264, 72, 2, 64), (65, 72, 136, 4, 32),
          (130, 200, 264, 7, 8), (700, 136, 520, 300, 16), (2042, 72, 392, 4, 128), (4099, 136, 1096, 11, 40),
          (16379, 72, 1032, 3, 64)]


def make_ids(dev, T, n, how):
    g = torch.Generator().manual_seed(T + n)
    if how == "mixed":
        ids = torch.randint(-1, n, (T,), generator=g)
    elif how == "runs":
        ids = torch.sort(torch.randint(0, n, (T,), generator=g)).values
        ids[T // 2: T // 2 + 3] = -1
    elif how == "none":
        ids = torch.full((T,), -1)
    else:  # ids that are no adapter's
        ids = torch.randint(0, n, (T,), generator=g)
        ids[::3] = n
        ids[1::3] = -7
    return ids.to(dev)


@pytest.mark.parametrize("how", ["mixed", "runs", "none", "outside"])
@pytest.mark.parametrize("T,K,N,n,r", LINEAR)
def test_linear(dev, T, K, N, n, r, how):
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N)
    ids = make_ids(dev, T, n, how)
    y = kmoe.adapted_linear(x, w, ad, ids)
    B.check("y", y, B.adapted(B.V(x), B.V(w), ad, ids))
    assert torch.equal(kmoe.adapted_linear(x, w, ad, ids.to(torch.int32)), y)
    if how == "none":
        assert torch.equal(kmoe.adapted_linear(x, w), y)


@pytest.mark.parametrize("how", ["mixed", "runs", "none", "outside"])
@pytest.mark.parametrize("T,K,N,n,r", LINEAR)
def test_linear_backward(dev, T, K, N, n, r, how):
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N)
    ids, dy = make_ids(dev, T, n, how), rnd(dev, T, N)
    lx, lw, la, lb = (t.clone().requires_grad_(True) for t in (x, w, ad.a, ad.b))
    y = kmoe.adapted_linear(lx, lw, kmoe.Adapters(la, lb, ad.scale), ids)
    dx, dw, da, db = torch.autograd.grad(y, (lx, lw, la, lb), dy)
    B.check("y", y.detach(), B.adapted(B.V(x), B.V(w), ad, ids))
    # dx is the adapted projection of dy by the transposed factors
    back = kmoe.Adapters(ad.b.transpose(1, 2), ad.a.transpose(1, 2), ad.scale)
    B.check("dx", dx, B.adapted(B.V(dy), B.V(w.t()), back, ids))
    B.check("dw", dw, B.mm(B.V(dy).t(), B.V(x)))
    for i in range(n) if n < 20 else (0, 1, n - 1):
        t = (ids == i).nonzero().squeeze(1)
        if t.numel() == 0:
            assert not bool(da[i].any()) and not bool(db[i].any())
            continue
        s = float(ad.scale[i])
        u = (B.mm(B.V(dy[t]), B.V(ad.b[i])) * s).bf16()
        v = (B.mm(B.V(x[t]), B.V(ad.a[i]).t()) * s).bf16()
        B.check(("da", i), da[i], B.mm(u.t(), B.V(x[t])))
        B.check(("db", i), db[i], B.mm(B.V(dy[t]).t(), v))


FACTORS = [(300, 72, 136, 3, 16), (257, 1032, 1032, 16, 8), (513, 264, 1544, 5, 16), (2042, 2048, 2048, 16, 16), (4099, 136, 264, 2, 40)]


@pytest.mark.parametrize("need", [(0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 0, 0), (0, 1, 0, 0), (1, 0, 0, 1), (0, 1, 1, 0), (1, 1, 1, 1)])
@pytest.mark.parametrize("T,K,N,n,r", FACTORS)
def test_linear_some_gradients(dev, T, K, N, n, r, need):
    """Frozen factors, weights and inputs, at sizes where one factor's gradient takes more runs of rows
    than both."""
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N)
    ids, dy = make_ids(dev, T, n, "mixed"), rnd(dev, T, N)
    lx, lw, la, lb = (t.clone().requires_grad_(bool(k)) for t, k in zip((x, w, ad.a, ad.b), need))
    kmoe.adapted_linear(lx, lw, kmoe.Adapters(la, lb, ad.scale), ids).backward(dy)
    for t, k in zip((lx, lw, la, lb), need):
        assert (t.grad is not None) == bool(k)
    if need[0]:
        back = kmoe.Adapters(ad.b.transpose(1, 2), ad.a.transpose(1, 2), ad.scale)
        B.check("dx", lx.grad, B.adapted(B.V(dy), B.V(w.t()), back, ids))
    if need[1]:
        B.check("dw", lw.grad, B.mm(B.V(dy).t(), B.V(x)))
    for i in range(n):
        t, s = (ids == i).nonzero().squeeze(1), float(ad.scale[i])
        if need[2]:
            B.check(("da", i), la.grad[i], B.mm((B.mm(B.V(dy[t]), B.V(ad.b[i])) * s).bf16().t(), B.V(x[t])))
        if need[3]:
            B.check(("db", i), lb.grad[i], B.mm(B.V(dy[t]).t(), (B.mm(B.V(x[t]), B.V(ad.a[i]).t()) * s).bf16()))


@pytest.mark.parametrize("which", ["da", "db", "both"])
@pytest.mark.parametrize("T,K,N,n,r", FACTORS)
def test_adapter_gradients_stay_in_their_workspace(dev, T, K, N, n, r, which):
    """The C entry with exactly the workspace that it asks for, and bytes of a pattern behind it."""
    x, w, ad, dy = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N), rnd(dev, T, N)
    ids = make_ids(dev, T, n, "mixed").to(torch.int32)
    ws1 = _lib.load().kmoe_adapted_linear_workspace_bytes(T, K, N, r)
    fwd, y = torch.empty(ws1, device=dev, dtype=torch.uint8), torch.empty_like(dy)
    need = _lib.load().kmoe_adapted_linear_backward_workspace_bytes(T, K, N, n, r)
    buf = torch.full((need + (16 << 20),), 0xA5, device=dev, dtype=torch.uint8)
    da = torch.empty_like(ad.a) if which != "db" else None
    db = torch.empty_like(ad.b) if which != "da" else None
    a = _lib.Adapter(ad.a.data_ptr(), ad.b.data_ptr(), ad.scale.data_ptr(), r)
    s = _lib.stream_ptr(dev)
    _lib.call("kmoe_adapted_linear", x.data_ptr(), T, K, w.data_ptr(), N, ids.data_ptr(), n, ctypes.byref(a), y.data_ptr(),
              fwd.data_ptr(), ws1, s)
    _lib.call("kmoe_adapted_linear_backward", dy.data_ptr(), x.data_ptr(), T, K, w.data_ptr(), N, ids.data_ptr(), n,
              ctypes.byref(a), fwd.data_ptr(), None, _lib.ptr(da), _lib.ptr(db), buf.data_ptr(), need, s)
    torch.cuda.synchronize()
    assert bool((buf[need:] == 0xA5).all())
    for i in (0, n - 1):
        t, f = (ids == i).nonzero().squeeze(1), float(ad.scale[i])
        if da is not None:
            B.check("da", da[i], B.mm((B.mm(B.V(dy[t]), B.V(ad.b[i])) * f).bf16().t(), B.V(x[t])))
        if db is not None:
            B.check("db", db[i], B.mm(B.V(dy[t]).t(), (B.mm(B.V(x[t]), B.V(ad.a[i]).t()) * f).bf16()))


@pytest.mark.parametrize("T", [3, 50, 300])
@pytest.mark.parametrize("which", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)])
def test_ffn_adapters(dev, T, which):
    d, F, n = 136, 200, 5
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    ads = [make_ad(dev, n, r, *kn) if k else None for k, kn, r in zip(which, ((d, F), (d, F), (F, d)), (16, 16, 24))]
    ids = make_ids(dev, T, n, "mixed")
    with torch.no_grad():
        y = kmoe.gated_ffn(x, wg, wu, wd, "silu", kmoe.FFNAdapters(*ads), ids)
    B.check("y", y, B.ffn(x, wg, wu, wd, "silu", ads, ids)[0])
    # the composed pass that trains is the same function
    lead = [t.clone().requires_grad_(True) for t in (x, *(a.a for a in ads if a))]
    it = iter(lead[1:])
    z = kmoe.gated_ffn(lead[0], wg, wu, wd, "silu", kmoe.FFNAdapters(*(a and a._replace(a=next(it)) for a in ads)), ids)
    # (it rounds the pre-activations to bf16, half a step of each, on top)
    g, u = (B.adapted(B.V(x), B.V(w), a, ids).bf16() for w, a in ((wg, ads[0]), (wu, ads[1])))
    a_, _ = B.act("silu", g)
    B.check("z", z.detach(), B.adapted((a_ * u).bf16(), B.V(wd), ads[2], ids).bf16())
    grads = torch.autograd.grad(z.float().square().sum(), lead)
    assert all(bool(torch.isfinite(t).all()) and float(t.float().abs().max()) > 0 for t in grads)


@pytest.mark.parametrize("T", [40, 300])
def test_adapters_stay_apart(dev, T):
    """An adapter of NaN reaches the rows that have it, and no others: forward and backward."""
    K, N, n, r = 72, 136, 4, 16
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=0.1), make_ad(dev, n, r, K, N)
    ids, dy = make_ids(dev, T, n, "mixed"), rnd(dev, T, N)
    bad = kmoe.Adapters(ad.a.clone(), ad.b.clone(), ad.scale)
    bad.a[2], bad.b[2, 5] = float("nan"), float("inf")
    xb = x.clone()
    xb[(ids == 2).nonzero()[0, 0]] = float("nan")

    def run(x, ad):
        lx, la, lb = (t.clone().requires_grad_(True) for t in (x, ad.a, ad.b))
        y = kmoe.adapted_linear(lx, w, kmoe.Adapters(la, lb, ad.scale), ids)
        return (y.detach(), *torch.autograd.grad(y, (lx, la, lb), dy), kmoe.adapted_linear(x, w, ad, ids))
    good, got = run(x, ad), run(xb, bad)
    rows, others = ids != 2, torch.tensor([0, 1, 3], device=dev)
    for k in (0, 1, 4):
        assert torch.equal(got[k][rows], good[k][rows]) and bool(got[k][~rows].isnan().any())
    for k in (2, 3):
        assert torch.equal(got[k][others], good[k][others])


@pytest.mark.parametrize("r", [8, 16, 40])
@pytest.mark.parametrize("T", [5, 20, 60, 300, 2042])
def test_block_adapters_stay_apart(dev, T, r):
    """The same of the block's three adapters, for each number of them that share a matrix instruction."""
    d, F, n = 72, 264, 4
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    ids = make_ids(dev, T, n, "mixed")
    ads = [make_ad(dev, n, k, *kn) for kn, k in (((d, F), r), ((d, F), r), ((F, d), 8))]
    bad = [a._replace(a=a.a.clone(), b=a.b.clone()) for a in ads]
    bad[0].b[2, 5], bad[1].b[2, 7, 0], bad[2].b[1, 3] = float("inf"), float("nan"), float("-inf")
    with torch.no_grad():
        y, z = (kmoe.gated_ffn(x, wg, wu, wd, "silu", kmoe.FFNAdapters(*a), ids) for a in (ads, bad))
    rows = (ids != 2) & (ids != 1)
    assert torch.equal(y[rows], z[rows])
    assert not bool(torch.isfinite(z[ids == 2]).any()) and not bool(torch.isfinite(z[ids == 1][:, 3]).any())
    assert torch.equal(y[ids == 1][:, 4:], z[ids == 1][:, 4:])


@pytest.mark.parametrize("T,K,N", [(8195, 1032, 1096), (2042, 1032, 5640), (48, 2056, 520), (1030, 2056, 2056)])
def test_linear_large(dev, T, K, N):
    """The large tiles with adapters, and runs of K."""
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, 5, 24, K, N)
    ids = make_ids(dev, T, 5, "runs")
    with torch.no_grad():
        B.check("y", kmoe.adapted_linear(x, w, ad, ids), B.adapted(B.V(x), B.V(w), ad, ids))
        B.check("without", kmoe.adapted_linear(x, w), B.mm(B.V(x), B.V(w).t()))


@pytest.mark.parametrize("r", [8, 16, 32])
def test_results_repeat(dev, r):
    """Which adapters share a matrix instruction is not told by the input; the results are, bit for bit."""
    T, K, N, n = 2042, 136, 2056, 200
    x, w, ad, dy = rnd(dev, T, K), rnd(dev, N, K, std=0.1), make_ad(dev, n, r, K, N), rnd(dev, T, N)
    ids = make_ids(dev, T, n, "mixed")

    def run():
        leaves = [t.clone().requires_grad_(True) for t in (x, ad.a, ad.b)]
        y = kmoe.adapted_linear(leaves[0], w, kmoe.Adapters(leaves[1], leaves[2], ad.scale), ids)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    first = run()
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_rank_is_filled_up(dev):
    """A rank that is not a multiple of 8, with its gradients."""
    T, K, N, n, r = 70, 72, 136, 3, 5
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=0.1), make_ad(dev, n, r, K, N, scale=False)
    ids, dy = make_ids(dev, T, n, "mixed"), rnd(dev, T, N)
    la, lb = (t.clone().requires_grad_(True) for t in (ad.a, ad.b))
    y = kmoe.adapted_linear(x, w, kmoe.Adapters(la, lb), ids)
    B.check("y", y.detach(), B.adapted(B.V(x), B.V(w), ad, ids))
    da, db = torch.autograd.grad(y, (la, lb), dy)
    assert da.shape == ad.a.shape and db.shape == ad.b.shape
    for i in range(n):
        t = ids == i
        u = B.mm(B.V(dy[t]), B.V(ad.b[i])).bf16()
        B.check("da", da[i], B.mm(u.t(), B.V(x[t])))


def test_ids_past_32_bits(dev):
    x, w, ad = rnd(dev, 4, 64), rnd(dev, 72, 64), make_ad(dev, 2, 8, 64, 72)
    ids = torch.tensor([1 << 32, -(1 << 40), (1 << 32) + 1, 0], device=dev)
    y = kmoe.adapted_linear(x, w, ad, ids)
    plain = kmoe.adapted_linear(x, w)
    assert torch.equal(y[:3], plain[:3]) and not torch.equal(y[3], plain[3])


# ---------------------------------------------------------------- graphs, streams, use together
def test_captured_block(dev):
    """Replays of a captured forward, with eager calls between them, and of a training step."""
    x, wg, wu, wd = make_ffn(dev, 40, 64, 136)
    ads = kmoe.FFNAdapters(make_ad(dev, 3, 8, 64, 136), None, make_ad(dev, 3, 8, 136, 64))
    ids = make_ids(dev, 40, 3, "mixed").to(torch.int32)
    with torch.no_grad():
        kmoe.gated_ffn(x, wg, wu, wd, "silu", ads, ids)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = kmoe.gated_ffn(x, wg, wu, wd, "silu", ads, ids)
        for k in range(4):
            x.copy_(rnd(dev, 40, 64))
            ids.copy_(ids.roll(1))
            wg.mul_(-1.0)
            eager = kmoe.gated_ffn(x, wg, wu, wd, "silu", ads, ids)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    dy = rnd(dev, 40, 64)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(kmoe.gated_ffn(*leaves), leaves, dy)
    for k in range(3):
        with torch.no_grad():
            leaves[0].copy_(rnd(dev, 40, 64))
            leaves[3].mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        other = [t.detach().clone().requires_grad_(True) for t in leaves]
        want = torch.autograd.grad(kmoe.gated_ffn(*other), other, dy)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_projection(dev):
    """Replays of a projection in runs of K with adapters, and of its backward; two graphs in turn."""
    x, w, ad = rnd(dev, 48, 1032), rnd(dev, 264, 1032, std=0.03), make_ad(dev, 3, 16, 1032, 264)
    ids, dy = make_ids(dev, 48, 3, "mixed").to(torch.int32), rnd(dev, 48, 264)
    with torch.no_grad():
        kmoe.adapted_linear(x, w, ad, ids)
        graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
        for k, graph in enumerate(graphs):
            with torch.cuda.graph(graph):
                outs.append(kmoe.adapted_linear(x[: 48 - 16 * k], w, ad, ids[: 48 - 16 * k]))
        for _ in range(3):
            x.copy_(rnd(dev, 48, 1032))
            ids.copy_(ids.roll(1))
            for graph in graphs:
                graph.replay()
            eager = kmoe.adapted_linear(x, w, ad, ids), kmoe.adapted_linear(x[:32], w, ad, ids[:32])
            torch.cuda.synchronize()
            assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
    leaves = [t.clone().requires_grad_(True) for t in (x, ad.a, ad.b)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kmoe.adapted_linear(leaves[0], w, kmoe.Adapters(leaves[1], leaves[2], ad.scale), ids)
        got = torch.autograd.grad(y, leaves, dy)
    for _ in range(3):
        with torch.no_grad():
            leaves[0].copy_(rnd(dev, 48, 1032))
        graph.replay()
        torch.cuda.synchronize()
        other = [t.detach().clone().requires_grad_(True) for t in leaves]
        z = kmoe.adapted_linear(other[0], w, kmoe.Adapters(other[1], other[2], ad.scale), ids)
        assert torch.equal(y, z) and all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(z, other, dy)))


def test_capture_beside_a_live_graph_is_refused(dev):
    leaves = [t.requires_grad_(True) for t in make_ffn(dev, 8, 64, 72)]
    live = kmoe.gated_ffn(*leaves)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            kmoe.gated_ffn(*leaves)
    del live


def test_two_streams(dev):
    x, wg, wu, wd = make_ffn(dev, 300, 136, 264)
    ad, ids = make_ad(dev, 4, 16, 136, 264), make_ids(dev, 300, 4, "mixed")
    y, z = kmoe.gated_ffn(x, wg, wu, wd), kmoe.adapted_linear(x, wg, ad, ids)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(5):
        for s in (a, b):
            with torch.cuda.stream(s):
                outs.append((kmoe.gated_ffn(x, wg, wu, wd), kmoe.adapted_linear(x, wg, ad, ids)))
    torch.cuda.synchronize()
    assert all(torch.equal(p, y) and torch.equal(q, z) for p, q in outs)


def test_a_written_weight_is_noticed(dev):
    leaves = [t.requires_grad_(True) for t in make_ffn(dev, 8, 64, 72)]
    y = kmoe.gated_ffn(*leaves)
    with torch.no_grad():
        leaves[1].mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def _layer(dev, **kw):
    c = kmoe.AdvancedMoEConfig(d_model=128, d_ff_expert=136, n_experts=4, moe_shared_d_ff=264, mod_enabled=False,
                               residual_dropout=0.0, **kw)
    torch.manual_seed(5)
    return c, kmoe.MoELayer(c).to(dev).to(BF)


def test_shared_expert(dev):
    """The layer with a shared expert is the layer without plus the block, in every kind of pass."""
    for routing in ("token_choice", "expert_choice"):
        c, layer = _layer(dev, moe_routing=routing)
        x = rnd(dev, 2, 40, 128)
        shared = layer.shared_expert
        for mode in (True, False):
            layer.train(mode)
            with torch.no_grad():
                y = layer(x)
                layer._modules["shared_expert"] = None
                base = layer(x)
                layer._modules["shared_expert"] = shared
                assert torch.equal(y, base + shared(x))
        xg = x.clone().requires_grad_(True)
        layer.train()(xg).float().square().sum().backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in layer.parameters())
        sd = layer.state_dict()
        assert {k for k in sd if k.startswith("shared")} == {f"shared_expert.w{i}.weight" for i in (1, 2, 3)}


@pytest.mark.parametrize("mod", [False, True])
def test_shared_expert_in_a_block(dev, mod):
    c = kmoe.AdvancedMoEConfig(d_model=128, d_ff_expert=136, n_experts=4, moe_shared_d_ff=264, mod_enabled=mod,
                               residual_dropout=0.0)
    torch.manual_seed(6)
    blk = kmoe.MoEFFNBlock(c).to(dev).to(BF).train()
    x = rnd(dev, 2, 64, 128).requires_grad_(True)
    out = blk(x)
    (out.float().square().sum() + blk.aux_loss).backward()
    assert blk.last_path == "unfused"
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for n, p in blk.named_parameters()
               if "aux_router" not in n)
    with torch.no_grad():
        blk.eval()
        y = blk(x)
        want = x + (lambda n: blk.ffn(n))(blk.ffn_norm(x))
        assert torch.equal(y, want)


def test_train_and_serve_together(dev):
    """A layer with a shared expert trained by AdamW for some steps, then adapters of its block trained
    over the frozen weights, then served: each step's weights are what the next pass takes."""
    c, layer = _layer(dev)
    layer.train()
    opt = kmoe.AdamW(layer.parameters(), lr=1e-2, state_bits=8, master_weights=True)
    x = rnd(dev, 2, 40, 128)
    for step in range(3):
        opt.zero_grad()
        y = layer(x)
        (y.float().square().mean() + layer.aux_loss).backward()
        before = {n: p.detach().clone() for n, p in layer.named_parameters()}
        opt.step()
        assert all(not torch.equal(p, before[n]) for n, p in layer.named_parameters())
        fresh = kmoe.MoELayer(c).to(dev).to(BF).train()
        fresh.load_state_dict(layer.state_dict())
        with torch.no_grad():
            assert torch.equal(layer(x), fresh(x))  # no packed copy of an old weight is left
    layer.eval().requires_grad_(False)
    ffn = layer.shared_expert
    n, r = 3, 8
    ps = [torch.nn.Parameter(rnd(dev, n, r, 128, std=0.1)), torch.nn.Parameter(torch.zeros(n, 264, r, device=dev, dtype=BF)),
          torch.nn.Parameter(rnd(dev, n, r, 264, std=0.1)), torch.nn.Parameter(torch.zeros(n, 128, r, device=dev, dtype=BF))]
    ads = kmoe.FFNAdapters(kmoe.Adapters(ps[0], ps[1]), None, kmoe.Adapters(ps[2], ps[3]))
    ids = make_ids(dev, 80, n, "mixed").view(2, 40)
    with torch.no_grad():
        assert torch.equal(ffn(x, ads, ids), ffn(x))  # outer factors of zero
    opt = kmoe.AdamW(ps, lr=1e-2)
    for step in range(2):
        opt.zero_grad()
        ffn(x, ads, ids).float().square().mean().backward()
        opt.step()
    with torch.no_grad():
        y = ffn(x, ads, ids)
        plain = ffn(x)
        assert torch.equal(y[ids < 0], plain[ids < 0]) and not torch.equal(y[ids >= 0], plain[ids >= 0])
        ws = [w.weight for w in (ffn.w1, ffn.w2, ffn.w3)]
        B.check("served", y.view(80, 128), B.ffn(x.view(80, 128), *ws, "silu", ads, ids.view(-1))[0])


def test_f32_module_follows_its_weights(dev):
    """Casts of f32 weights are kept between calls, until a weight changes."""
    ffn = kmoe.GatedFFN(64, 72).to(dev).requires_grad_(False)
    x = rnd(dev, 9, 64)
    y = ffn(x)
    assert ffn._bf16_cache is not None and torch.equal(ffn(x), y)
    ffn.w2.weight.mul_(2.0)
    z = ffn(x)
    assert torch.equal(z, kmoe.gated_ffn(x, ffn.w1.weight, ffn.w2.weight, ffn.w3.weight)) and not torch.equal(z, y)
    ffn.w1.weight.data.mul_(2.0)
    kmoe.weights_changed(ffn)
    assert not torch.equal(ffn(x), z)


# ---------------------------------------------------------------- values that are not finite
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [5, 40, 300])
def test_a_nan_of_the_gate_shows(dev, T, act):
    """In the result and in the gradients where the formula (torch's, in 64 bits) has it; of one row's
    adapter in that row."""
    x, wg, wu, wd = make_ffn(dev, T, 72, 136)
    dy = rnd(dev, T, 72)
    wg[9, 3] = float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves, act)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    lx, lg, lu, ld = ref = [t.double().requires_grad_(True) for t in (x, wg, wu, wd)]
    z = (B.TORCH_ACT[act](lx @ lg.t()) * (lx @ lu.t())) @ ld.t()
    for g, w in zip(got, (z.detach(), *torch.autograd.grad(z, ref, dy.double()))):
        assert torch.equal(g.isnan(), w.isnan())
    x, wg, wu, wd = make_ffn(dev, T, 72, 136)
    ad, ids = make_ad(dev, 3, 8, 72, 136), make_ids(dev, T, 3, "mixed")
    ids[2] = 1
    ad.b[1, 17] = float("nan")
    with torch.no_grad():
        y = kmoe.gated_ffn(x, wg, wu, wd, act, kmoe.FFNAdapters(gate=ad), ids)
    assert torch.equal(y.isnan(), (ids == 1)[:, None].expand_as(y))


def same_infinities(got, want):
    """Infinite where the formula is, of its sign, and finite elsewhere."""
    inf = want.isinf()
    assert not bool(want.isnan().any()) and bool(inf.any())
    assert torch.equal(got.isinf(), inf) and torch.equal(got[inf].double(), want[inf]) and not bool(got.isnan().any())


@pytest.mark.parametrize("r,j", [(8, 0), (16, 9), (24, 0), (32, 0), (40, 0), (40, 33), (56, 7)])
@pytest.mark.parametrize("T", [5, 20, 60, 300, 2042])
def test_infinite_factors(dev, T, r, j):
    """An infinity of an adapter's factor makes one of its sign in the rows that have the adapter: ranks past
    the last one and what the inner products lost add nothing to it."""
    d, F, n = 72, 264, 4
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    ids = make_ids(dev, T, n, "mixed")
    ids[1] = 2
    ad, up = make_ad(dev, n, r, d, F), make_ad(dev, n, r, d, F)
    delta = lambda t, ad, i: float(ad.scale[i]) * (t @ ad.a[i].double().t()) @ ad.b[i].double().t()

    def formula(t, w, ad):
        y = t @ w.double().t()
        for i in range(n):
            y[ids == i] += delta(t[ids == i], ad, i)
        return y
    ad.b[2, 130, j] = float("inf")
    with torch.no_grad():
        y = kmoe.adapted_linear(x, wu, ad, ids)
        same_infinities(y, formula(x.double(), wu, ad))
        up.b[2, 130, j] = float("-inf")
        y = kmoe.gated_ffn(x, wg, wu, wd, "silu", kmoe.FFNAdapters(up=up), ids)
        h = torch.nn.functional.silu(x.double() @ wg.double().t()) * formula(x.double(), wu, up)
        same_infinities(y, h @ wd.double().t())
    # backward: the other factor's
    ad = make_ad(dev, n, r, d, F)
    ad.a[2, j, 40] = float("inf")
    w, dy = rnd(dev, F, d, std=0.1), rnd(dev, T, F)
    lx = rnd(dev, T, d).requires_grad_(True)
    (dx,) = torch.autograd.grad(kmoe.adapted_linear(lx, w, ad, ids), lx, dy)
    back = kmoe.Adapters(ad.b.transpose(1, 2), ad.a.transpose(1, 2), ad.scale)
    same_infinities(dx, formula(dy.double(), w.t(), back))


@pytest.mark.parametrize("T", [1, 5, 8, 9, 20, 32, 40])
def test_infinite_weights(dev, T):
    """An infinity of the down projection meets the hidden values, not what these lost by their rounding."""
    for d, F in ((72, 136), (72, 2056)):
        x, wg, wu, wd = make_ffn(dev, T, d, F)
        wd[5, 77], wd[60, 3] = float("inf"), float("-inf")
        with torch.no_grad():
            y = kmoe.gated_ffn(x, wg, wu, wd)
        z = kmoe.gated_ffn(x.clone().requires_grad_(True), wg, wu, wd).detach()
        xs = x.double()
        want = (torch.nn.functional.silu(xs @ wg.double().t()) * (xs @ wu.double().t())) @ wd.double().t()
        same_infinities(y, want)
        same_infinities(z, want)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("T", [5, 40])
def test_huge_gates(dev, T, act):
    """Pre-activations whose square f32 does not hold: the activations are 0 or the gate, their slopes 0 or 1."""
    x, wg, wu, wd = make_ffn(dev, T, 72, 136)
    dy = rnd(dev, T, 72)
    wg[9] *= 1e25
    wu[9] *= 1e-25
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves, act)
    got = (y.detach(), *torch.autograd.grad(y, leaves, dy))
    assert all(bool(torch.isfinite(g).all()) for g in got)
    # row 9 of dwg: each term is off by the rounding of dgate and little else, the sum by its own
    xs, gate, up = x.double(), x.double() @ wg[9].double(), x.double() @ wu[9].double()
    on = (gate > 0).double() * up
    want = (dy.double() @ wd[:, 9].double() * on) @ xs
    terms = (dy.double().abs() @ wd[:, 9].double().abs() * on.abs()) @ xs.abs()
    assert bool((gate.abs() > 2e19).all())
    assert bool(((got[2][9].double() - want).abs() <= 4 * B.H * terms).all())


@pytest.mark.parametrize("T,F", [(5, 24), (33, 264)])
def test_saved_values_are_rounded(dev, T, F):
    """act(gate), kept in 24 bits for the backward: half a step (2^-16) off at most, to either side."""
    d = 8
    g = torch.Generator().manual_seed(T)
    x, wg, wu = torch.zeros(T, d), torch.zeros(F, d), torch.zeros(F, d)
    x[:, 0], x[:, 1] = 1.0, torch.randint(1, 3, (T,), generator=g).float()
    # gates of up to 18 bits, exact in f32
    wg[:, 0] = torch.randint(128, 256, (F,), generator=g) / 128
    wg[:, 1] = torch.randint(128, 256, (F,), generator=g) * 2.0 ** -18
    wu[:, 0] = 1.0
    want = x.double() @ wg.double().t()
    assert torch.equal(want.float().double(), want)
    wg[3, 0], wg[4, 0], wg[5, 0] = float("nan"), float("inf"), 3.3e38
    x, wg, wu = (t.to(BF).to(dev) for t in (x, wg, wu))
    wg.view(torch.int16)[6:8, 0] = torch.tensor([0x7fff, -1], dtype=torch.int16, device=dev)  # other NaN
    h = torch.empty(T, F, device=dev, dtype=BF)
    saved = torch.zeros(_lib.load().kmoe_dense_saved_bytes(T, F), device=dev, dtype=torch.uint8)
    _lib.call("kmoe_dense_gate_up", x.data_ptr(), T, d, wg.data_ptr(), wu.data_ptr(), F, _lib.ACTIVATIONS["relu"], h.data_ptr(), 0,
              saved.data_ptr(), _lib.stream_ptr(dev))
    # blocks of 16 x 16: both values, 64 lanes (4 columns / row), 4 columns, 3 bytes
    b = saved.cpu().long().view(-(-T // 16), -(-F // 16), 2, 4, 16, 4, 3)
    bits = (b[..., 0] << 8) | (b[..., 1] << 16) | (b[..., 2] << 24)
    v = bits.to(torch.int64).where(bits < 1 << 31, bits - (1 << 32)).to(torch.int32).view(torch.float32)
    v = v.permute(2, 0, 4, 1, 3, 5).reshape(2, b.shape[0] * 16, b.shape[1] * 16)[:, :T, :F]
    up, a = v[0], v[1].double()
    plain = [f for f in range(F) if f not in (3, 4, 5, 6, 7)]
    assert bool((up[:, plain] == 1).all()) and bool(a[:, [3, 6, 7]].isnan().all()) and bool((a[:, 4] == float("inf")).all())
    assert bool((a[:, 5] >= 3.2e38).all())
    off = (a - want)[:, plain] / want[:, plain]
    assert float(off.abs().max()) <= 2.0 ** -16
    # (of n values, each within half a step to either side: 5 deviations of their mean)
    assert abs(float(off.mean())) <= 5 * 2.0 ** -16 / (3 * off.numel()) ** 0.5


@pytest.mark.parametrize("r", [5, 8])
def test_captured_adapters_of_any_rank(dev, r):
    """A training step of adapters is refused beside a live graph of theirs, and else replays as it runs."""
    T, K, N, n = 70, 72, 136, 3
    x, w, ids, dy = rnd(dev, T, K), rnd(dev, N, K, std=0.1), make_ids(dev, T, n, "mixed").to(torch.int32), rnd(dev, T, N)
    a, b = rnd(dev, n, r, K, std=0.1).requires_grad_(True), rnd(dev, n, N, r, std=0.3).requires_grad_(True)
    live = kmoe.adapted_linear(x, w, kmoe.Adapters(a, b), ids)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            kmoe.adapted_linear(x, w, kmoe.Adapters(a, b), ids)
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            kmoe.gated_ffn(x, w, w, w.t().contiguous(), "silu", kmoe.FFNAdapters(gate=kmoe.Adapters(a, b)), ids)
    del live
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(kmoe.adapted_linear(x, w, kmoe.Adapters(a, b), ids), (a, b), dy)
    for _ in range(3):
        with torch.no_grad():
            x.copy_(rnd(dev, T, K))
            a.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        other = [t.detach().clone().requires_grad_(True) for t in (a, b)]
        want = torch.autograd.grad(kmoe.adapted_linear(x, w, kmoe.Adapters(*other), ids), other, dy)
        assert all(torch.equal(s, t) and s.shape == u.shape and s.is_contiguous() for s, t, u in zip(got, want, (a, b)))


def test_training_keeps_what_it_reads(dev):
    """For the backward of a projection in runs of K: the inner products, not the runs' partial sums with them;
    nothing of them where the outer factor is frozen."""
    T, K, N, n, r = 64, 5632, 2048, 3, 16
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N)
    ids, dy = make_ids(dev, T, n, "mixed"), rnd(dev, T, N)
    assert _lib.load().kmoe_adapted_linear_workspace_bytes(T, K, N, r) > 8 * T * r  # (it has runs)
    a, b = (t.clone().requires_grad_(True) for t in ad[:2])
    y = kmoe.adapted_linear(x, w, kmoe.Adapters(a, b, ad.scale), ids)
    assert sum(t.untyped_storage().nbytes() for t in y.grad_fn.saved_tensors if t is not None and t.dtype == torch.uint8) == 4 * T * r
    da, db = torch.autograd.grad(y, (a, b), dy)
    z = kmoe.adapted_linear(x, w, kmoe.Adapters(a, ad.b, ad.scale), ids)
    assert all(t is None or t.dtype != torch.uint8 for t in z.grad_fn.saved_tensors)
    assert torch.equal(torch.autograd.grad(z, a, dy)[0], da)
    for i in range(n):
        t = (ids == i).nonzero().squeeze(1)
        v = (B.mm(B.V(x[t]), B.V(ad.a[i]).t()) * float(ad.scale[i])).bf16()
        B.check("db", db[i], B.mm(B.V(dy[t]).t(), v))


@pytest.mark.parametrize("routing", ["token_choice", "expert_choice"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32, BF])
def test_shared_expert_keeps_the_result_type(dev, dtype, routing):
    """The layer's result with a shared expert has the rows' type, as without one."""
    c, layer = _layer(dev, moe_routing=routing)
    layer.eval()
    x = rnd(dev, 2, 40, 128, std=200.0, dtype=dtype)
    shared = layer.shared_expert
    with torch.no_grad():
        layer._modules["shared_expert"] = None
        base = layer(x)
        layer._modules["shared_expert"] = shared
        y = layer(x)
        assert y.dtype == base.dtype == dtype and torch.equal(y, base + shared(x))
    layer.train()
    z = layer(x.requires_grad_(True))
    z.float().sum().backward()
    assert z.dtype == y.dtype and x.grad.dtype == dtype


# ---------------------------------------------------------------- how far off, all values together
def check_rms(name, got, want, most):
    """The root mean square of got's distance from want, against that of one rounding to bf16 of want itself.
    Where a value passes two roundings of one size on its way, as a sum's own and its terms', it is
    2^0.5 times as much; terms that went missing show, which the worst cases of long sums would cover."""
    w = want.v
    one = (w.to(BF).double() - w).square().mean().sqrt()
    off = (got.double() - w).square().mean().sqrt()
    assert float(off) <= most * float(one), (name, float(off / one))


@pytest.mark.parametrize("T,d,F", [(300, 520, 264), (2042, 136, 1544), (16379, 136, 1096)] + LARGE)
def test_block_is_two_roundings_off(dev, T, d, F):
    """Past 32 rows h, dgate and dup are rounded to bf16, and so is each result."""
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    dy = rnd(dev, T, d)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves)
    want, h, p, q = B.ffn(x, wg, wu, wd, "silu")
    for name, g, w in zip(("y", "dx", "dwg", "dwu", "dwd"), (y.detach(), *torch.autograd.grad(y, leaves, dy)),
                          (want, *B.ffn_grads(x, wg, wu, wd, dy, h, p, q))):
        check_rms(name, g, w, 1.5)


@pytest.mark.parametrize("T,d,F", [(8, 520, 264), (24, 2056, 1096)])
def test_few_rows_are_one_rounding_off(dev, T, d, F):
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    dy = rnd(dev, T, d)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves)
    want, h, p, q = B.ffn(x, wg, wu, wd, "silu")
    for name, g, w in zip(("y", "dx", "dwg", "dwu", "dwd"), (y.detach(), *torch.autograd.grad(y, leaves, dy)),
                          (want, *B.ffn_grads(x, wg, wu, wd, dy, h, p, q))):
        check_rms(name, g, w, 1.1)


@pytest.mark.parametrize("T,K,N,n,r", [(300, 520, 264, 3, 16), (2042, 1032, 2056, 4, 16), (8195, 264, 1096, 11, 40)])
def test_projection_is_two_roundings_off(dev, T, K, N, n, r):
    """The result and dx have an adapter's inner products in bf16 at most; the factors' gradients those in two."""
    x, w, ad = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N)
    ids, dy = make_ids(dev, T, n, "mixed"), rnd(dev, T, N)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, ad.a, ad.b)]
    y = kmoe.adapted_linear(leaves[0], leaves[1], kmoe.Adapters(leaves[2], leaves[3], ad.scale), ids)
    dx, dw, da, db = torch.autograd.grad(y, leaves, dy)
    back = kmoe.Adapters(ad.b.transpose(1, 2), ad.a.transpose(1, 2), ad.scale)
    check_rms("y", y.detach(), B.adapted(B.V(x), B.V(w), ad, ids), 1.5)
    check_rms("dx", dx, B.adapted(B.V(dy), B.V(w.t()), back, ids), 1.5)
    check_rms("dw", dw, B.mm(B.V(dy).t(), B.V(x)), 1.1)
    for i in range(n):
        t, s = (ids == i).nonzero().squeeze(1), float(ad.scale[i])
        check_rms("da", da[i], B.mm((B.mm(B.V(dy[t]), B.V(ad.b[i])) * s).t(), B.V(x[t])), 1.1)
        check_rms("db", db[i], B.mm(B.V(dy[t]).t(), B.mm(B.V(x[t]), B.V(ad.a[i]).t()) * s), 1.1)


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("T", [3, 50, 300])
@pytest.mark.parametrize("which", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1)])
def test_block_adapters_gradients(dev, T, which, act):
    """Every gradient of the block with adapters against the formula's, with the roundings of its three
    projections: pre-activations, h and the gradients between the projections are bf16."""
    d, F, n = 136, 200, 4
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    ads = [make_ad(dev, n, r, *kn) if k else None for k, kn, r in zip(which, ((d, F), (d, F), (F, d)), (16, 16, 24))]
    ids, dy = make_ids(dev, T, n, "mixed"), rnd(dev, T, d)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, wd)]
    factors = [tuple(t.clone().requires_grad_(True) for t in ad[:2]) if ad else None for ad in ads]
    y = kmoe.gated_ffn(*leaves, act, kmoe.FFNAdapters(*(f and kmoe.Adapters(*f, ad.scale) for f, ad in zip(factors, ads))), ids)
    every = leaves + [t for f in factors if f for t in f]
    got = dict(zip(map(id, every), torch.autograd.grad(y, every, dy)))
    V, turned = B.V, [ad and kmoe.Adapters(ad.b.transpose(1, 2), ad.a.transpose(1, 2), ad.scale) for ad in ads]
    g, u = B.adapted(V(x), V(wg), ads[0], ids).bf16(), B.adapted(V(x), V(wu), ads[1], ids).bf16()
    a, slope = B.act(act, g)
    h = (a * u).bf16()
    dh = B.adapted(V(dy), V(wd).t(), turned[2], ids).bf16()
    dg, du = (dh * u * slope).bf16(), (dh * a).bf16()
    dx = B.adapted(dg, V(wg).t(), turned[0], ids).bf16() + B.adapted(du, V(wu).t(), turned[1], ids).bf16()
    # eight roundings to bf16 on the way to any of them, independent and each of 2^-8 3^-0.5 of its value at most
    # in the root mean square; the pre-activations' reach h and the slopes by up to 1.13: 3 2^-8 in all
    def close(name, a, b):
        B.check(name, a, b)
        assert float((a.double() - b.v).norm()) <= 3 * 2.0 ** -8 * float(b.v.norm()), name
    close("dx", got[id(leaves[0])], dx)
    for name, leaf, w in zip(("dwg", "dwu", "dwd"), leaves[1:], (B.mm(dg.t(), V(x)), B.mm(du.t(), V(x)), B.mm(V(dy).t(), h))):
        close(name, got[id(leaf)], w)
    for name, ad, f, rows, grad in zip(("gate", "up", "down"), ads, factors, (V(x), V(x), h), (dg, du, V(dy))):
        for i in range(n) if ad else ():
            t, s = (ids == i).nonzero().squeeze(1), float(ad.scale[i])
            if t.numel() == 0:
                assert not bool(got[id(f[0])][i].any()) and not bool(got[id(f[1])][i].any())
                continue
            rt, gt = V(rows.v[t], rows.e[t]), V(grad.v[t], grad.e[t])
            close((name, "da"), got[id(f[0])][i], B.mm((B.mm(gt, V(ad.b[i])) * s).bf16().t(), rt))
            close((name, "db"), got[id(f[1])][i], B.mm(gt.t(), (B.mm(rt, V(ad.a[i]).t()) * s).bf16()))
    # the formula itself, by torch's gradients in 64 bits
    ref = [t.detach().double().requires_grad_(True) for t in every]
    it = iter(ref[4:])
    pairs = [(next(it), next(it)) if f else None for f in factors]

    def project(v, w, ad, f):
        out = v @ w.t()
        for i in range(n) if f else ():
            out = out + (ids == i)[:, None] * (float(ad.scale[i]) * (v @ f[0][i].t()) @ f[1][i].t())
        return out
    gates = [project(ref[0], w, ad, f) for w, ad, f in zip(ref[1:3], ads, pairs)]
    out = project(B.TORCH_ACT[act](gates[0]) * gates[1], ref[3], ads[2], pairs[2])
    for leaf, w in zip(every, torch.autograd.grad(out, ref, dy.double())):
        assert float((got[id(leaf)].double() - w).norm()) <= 3 * 2.0 ** -8 * float(w.norm())


def test_shared_expert_under_mod_by_value(dev):
    """With a shared expert the kept rows' outputs are those without it plus the block's, weighted alike."""
    c = kmoe.AdvancedMoEConfig(d_model=128, d_ff_expert=136, n_experts=4, moe_shared_d_ff=264, mod_enabled=True,
                               residual_dropout=0.0)
    torch.manual_seed(8)
    mod = kmoe.MoDMoE(c).to(dev).to(BF).train()
    x, res = rnd(dev, 2, 64, 128), rnd(dev, 2, 64, 128)
    shared = mod.ffn.shared_expert
    with torch.no_grad():
        y = mod(x, res)
        mod.ffn._modules["shared_expert"] = None
        base = mod(x, res)
        mod.ffn._modules["shared_expert"] = shared
        sel = mod.ffn_mod_router.select(x)
        rows = sel.sel_idx.long()
        s = shared(torch.stack([x[b, rows[b]] for b in range(2)])).double()
    add = torch.zeros(2, 64, 128, device=dev, dtype=torch.float64)
    for b in range(2):
        add[b, rows[b]] = sel.sel_w[b].double()[:, None] * s[b]
    want = base.double() + add
    # half a step of bf16 each: base's and y's own rounding; the experts' rows twice (theirs and their sum with
    # the block's) and the block's twice, with the rows' weights
    off = B.H * (base.double().abs() + want.abs() + 2 * (base.double() - res.double()).abs() + 2 * add.abs())
    assert bool(((y.double() - want).abs() <= 1.01 * off + 1e-6).all())
    assert float(add.abs().max()) > 0.01


def test_no_rows_with_adapters(dev):
    """No tokens: results of no rows, zero gradients of the adapters."""
    x, wg, wu, wd = make_ffn(dev, 3, 64, 72)
    ads = [make_ad(dev, 2, 8, 64, 72), make_ad(dev, 2, 8, 64, 72), make_ad(dev, 2, 5, 72, 64)]
    e, ids = x[:0].clone().requires_grad_(True), torch.zeros(0, device=dev, dtype=torch.int64)
    with torch.no_grad():
        assert kmoe.gated_ffn(e, wg, wu, wd, "silu", kmoe.FFNAdapters(*ads), ids).shape == (0, 64)
        assert kmoe.adapted_linear(e, wg, ads[0], ids).shape == (0, 72)
    f = [t.clone().requires_grad_(True) for a in ads for t in a[:2]]
    y = kmoe.gated_ffn(e, wg, wu, wd, "silu", kmoe.FFNAdapters(*(kmoe.Adapters(*f[2 * i:2 * i + 2]) for i in range(3))), ids)
    y.sum().backward()
    assert e.grad.shape == (0, 64) and all(bool((t.grad == 0).all()) for t in f)


# ---------------------------------------------------------------- offsets past 32 bits
def test_rows_past_32_bits(dev):
    """More than 2^31 values of x, of dy's gradient and of h."""
    T, K, N, n, r = (1 << 20) + 5, 2056, 72, 3, 8
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.empty(T, K, device=dev, dtype=BF).normal_(generator=g)
    w, ad, dy = rnd(dev, N, K, std=K ** -0.5), make_ad(dev, n, r, K, N), torch.empty(T, N, device=dev, dtype=BF).normal_(generator=g)
    ids = torch.randint(-1, n, (T,), device=dev, generator=g)
    leaves = [t.requires_grad_(True) for t in (x, ad.a, ad.b)]
    y = kmoe.adapted_linear(x, w, kmoe.Adapters(leaves[1], leaves[2], ad.scale), ids)
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    y, x, a, b = (t.detach() for t in (y, *leaves))
    ad, back = kmoe.Adapters(a, b, ad.scale), kmoe.Adapters(b.transpose(1, 2), a.transpose(1, 2), ad.scale)
    for rows in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        B.check("y", y[rows], B.adapted(B.V(x[rows]), B.V(w), ad, ids[rows]))
        B.check("dx", dx[rows], B.adapted(B.V(dy[rows]), B.V(w.t()), back, ids[rows]))
    wa, wb = torch.zeros(n, r, K, device=dev, dtype=torch.float64), torch.zeros(n, N, r, device=dev, dtype=torch.float64)
    for t0 in range(0, T, 1 << 17):
        xs, ds, own = x[t0:t0 + (1 << 17)].double(), dy[t0:t0 + (1 << 17)].double(), ids[t0:t0 + (1 << 17)]
        for i in range(n):
            on = (own == i)[:, None] * float(ad.scale[i])
            wa[i] += (ds @ b[i].double() * on).t() @ xs
            wb[i] += ds.t() @ (xs @ a[i].double().t() * on)
    check_rms("da", da, B.V(wa), 1.1)
    check_rms("db", db, B.V(wb), 1.1)


def test_block_past_32_bits(dev):
    T, d, F = (1 << 18) + 3, 72, 8200
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    dy = rnd(dev, T, d)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = kmoe.gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    y, x, wg, wu, wd = (t.detach() for t in (y, *leaves))
    sums = [torch.zeros(F, d, device=dev, dtype=torch.float64), torch.zeros(F, d, device=dev, dtype=torch.float64),
            torch.zeros(d, F, device=dev, dtype=torch.float64)]
    for t0 in range(0, T, 1 << 14):
        rows = slice(t0, t0 + (1 << 14))
        xs, ds = x[rows].double(), dy[rows].double()
        gate, up = xs @ wg.double().t(), xs @ wu.double().t()
        s = torch.sigmoid(gate)
        a, dh = gate * s, ds @ wd.double()
        dg, du = dh * up * s * (1 + gate * (1 - s)), dh * a
        check_rms("y", y[rows], B.V((a * up) @ wd.double().t()), 1.5)
        check_rms("dx", grads[0][rows], B.V(dg @ wg.double() + du @ wu.double()), 1.5)
        for total, part in zip(sums, (dg.t() @ xs, du.t() @ xs, ds.t() @ (a * up))):
            total += part
    for name, g, w in zip(("dwg", "dwu", "dwd"), grads[1:], sums):
        check_rms(name, g, B.V(w), 1.5)


def test_adapters_past_32_bits(dev):
    """Factors of many adapters: more than 2^31 values each, the last ones used."""
    T, K, N, n, r = 130, 1032, 1032, 16500, 128
    x, w, dy = rnd(dev, T, K), rnd(dev, N, K, std=K ** -0.5), rnd(dev, T, N)
    a, b = torch.zeros(n, r, K, device=dev, dtype=BF), torch.zeros(n, N, r, device=dev, dtype=BF)
    used = (0, n // 2, n - 2, n - 1)
    for i in used:
        a[i], b[i] = rnd(dev, r, K, std=K ** -0.5), rnd(dev, N, r, std=0.3)
    ids = torch.tensor(used, device=dev)[torch.arange(T, device=dev) % 4]
    ad = kmoe.Adapters(a.requires_grad_(True), b.requires_grad_(True))
    lx = x.clone().requires_grad_(True)
    y = kmoe.adapted_linear(lx, w, ad, ids)
    dx, da, db = torch.autograd.grad(y, (lx, a, b), dy)
    few = kmoe.Adapters(a.detach()[list(used)], b.detach()[list(used)])
    back, at = kmoe.Adapters(few.b.transpose(1, 2), few.a.transpose(1, 2)), torch.arange(T, device=dev) % 4
    for rows in (slice(0, T), slice(0, 5)):
        with torch.no_grad():
            B.check("y", kmoe.adapted_linear(x[rows], w, ad, ids[rows]), B.adapted(B.V(x[rows]), B.V(w), few, at[rows]))
    B.check("dx", dx, B.adapted(B.V(dy), B.V(w.t()), back, at))
    for k, i in enumerate(used):
        t = at == k
        B.check("da", da[i], B.mm(B.mm(B.V(dy[t]), B.V(few.b[k])).bf16().t(), B.V(x[t])))
        B.check("db", db[i], B.mm(B.V(dy[t]).t(), B.mm(B.V(x[t]), B.V(few.a[k]).t()).bf16()))
    assert not bool(da[1:n // 2].any()) and not bool(db[n // 2 + 1:n - 2].any())


@pytest.mark.parametrize("r", [8, 16, 32])
@pytest.mark.parametrize("T", [14, 30, 60, 300])
def test_many_infinite_adapters_stay_apart(dev, T, r):
    """Every second of many adapters with infinities: turns of the tile with and without them, in every place of
    a group of turns; the others' rows are the same bit for bit, and theirs are the formula's."""
    d, F, n = 72, 264, 150
    x, wg, wu, wd = make_ffn(dev, T, d, F)
    ads = [make_ad(dev, n, k, *kn) for kn, k in (((d, F), r), ((d, F), r), ((F, d), r))]
    bad = [a._replace(b=a.b.clone()) for a in ads]
    ids = torch.arange(T, device=dev) * 7 % n
    for i in range(0, n, 3):
        bad[1].b[i, i % F, i % r], bad[2].b[i, i % d, (i + 1) % r] = float("inf"), float("-inf")
    clean = ids % 3 != 0
    with torch.no_grad():
        y, z = (kmoe.gated_ffn(x, wg, wu, wd, "silu", kmoe.FFNAdapters(*a), ids) for a in (ads, bad))
        assert torch.equal(y[clean], z[clean]) and not bool(torch.isfinite(z[~clean]).all(dim=1).any())
        p, q = (kmoe.adapted_linear(x, wu, a, ids) for a in (ads[1], bad[1]))
    assert torch.equal(p[clean], q[clean])
    finite = ~(torch.arange(F, device=dev)[None] == (ids % F)[:, None])
    assert torch.equal(p[~clean][finite[~clean]], q[~clean][finite[~clean]])
    want = x.double() @ wu.double().t()
    for t in range(T):
        i = int(ids[t])
        want[t] += float(ads[1].scale[i]) * (x[t].double() @ ads[1].a[i].double().t()) @ bad[1].b[i].double().t()
    same_infinities(q, want)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("T", [12, 300])
def test_captured_training_steps(dev, T, bits):
    """Forward, backward and optimizer step of the block and of adapters on it in one graph: its replays are the
    eager steps, bit for bit, with eager passes of the same weights between them."""
    x, dy = rnd(dev, T, 72), rnd(dev, T, 72)
    ids = make_ids(dev, T, 3, "mixed").to(torch.int32)
    start = [*make_ffn(dev, T, 72, 136)[1:], *make_ad(dev, 3, 5, 72, 136)[:2], *make_ad(dev, 3, 8, 136, 72)[:2]]

    def make():
        ps = [torch.nn.Parameter(t.clone()) for t in start]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, kmoe.AdamW(ps, lr=1e-2, state_bits=bits, master_weights=True)

    def run(ps, opt):
        ads = kmoe.FFNAdapters(kmoe.Adapters(ps[3], ps[4]), None, kmoe.Adapters(ps[5], ps[6]))
        y = kmoe.gated_ffn(x, *ps[:3], "gelu", ads, ids)
        for p, g in zip(ps, torch.autograd.grad(y, ps, dy)):
            p.grad.copy_(g)
        opt.step()
        return y.detach()
    (ps, opt), (qs, eager) = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(ps, opt)
        run(qs, eager)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run(ps, opt)
    for _ in range(4):
        x.mul_(-1.0)
        ids.copy_(ids.roll(1))
        graph.replay()
        with torch.no_grad():
            kmoe.gated_ffn(x, *ps[:3], "gelu")
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            want = run(qs, eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(ps, qs))
        assert all(torch.equal(opt.state[p][k], eager.state[q][k]) for p, q in zip(ps, qs) for k in opt.state[p])
