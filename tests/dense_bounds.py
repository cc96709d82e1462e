"""Values in 64 bits with a bound on how far the kernels' may be off, carried through the formulas of
the dense operators: every product's f32 sums, every rounding to bf16, every activation."""
import math

import torch

U = 2.0 ** -24   # half a step of f32
H = 2.0 ** -8    # half a step of bf16


TORCH_ACT = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh"), "relu": torch.relu}


class V:
    """A value and a bound on the distance of the kernel's from it."""

    def __init__(self, v, e=None):
        self.v, self.e = v.double(), torch.zeros_like(v, dtype=torch.float64) if e is None else e

    def t(self):
        return V(self.v.t(), self.e.t())

    def __add__(self, o):  # a sum in f32
        v = self.v + o.v
        return V(v, self.e + o.e + U * v.abs())

    def __mul__(self, o):  # a product in f32
        if not isinstance(o, V):
            return V(self.v * o, self.e * abs(o) + U * (self.v * o).abs())
        v = self.v * o.v
        return V(v, self.e * o.v.abs() + self.v.abs() * o.e + self.e * o.e + U * v.abs())

    def bf16(self):
        return V(self.v, self.e + H * (self.v.abs() + self.e) + 1e-40)

    def twice(self):  # as two bf16, the second what the first lost
        return V(self.v, self.e + H * H * (self.v.abs() + self.e) + 1e-40)


def mm(a, b):
    """A matrix product with f32 sums of K terms: products of bf16 numbers are exact, each sum
    may lose a whole step (the matrix cores' rounding is not told)."""
    K = a.v.shape[1]
    aa, bb = a.v.abs(), b.v.abs()
    return V(a.v @ b.v, a.e @ bb + aa @ b.e + a.e @ b.e + 2 * K * U * (aa @ bb))


def act(name, g):
    """(act(g), act'(g)): the input's bound by the steepest slope (1.13) and curvature (0.8, relu: a
    step at 0), and what the hardware's exponential and reciprocal are off (2^-16 of the value
    covers arguments up to 80; the tails of both gelus cancel in f32: 2^-21 |g|)."""
    x = g.v
    if name == "silu":
        s = torch.sigmoid(x)
        a, d = x * s, s * (1 + x * (1 - s))
    elif name == "gelu":
        c = 0.5 * (1 + torch.erf(x / math.sqrt(2.0)))
        a, d = x * c, c + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    elif name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x ** 3))
        a, d = 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 0.134145 * x * x)
    else:
        return V(torch.relu(x), g.e), V((x > 0).double(), (x.abs() <= g.e).double())
    off = 2.0 ** -16
    # (the derivatives' terms reach 1 + |g|)
    return V(a, 1.13 * g.e + off * a.abs() + 2.0 ** -21 * x.abs()), V(d, 0.8 * g.e + off * (1 + d.abs()))


def adapted(x, w, ad, ids, to=V.bf16):
    """x w^T + scale (x a^T) b^T of each row's adapter, before its last rounding."""
    y = mm(x, w.t())
    if ad is None:
        return y
    a, b, scale = ad
    v, e = y.v.clone(), y.e.clone()
    for i in range(a.shape[0]):
        t = (ids == i).nonzero().squeeze(1)
        if t.numel():
            s = 1.0 if scale is None else float(scale[i])
            inner = to(mm(V(x.v[t], x.e[t]), V(a[i]).t()) * s)
            d = mm(inner, V(b[i]).t())
            v[t] += d.v
            e[t] += d.e + U * v[t].abs()
    return V(v, e)


def cut24(a):
    """A value cut to the top 24 bits of its f32: up to 2^-15 of it lost."""
    return V(a.v, a.e + 2.0 ** -15 * (a.v.abs() + a.e) + 1e-40)


def ffn(x, wg, wu, wd, name, ads=(None, None, None), ids=None, to=V.bf16):
    """(y before its last rounding, and for the backward h, p, q) of the gated block; to: how h and the
    adapters' inner products are held."""
    x, wg, wu, wd = V(x), V(wg), V(wu), V(wd)
    g, u = adapted(x, wg, ads[0], ids, to), adapted(x, wu, ads[1], ids, to)
    a, d = act(name, g)
    h = to(a * u)
    return adapted(h, wd, ads[2], ids, to), h, cut24(d * u), cut24(a)


def ffn_grads(x, wg, wu, wd, dy, h, p, q, to=V.bf16):
    """Bounded gradients of x, wg, wu, wd before their last rounding; to: how dgate and dup are held."""
    dh = mm(V(dy), V(wd))
    dg, du = to(dh * p), to(dh * q)
    # (one sum over both parts)
    cat = lambda a, b, k: V(torch.cat((a.v, b.v), k), torch.cat((a.e, b.e), k))
    dx = mm(cat(dg, du, 1), cat(V(wg), V(wu), 0))
    return dx, mm(dg.t(), V(x)), mm(du.t(), V(x)), mm(V(dy).t(), h)


def check(name, got, want, dtype=torch.bfloat16):
    """got within want's bound and the rounding to its type."""
    e = want.e + (H if dtype == torch.bfloat16 else U) * (want.v.abs() + want.e) + 1e-30
    off = (got.double() - want.v).abs()
    assert got.dtype == dtype and got.shape == want.v.shape, (name, got.dtype, got.shape, want.v.shape)
    bad = ~(off <= e)
    assert not bool(bad.any()), (name, int(bad.sum()), float((off / e).max()), bad.nonzero()[:3].tolist())
    return float((off / e).max())
