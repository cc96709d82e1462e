"""Dense operators beside the routed experts, on weights as torch.nn.Linear holds them.

* gated_ffn: the gated feed-forward block (act(x Wg^T) * (x Wu^T)) Wd^T (SwiGLU of
  moe_arch/model/ffn.py:17-64 with act = silu), the layers without experts and the expert that all
  tokens share (MoELayer's moe_shared_d_ff); without gradients in one native call, with its
  backward on the HIP kernels.  No packed copies: a step's new weights cost nothing.
* adapted_linear: a shared projection with low-rank adapters of many requests in one batch,
  row t with the adapter ids[t]; also on all three projections of the block.

Numerics: bf16 operands, f32 sums.  What is rounded to bf16 between the products: the block's hidden
values h = act(g) u and the gradients of its pre-activations (of up to 32 rows both keep 16 bits, as
two bf16: in few results a rounding does not average out), and an adapter's inner products with
their scale (16 bits for the factors' gradients).  What the backward keeps of the pre-activations,
u act'(g) and act(g), has 16 bits of precision.  An infinite weight or factor gives the infinities of the
formula in the results of its rows; gradients summed over a row with an infinity are not finite.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from . import backward as _bwd
from ._lib import ptr
from .derived import derived
from .ops import _BF16, _contig, _device, _one_gpu, _Stage, _stream


class Adapters(NamedTuple):
    """n low-rank adapters of one projection (N, K): row t gets scale[i] (x a[i]^T) b[i]^T, i = ids[t].
    a (n, r, K), b (n, N, r); scale (n,) f32, None for 1.  Ranks up to 128; one that is not a
    multiple of 8 is filled up with zeros in every call, so a program that serves keeps it filled."""
    a: torch.Tensor
    b: torch.Tensor
    scale: Optional[torch.Tensor] = None


class FFNAdapters(NamedTuple):
    """Adapters of a gated block's projections, None where there are none; the gate's and the up
    projection's have one rank."""
    gate: Optional[Adapters] = None
    up: Optional[Adapters] = None
    down: Optional[Adapters] = None


# ---------------------------------------------------------------- checks
def _act(activation) -> int:
    try:
        return _lib.ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"kmoe.gated_ffn: activation {activation!r} is none of {sorted(_lib.ACTIVATIONS)}") from None


def _weight(w, rows, cols, who, name):
    if w.dim() != 2 or (rows is not None and w.shape[0] != rows) or (cols is not None and w.shape[1] != cols):
        raise ValueError(f"kmoe.{who}: {name} must be ({'N' if rows is None else rows}, {'K' if cols is None else cols}), got "
                         f"{tuple(w.shape)}")
    if w.dtype not in (_BF16, torch.float32):
        raise ValueError(f"kmoe.{who}: {name} is bf16 or f32, got {w.dtype}")
    if w.shape[0] % 8 or w.shape[1] % 8 or not w.numel():
        raise ValueError(f"kmoe.{who}: {name} {tuple(w.shape)}: sizes are positive multiples of 8")


def _rows(x, K, who):
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"kmoe.{who}: x {tuple(x.shape)} has rows of {K} values for these weights")
    if not x.dtype.is_floating_point:
        raise ValueError(f"kmoe.{who}: x is floating point, got {x.dtype}")


def _adapters(ad, K, N, who, name):
    """The adapters checked."""
    a, b, scale = ad
    n, r = a.shape[:2] if a.dim() == 3 else (0, 0)
    if not 1 <= r <= _lib.MAX_RANK or not 1 <= n <= 32767 or a.shape[2] != K or b.shape != (n, N, r):
        raise ValueError(f"kmoe.{who}: {name}a must be (n, r, {K}) and b (n, {N}, r), n up to 32767 and r up to "
                         f"{_lib.MAX_RANK}, got {tuple(a.shape)}, {tuple(b.shape)}")
    if scale is not None:
        if scale.shape != (n,):
            raise ValueError(f"kmoe.{who}: {name}scale must be ({n},), got {tuple(scale.shape)}")
        if scale.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"kmoe.{who}: {name}scale has no gradient here: pass it detached")
        scale = _contig(scale.detach(), torch.float32)
    return Adapters(a, b, scale)


def _ids(ids, x, n, who):
    if ids is None:
        raise ValueError(f"kmoe.{who}: adapters need ids, the adapter of each row (-1: none)")
    if ids.shape != x.shape[:-1]:
        raise ValueError(f"kmoe.{who}: ids {tuple(ids.shape)} are not one for each row of x {tuple(x.shape)}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"kmoe.{who}: ids are int32 or int64, got {ids.dtype}")
    if ids.dtype == torch.int64:  # (an id past 32 bits is no adapter, not another one's)
        ids = ids.clamp(-1, n).to(torch.int32)
    return ids.reshape(-1).contiguous()


def _struct(ad):
    """kmoe_adapter of bf16 contiguous adapters (the caller keeps the tensors)."""
    return None if ad is None else ctypes.byref(_lib.Adapter(ad.a.data_ptr(), ad.b.data_ptr(), ptr(ad.scale), ad.a.shape[1]))


def _held(ad):
    """The adapters as the kernels take them: bf16, ranks filled up to a multiple of 8 with zeros."""
    if ad is None:
        return None
    a, b = _ready(ad.a), _ready(ad.b)
    fill = -a.shape[1] % 8
    if fill:
        a, b = nn.functional.pad(a, (0, 0, 0, fill)), nn.functional.pad(b, (0, fill))
    return Adapters(a, b, ad.scale)


def _ready(t):
    """t's values in bf16, contiguous, at a multiple of 16 bytes: t itself where it is so already."""
    if t.dtype is _BF16 and t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    t = _contig(t.detach(), _BF16)
    return t if t.data_ptr() % 16 == 0 else t.clone()


@functools.lru_cache(maxsize=1024)
def _ffn_workspace(device, T, d, F, rgu, rd) -> int:
    return _lib.load().kmoe_gated_ffn_workspace_bytes(T, d, F, rgu, rd)


@functools.lru_cache(maxsize=1024)
def _linear_workspace(device, T, K, N, r) -> int:
    return _lib.load().kmoe_adapted_linear_workspace_bytes(T, K, N, r)


@functools.lru_cache(maxsize=1024)
def _linear_backward_workspace(device, T, K, N, n, r) -> int:
    return _lib.load().kmoe_adapted_linear_backward_workspace_bytes(T, K, N, n, r)


# ---------------------------------------------------------------- without gradients
def _ffn_forward(x, wg, wu, wd, act, ads, ids):
    F, d = wg.shape
    T = x.numel() // d
    dev = x.device
    y = torch.empty_like(x)
    gate, up, down = ads if ads is not None else (None, None, None)
    some = gate or up or down
    rgu = gate.a.shape[1] if gate is not None else up.a.shape[1] if up is not None else 0
    with _device(dev), _Stage("gated_ffn"):
        wsb = _ffn_workspace(dev.index, T, d, F, rgu, down.a.shape[1] if down is not None else 0)
        ws = torch.empty(wsb, device=dev, dtype=torch.uint8)
        _lib.call("kmoe_gated_ffn", x.data_ptr(), T, d, F, wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), act, ptr(ids),
                  some.a.shape[0] if some else 0, _struct(gate), _struct(up), _struct(down), y.data_ptr(), ws.data_ptr(), wsb,
                  _stream(x))
    return y


def _linear_forward(x, w, ad, ids):
    N, K = w.shape
    T = x.numel() // K
    dev = x.device
    y = x.new_empty(x.shape[:-1] + (N,))
    n, r = ad.a.shape[:2] if ad is not None else (0, 0)
    with _device(dev), _Stage("adapted_linear"):
        wsb = _linear_workspace(dev.index, T, K, N, r)
        ws = torch.empty(wsb, device=dev, dtype=torch.uint8) if wsb else None
        _lib.call("kmoe_adapted_linear", x.data_ptr(), T, K, w.data_ptr(), N, ptr(ids), n, _struct(ad), y.data_ptr(), ptr(ws),
                  wsb, _stream(x))
    return y, ws


# ---------------------------------------------------------------- parts of the backward
def _dense_dx(dy, w, T, dy2=None, w2=None):
    """dy w (+ dy2 w2) of T rows; rows behind those are what they lost by their rounding."""
    N, K = w.shape
    dx = torch.empty(T, K, device=dy.device, dtype=_BF16)
    _lib.call("kmoe_dense_dx", ptr(dy), ptr(dy2), int(dy.shape[0] > T), T, N, ptr(w), ptr(w2), K, ptr(dx), _stream(dy))
    return dx


def _dense_wgrad(a, b, T, dtype):
    """a^T b of T rows, (M, N), in the weight's type; rows behind those (of one of the two) are what they
    lost by their rounding."""
    M, N = a.shape[1], b.shape[1]
    dt = torch.float32 if dtype == torch.float32 else _BF16
    c = torch.empty(M, N, device=a.device, dtype=dt)
    a2, b2 = (a[-T:], b[-T:]) if T and max(a.shape[0], b.shape[0]) > T else (None, None)
    _lib.call("kmoe_dense_wgrad", ptr(a), ptr(b), ptr(a2), ptr(b2), T, M, N, ptr(c),
              _lib.DTYPE_F32 if dt == torch.float32 else _lib.DTYPE_BF16, _stream(a))
    return c


# ---------------------------------------------------------------- the gated block
def _copied(*pairs):
    """The tensors whose values in bf16 are copies.  They are saved too, so that a write to one before the
    backward is refused; of the others the saved values are the tensor itself."""
    return tuple(t for t, held in pairs if t is not None and held is not t)


class _GatedFFNFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, wg, wu, wd, act):
        _bwd.leaves_of(ctx, x, wg, wu, wd)
        xr, bg, bu, bd = _ready(x), _ready(wg), _ready(wu), _ready(wd)
        F, d = bg.shape
        T = xr.numel() // d
        lost = int(T <= _lib.LOST_ROWS)
        h = xr.new_empty((T + T * lost, F))
        saved = torch.empty(max(_lib.load().kmoe_dense_saved_bytes(T, F), 16), device=x.device, dtype=torch.uint8)
        y = xr.new_empty(x.shape)
        with _device(x.device):
            with _Stage("ffn_gate_up"):
                _lib.call("kmoe_dense_gate_up", ptr(xr), T, d, ptr(bg), ptr(bu), F, act, ptr(h), lost, ptr(saved), _stream(x))
            with _Stage("ffn_down"):
                _lib.call("kmoe_dense_linear", ptr(h), lost, T, F, ptr(bd), d, ptr(y), _stream(x))
        ctx.save_for_backward(xr, h, saved, bg, bu, bd, *_copied((x, xr), (wg, bg), (wu, bu), (wd, bd)))
        ctx.meta = (x.dtype, wg.dtype, wu.dtype, wd.dtype)
        return y if x.dtype is _BF16 else y.to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xr, h, saved, bg, bu, bd = ctx.saved_tensors[:6]
        dtypes = ctx.meta
        F, d = bg.shape
        T = xr.numel() // d
        need_x, need_g, need_u, need_d = ctx.needs_input_grad[:4]
        dy2, x2d = _ready(dy).view(T, d), xr.view(T, d)
        dx = dg = du = dwg = dwu = dwd = None
        with _device(xr.device):
            if need_x or need_g or need_u:
                dg, du = torch.empty_like(h), torch.empty_like(h)
                with _Stage("bwd_ffn_dh"):
                    _lib.call("kmoe_dense_dh", ptr(dy2), T, d, ptr(bd), F, ptr(saved), ptr(dg), ptr(du),
                              int(h.shape[0] > T), _stream(xr))
            if need_x:
                with _Stage("bwd_ffn_dx"):
                    dx = _dense_dx(dg, bg, T, du, bu).view(xr.shape).to(dtypes[0])
            with _Stage("bwd_ffn_wgrad"):
                if need_g:
                    dwg = _dense_wgrad(dg, x2d, T, dtypes[1])
                if need_u:
                    dwu = _dense_wgrad(du, x2d, T, dtypes[2])
                if need_d:
                    dwd = _dense_wgrad(dy2, h, T, dtypes[3])
        return dx, dwg, dwu, dwd, None


_ACT_FN = {"silu": nn.functional.silu, "gelu": nn.functional.gelu,
           "gelu_tanh": functools.partial(nn.functional.gelu, approximate="tanh"), "relu": torch.relu}


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def gated_ffn(x, w_gate, w_up, w_down, activation="silu", adapters: Optional[FFNAdapters] = None, ids=None):
    """(act(x w_gate^T) * (x w_up^T)) w_down^T for rows x (..., d): w_gate, w_up (F, d), w_down (d, F), bf16
    or f32 (cast to bf16 in the call), d and F multiples of 8; activation "silu", "gelu",
    "gelu_tanh" or "relu".  The result has x's type.  adapters with ids (..., int32 or int64): each row's
    own low-rank adapter on the three projections, -1 (or any id that is no adapter) for none.

    Differentiable in x, the weights and the adapters; with adapters the projections then run one by
    one and the activation between them is torch's."""
    act = _act(activation)
    _weight(w_gate, None, None, "gated_ffn", "w_gate")
    F, d = w_gate.shape
    _weight(w_up, F, d, "gated_ffn", "w_up")
    _weight(w_down, d, F, "gated_ffn", "w_down")
    _rows(x, d, "gated_ffn")
    if adapters is not None and not any(a is not None for a in adapters):
        adapters = None
    if adapters is None:
        _one_gpu("gated_ffn", x, w_gate, w_up, w_down)
        if _wants_grad(x, w_gate, w_up, w_down):
            return _GatedFFNFn.apply(x, w_gate, w_up, w_down, act)
        i32 = None
    else:
        sizes = dict(gate=(d, F), up=(d, F), down=(F, d))
        adapters = FFNAdapters(*(None if a is None else _adapters(a, *sizes[k], "gated_ffn", f"{k} adapters: ")
                                 for k, a in zip(sizes, adapters)))
        some = [a for a in adapters if a is not None]
        _one_gpu("gated_ffn", x, w_gate, w_up, w_down, ids, *(t for a in some for t in a))
        if len({a.a.shape[0] for a in some}) > 1:
            raise ValueError(f"kmoe.gated_ffn: the projections have as many adapters each, got {[a.a.shape[0] for a in some]}")
        if adapters.gate is not None and adapters.up is not None and len({-(-a.a.shape[1] // 8) for a in adapters[:2]}) > 1:
            raise ValueError(f"kmoe.gated_ffn: the gate's and the up projection's adapters have one rank, got "
                             f"{adapters.gate.a.shape[1]} and {adapters.up.a.shape[1]}")
        i32 = _ids(ids, x, some[0].a.shape[0], "gated_ffn")
        if _wants_grad(x, w_gate, w_up, w_down, *(t for a in some for t in a[:2])):
            g, u = (_adapted(x, w, a, i32) for w, a in ((w_gate, adapters.gate), (w_up, adapters.up)))
            return _adapted((_ACT_FN[activation](g.float()) * u.float()).to(_BF16), w_down, adapters.down, i32).to(x.dtype)
        adapters = FFNAdapters(*(_held(a) for a in adapters))
    y = _ffn_forward(_ready(x), _ready(w_gate), _ready(w_up), _ready(w_down), act, adapters, i32)
    return y if x.dtype is _BF16 else y.to(x.dtype)


# ---------------------------------------------------------------- adapted projections
class _AdaptedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, a, b, scale, ids):
        _bwd.leaves_of(ctx, x, w, a, b)
        xr, bw = _ready(x), _ready(w)
        # (odd ranks are filled up here: a node of torch's for it would be one more of the leaves')
        ad = None if a is None else _held(Adapters(a, b, scale))
        y, ws = _linear_forward(xr, bw, ad, ids)
        ba, bb, kept = (None, None, None) if a is None else (ad.a, ad.b, None)
        if a is not None and ctx.needs_input_grad[3] and ws is not None:
            # the workspace begins with the scaled inner products; partial sums behind them are not kept
            size = 4 * ids.numel() * ba.shape[1]
            kept = ws if ws.numel() < size + 256 else ws[:size].clone()
        ctx.save_for_backward(xr, bw, ba, bb, scale, ids, kept, *_copied((x, xr), (w, bw), (a, ba), (b, bb)))
        ctx.meta = (x.dtype, w.dtype, None if a is None else a.dtype, None if b is None else b.dtype)
        ctx.rank = 0 if a is None else a.shape[1]
        return y if x.dtype is _BF16 else y.to(x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xr, bw, ba, bb, scale, ids, v = ctx.saved_tensors[:7]
        dtypes = ctx.meta
        N, K = bw.shape
        T = xr.numel() // K
        need_x, need_w, need_a, need_b = ctx.needs_input_grad[:4]
        dy2 = _ready(dy)
        dx = dw = da = db = None
        with _device(xr.device), _Stage("bwd_adapted_linear"):
            if ba is not None and (need_x or need_a or need_b):
                n, r = ba.shape[:2]
                dx = torch.empty_like(xr) if need_x else None
                da = torch.empty_like(ba) if need_a else None
                db = torch.empty_like(bb) if need_b else None
                wsb = _linear_backward_workspace(xr.device.index, T, K, N, n, r)
                ws = torch.empty(max(wsb, 16), device=xr.device, dtype=torch.uint8)
                _lib.call("kmoe_adapted_linear_backward", ptr(dy2), ptr(xr), T, K, ptr(bw), N, ptr(ids), n,
                          _struct(Adapters(ba, bb, scale)), ptr(v), ptr(dx), ptr(da), ptr(db), ptr(ws), wsb, _stream(xr))
                if r != ctx.rank:
                    da = None if da is None else da[:, :ctx.rank].contiguous()
                    db = None if db is None else db[..., :ctx.rank].contiguous()
            elif need_x:
                dx = _dense_dx(dy2.view(T, N), bw, T).view(xr.shape)
            if need_w:
                dw = _dense_wgrad(dy2.view(T, N), xr.view(T, K), T, dtypes[1])
        return tuple(g if g is None or g.dtype is t else g.to(t) for g, t in zip((dx, dw, da, db), dtypes)) + (None, None)


def _adapted(x, w, ad, i32):
    """adapted_linear of checked arguments, with gradients."""
    a, b, scale = ad if ad is not None else (None, None, None)
    return _AdaptedFn.apply(x, w, a, b, scale, i32)


def adapted_linear(x, weight, adapters: Optional[Adapters] = None, ids=None):
    """x weight^T for rows x (..., K), weight (N, K) bf16 or f32 (cast to bf16 in the call), plus each
    row's low-rank adapter: row t gets scale[i] (x a[i]^T) b[i]^T, i = ids[t] (ids (...,) int32 or int64;
    -1, or any id that is no adapter: nothing).  K and N multiples of 8.  The result has x's
    type.  Differentiable in x, the weight and the adapters' a and b."""
    _weight(weight, None, None, "adapted_linear", "weight")
    N, K = weight.shape
    _rows(x, K, "adapted_linear")
    i32 = None
    if adapters is not None:
        adapters = _adapters(adapters, K, N, "adapted_linear", "")
        _one_gpu("adapted_linear", x, weight, ids, *adapters)
        i32 = _ids(ids, x, adapters.a.shape[0], "adapted_linear")
    else:
        _one_gpu("adapted_linear", x, weight)
    if _wants_grad(x, weight, *(adapters[:2] if adapters is not None else ())):
        return _adapted(x, weight, adapters, i32)
    y, _ = _linear_forward(_ready(x), _ready(weight), _held(adapters), i32)
    return y if x.dtype is _BF16 else y.to(x.dtype)


# ---------------------------------------------------------------- module
class GatedFFN(nn.Module):
    """The reference's gated block (SwiGLU, moe_arch/model/ffn.py:17-64: w1 gate, w2 up, w3 down, no
    biases) on the HIP kernels, for the layers without experts and for a shared expert."""

    def __init__(self, d_model: int, d_ff: int, activation: str = "silu"):
        super().__init__()
        _act(activation)
        if d_model <= 0 or d_ff <= 0 or d_model % 8 or d_ff % 8:
            raise ValueError(f"kmoe.GatedFFN: d_model={d_model}, d_ff={d_ff}: positive multiples of 8")
        self.d_model, self.d_ff, self.activation = d_model, d_ff, activation
        self.w1 = nn.Linear(d_model, d_ff, bias=False)
        self.w2 = nn.Linear(d_model, d_ff, bias=False)
        self.w3 = nn.Linear(d_ff, d_model, bias=False)
        self._bf16_cache = None

    def forward(self, x: torch.Tensor, adapters: Optional[FFNAdapters] = None, ids=None) -> torch.Tensor:
        ws = (self.w1.weight, self.w2.weight, self.w3.weight)
        if ws[0].dtype != _BF16 and not _wants_grad(x, *ws):
            # f32 weights: their casts are kept until one changes
            ws = derived(self.__dict__, "_bf16_cache", ws, lambda: tuple(w.detach().to(_BF16) for w in ws))
        return gated_ffn(x, *ws, self.activation, adapters, ids)
