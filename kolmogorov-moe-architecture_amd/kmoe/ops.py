"""Tensor-level wrappers over the kmoe C ABI (one function per entry point).

Every wrapper validates shapes/dtypes/devices on the host, allocates its
outputs with torch (the C ABI itself never allocates), and launches on
torch's current HIP stream.  There is no CPU path: inputs must live on a GPU.
"""
from __future__ import annotations

import functools
import math
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import ptr

_BF16 = torch.bfloat16


def _need_gpu(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("kmoe: tensors must be on a GPU (the HIP kernels are the only implementation)")


def _one_gpu(who, first, *ts):
    """All on one GPU, the first one's."""
    _need_gpu(first)
    dev = first.get_device()  # (an index: cheaper than a device, once a tensor and call)
    for t in ts:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"kmoe.{who}: tensors must be on one GPU, got {first.device} and {t.device}")


def _contig(t, dtype=None):
    if t is None:
        return None
    if dtype is not None and t.dtype != dtype:
        t = t.to(dtype)
    return t.contiguous()


def _stream(t):
    return _lib.stream_ptr(t.device)


class _Here:
    """Context of a call on the current device."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _device(dev):
    """Context that makes `dev` the current device (the launch's device, and the one whose CU
    count sizes grids), for nothing where it already is."""
    return _HERE if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


# ---------------------------------------------------------------- stage timing
# When a list is installed here (bench.py does), every stage records a pair of
# HIP events on the launch stream: (name, start, end).  Off by default.
_STAGE_EVENTS: Optional[list] = None


def _Stage(name):
    """Context of one stage: records its events when a recorder is installed."""
    return _NO_STAGE if _STAGE_EVENTS is None else _TimedStage(name)


class _NoStage:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_NO_STAGE = _NoStage()


class _TimedStage:
    def __init__(self, name):
        self.name = name
        self.on = _STAGE_ONLY is None or name in _STAGE_ONLY

    def __enter__(self):
        if self.on:
            self.start = torch.cuda.Event(enable_timing=True)
            self.start.record()
        return self

    def __exit__(self, *exc):
        if self.on:
            end = torch.cuda.Event(enable_timing=True)
            end.record()
            _STAGE_EVENTS.append((self.name, self.start, end))
        return False


_STAGE_ONLY: Optional[set] = None


def set_stage_timing(events: Optional[list], only: Optional[set] = None):
    """Install (a list) or remove (None) the per-stage event recorder; `only`
    restricts it to the named stages."""
    global _STAGE_EVENTS, _STAGE_ONLY
    _STAGE_EVENTS = events
    _STAGE_ONLY = set(only) if only is not None else None


class RouterOut(NamedTuple):
    logits: torch.Tensor          # (T, E) f32
    idx: Optional[torch.Tensor]   # (T, k) int64
    w: Optional[torch.Tensor]     # (T, k) f32
    partials: Optional[torch.Tensor]  # per-block aux partial sums (None: router(partials=False))
    hidden: Optional[torch.Tensor] = None  # (T, 128) f32 pre-activation (training router)
    rscale: Optional[torch.Tensor] = None  # (T,) f32 RMSNorm scale 1/sqrt(mean(x^2)+eps) (rms router)
    block_counts: Optional[torch.Tensor] = None  # (ceil(T/b), E) int32 per-block routed counts, b = router_block_tokens(T)


def router(x2d, w_in, w_out, k, bias=None, row_index=None, T=None, save_hidden=False,
           rms_eps=None, hist=True, partials=True, stage="router") -> RouterOut:
    """logits/top-k of the reference Router (moe.py:423-462) on the HIP kernel.

    x2d: (rows, d) bf16; w_in: (128, d); w_out: (E, 128); row_index: optional
    int32 (T,) selecting the rows of x2d that are the tokens.
    rms_eps: route RMSNorm(x) (embeddings.py:167-195) with the norm weight already
    folded into w_in's columns; the result carries the per-token scale (rscale).
    hist (k > 0, not rms): also return each router block's per-expert routed counts
    (blocks of router_block_tokens(T) tokens), which dispatch(block_counts=...) takes
    instead of counting them again.
    partials: write the per-block aux partial sums (aux_loss's input); False for a router
    that only needs its logits (like the MoD auxiliary router).
    stage: the name the per-stage timing records the launch under.
    """
    _need_gpu(x2d, w_in, w_out)
    x2d = _contig(x2d, _BF16)
    w_in = _contig(w_in, _BF16)
    w_out = _contig(w_out, _BF16)
    d = x2d.shape[1]
    E = w_out.shape[0]
    if w_in.shape != (_lib.ROUTER_HIDDEN, d) or w_out.shape[1] != _lib.ROUTER_HIDDEN:
        raise ValueError(f"kmoe.router: weight shapes {tuple(w_in.shape)}, {tuple(w_out.shape)} "
                         f"do not match d={d}, hidden={_lib.ROUTER_HIDDEN}")
    if T is None:
        T = row_index.shape[0] if row_index is not None else x2d.shape[0]
    dev = x2d.device
    logits = torch.empty(T, E, device=dev, dtype=torch.float32)
    idx = torch.empty(T, k, device=dev, dtype=torch.int64) if k > 0 else None
    w = torch.empty(T, k, device=dev, dtype=torch.float32) if k > 0 else None
    if partials:
        partials = torch.empty(max(_lib.load().kmoe_router_partials_len(T, E), 1), device=dev, dtype=torch.float32)
    else:
        partials = None
    bias = _contig(bias, torch.float32)
    hidden = torch.empty(T, _lib.ROUTER_HIDDEN, device=dev, dtype=torch.float32) if save_hidden else None
    if rms_eps is not None:
        if save_hidden:
            raise ValueError("kmoe.router: rms_eps is a forward-only (inference) path")
        rscale = torch.empty(max(T, 1), device=dev, dtype=torch.float32)
        with _Stage(stage):
            _lib.call("kmoe_router_rms", ptr(x2d), ptr(row_index), T, d, ptr(w_in), ptr(w_out), E, ptr(bias), k,
                      ptr(logits), ptr(idx), ptr(w), ptr(partials), float(rms_eps), ptr(rscale), _stream(x2d))
        return RouterOut(logits, idx, w, partials, None, rscale)
    if hist and k > 0 and T > 0:
        bc = torch.empty(-(-T // router_block_tokens(T)), E, device=dev, dtype=torch.int32)
        with _Stage(stage):
            _lib.call("kmoe_router_hist", ptr(x2d), ptr(row_index), T, d, ptr(w_in), ptr(w_out), E, ptr(bias), k,
                      ptr(logits), ptr(idx), ptr(w), ptr(partials), ptr(hidden), ptr(bc), _stream(x2d))
        return RouterOut(logits, idx, w, partials, hidden, None, bc)
    with _Stage(stage):
        _lib.call("kmoe_router_train", ptr(x2d), ptr(row_index), T, d, ptr(w_in), ptr(w_out), E, ptr(bias), k,
                  ptr(logits), ptr(idx), ptr(w), ptr(partials), ptr(hidden), _stream(x2d))
    return RouterOut(logits, idx, w, partials, hidden)


def router_block_tokens(T: int) -> int:
    """Tokens per router workgroup for a call over T tokens on the current device (32 when
    32-token tiles fit the device in one wave of workgroups, else 64): the token span of
    one row of the router's aux partials and block histograms."""
    return int(_lib.load().kmoe_router_block_tokens(T))


def balanced_topk(logits, k):
    """Capacity-balanced top-k of Router._balanced_topk_assignment (moe.py:353-421)
    from fp32 logits (T, E): returns (idx (T,k) int64, w (T,k) f32)."""
    _need_gpu(logits)
    logits = _contig(logits, torch.float32)
    T, E = logits.shape
    dev = logits.device
    idx = torch.empty(T, k, device=dev, dtype=torch.int64)
    w = torch.empty(T, k, device=dev, dtype=torch.float32)
    lib = _lib.load()
    wsb = lib.kmoe_balanced_workspace_bytes(E, k)
    ws = torch.empty(max(wsb, 4), device=dev, dtype=torch.uint8)
    with _Stage("router"):
        _lib.call("kmoe_balanced_topk", ptr(logits), T, E, k, ptr(idx), ptr(w), ptr(ws), wsb, _stream(logits))
    return idx, w


def aux_loss(partials, T, E, counts, k, w_lb, w_z):
    """(aux, load_balance, z) of MoELayer._compute_auxiliary_losses (moe.py:840-939)."""
    out = torch.empty(3, device=partials.device, dtype=torch.float32)
    with _Stage("aux"):
        _lib.call("kmoe_aux_loss", ptr(partials), T, E, ptr(counts), k, float(w_lb), float(w_z), ptr(out),
              _stream(partials))
    return out


def mod_aux_bce(logits, rows, weight):
    """The MoD auxiliary router's loss (mod.py:141-171) from its logits (T,) or (T, 1)
    f32 and the kept rows (int32): weight * mean BCE-with-logits, targets 1 at rows."""
    _need_gpu(logits, rows)
    logits = _contig(logits, torch.float32)
    rows = _contig(rows, torch.int32)
    out = torch.empty(1, device=logits.device, dtype=torch.float32)
    _lib.call("kmoe_mod_aux_bce", ptr(logits), logits.numel(), ptr(rows), rows.numel(), float(weight), ptr(out),
              _stream(logits))
    return out[0]


class DispatchOut(NamedTuple):
    counts: torch.Tensor     # (E,) int32 routed counts
    offsets: torch.Tensor    # (E+1,) int32 kept-row offsets
    row_token: torch.Tensor  # (T*k,) int32
    slot_row: torch.Tensor   # (T*k,) int32, -1 = dropped
    slot_w: torch.Tensor     # (T*k,) f32
    xperm: torch.Tensor      # (T*k, d) bf16 or uint8 (fp8 e4m3)
    xscale: Optional[torch.Tensor]  # (T*k,) f32 for fp8
    aux: Optional[torch.Tensor] = None  # (3,) f32 aux losses, when asked for (aux_loss's output)


def capacity_of(cf: float, T: int, k: int, E: int) -> int:
    """Per-expert capacity ceil(cf*T*k/E) of the token-choice drop rule."""
    return int(math.ceil(cf * T * k / E))


def dispatch(x2d, idx, w, E, capacity=0, fp8=False, row_index=None, materialize=True,
             no_alloc=False, block_counts=None, aux=None) -> DispatchOut:
    """Stable counting-sort dispatch (moe.py:238-272) + optional capacity drop.

    materialize=False (bf16 only) writes the routing tables but not the permuted
    rows: gemm_gate_up_rows gathers them itself (xperm is then None).
    no_alloc=True calls kmoe_dispatch_noalloc, whose histograms live in the library's
    own device scratch (no workspace allocation; calls on one GPU must not overlap).
    block_counts: the router's per-block histograms of idx (RouterOut.block_counts);
    kmoe_dispatch_counted then skips counting them.
    aux = (partials, w_lb, w_z) (with block_counts): the aux losses of aux_loss(partials, T,
    E, counts, k, w_lb, w_z) come back in DispatchOut.aux, computed inside the dispatch's
    table launch (kmoe_dispatch_counted_aux) instead of a launch of their own."""
    if not materialize and fp8:
        raise ValueError("kmoe.dispatch: the fp8 path needs the quantised permuted rows (materialize=True)")
    _need_gpu(x2d, idx, w)
    x2d = _contig(x2d, _BF16)
    idx = _contig(idx, torch.int64)
    if w.dtype not in (torch.float32, _BF16):
        w = w.float()
    w = w.contiguous()
    T, k = idx.shape
    d = x2d.shape[1]
    A = T * k
    dev = x2d.device
    lib = _lib.load()
    counts = torch.empty(E, device=dev, dtype=torch.int32)
    offsets = torch.empty(E + 1, device=dev, dtype=torch.int32)
    row_token = torch.empty(max(A, 1), device=dev, dtype=torch.int32)
    slot_row = torch.empty(max(A, 1), device=dev, dtype=torch.int32)
    slot_w = torch.empty(max(A, 1), device=dev, dtype=torch.float32)
    xperm = torch.empty(max(A, 1), d, device=dev, dtype=torch.uint8 if fp8 else _BF16) if materialize else None
    xscale = torch.empty(max(A, 1), device=dev, dtype=torch.float32) if fp8 else None
    wdt = _lib.DTYPE_F32 if w.dtype == torch.float32 else _lib.DTYPE_BF16
    if no_alloc:
        with _Stage("dispatch"):
            _lib.call("kmoe_dispatch_noalloc", ptr(x2d), ptr(row_index), T, d, ptr(idx), ptr(w), wdt, k, E,
                      int(capacity), ptr(counts), ptr(offsets), ptr(row_token), ptr(slot_row), ptr(slot_w), ptr(xperm),
                      _lib.DTYPE_FP8_E4M3 if fp8 else _lib.DTYPE_BF16, ptr(xscale), _stream(x2d))
        return DispatchOut(counts, offsets, row_token, slot_row, slot_w, xperm, xscale)
    wsb = lib.kmoe_dispatch_workspace_bytes(T, k, E)
    ws = torch.empty(wsb, device=dev, dtype=torch.uint8)
    if aux is not None and (block_counts is None or no_alloc or T == 0):
        raise ValueError("kmoe.dispatch: aux needs block_counts (and T > 0, not no_alloc)")
    if block_counts is not None:
        hb = router_block_tokens(T)
        if block_counts.dtype != torch.int32 or block_counts.numel() != -(-T // hb) * E:
            raise ValueError(f"kmoe.dispatch: block_counts must be int32 (ceil(T/{hb}), E) "
                             f"(router_block_tokens)")
        if aux is not None:
            partials, w_lb, w_z = aux
            aux_out = torch.empty(3, device=dev, dtype=torch.float32)
            with _Stage("dispatch"):
                _lib.call("kmoe_dispatch_counted_aux", ptr(x2d), ptr(row_index), T, d, ptr(idx), ptr(w), wdt, k, E,
                          int(capacity), ptr(block_counts), ptr(counts), ptr(offsets), ptr(row_token), ptr(slot_row),
                          ptr(slot_w), ptr(xperm), _lib.DTYPE_FP8_E4M3 if fp8 else _lib.DTYPE_BF16, ptr(xscale),
                          ptr(ws), wsb, ptr(partials), float(w_lb), float(w_z), ptr(aux_out), _stream(x2d))
            return DispatchOut(counts, offsets, row_token, slot_row, slot_w, xperm, xscale, aux_out)
        with _Stage("dispatch"):
            _lib.call("kmoe_dispatch_counted", ptr(x2d), ptr(row_index), T, d, ptr(idx), ptr(w), wdt, k, E,
                      int(capacity), ptr(block_counts), ptr(counts), ptr(offsets), ptr(row_token), ptr(slot_row),
                      ptr(slot_w), ptr(xperm), _lib.DTYPE_FP8_E4M3 if fp8 else _lib.DTYPE_BF16, ptr(xscale),
                      ptr(ws), wsb, _stream(x2d))
        return DispatchOut(counts, offsets, row_token, slot_row, slot_w, xperm, xscale)
    with _Stage("dispatch"):
        _lib.call("kmoe_dispatch", ptr(x2d), ptr(row_index), T, d, ptr(idx), ptr(w), wdt, k, E, int(capacity),
              ptr(counts), ptr(offsets), ptr(row_token), ptr(slot_row), ptr(slot_w), ptr(xperm),
              _lib.DTYPE_FP8_E4M3 if fp8 else _lib.DTYPE_BF16, ptr(xscale), ptr(ws), wsb, _stream(x2d))
    return DispatchOut(counts, offsets, row_token, slot_row, slot_w, xperm, xscale)


def gather_rows(x2d, row_token, n_rows, fp8=False, n_rows_dev=None):
    _need_gpu(x2d, row_token)
    x2d = _contig(x2d, _BF16)
    d = x2d.shape[1]
    out = torch.empty(max(n_rows, 1), d, device=x2d.device, dtype=torch.uint8 if fp8 else _BF16)
    scale = torch.empty(max(n_rows, 1), device=x2d.device, dtype=torch.float32) if fp8 else None
    with _Stage("gather"):
        _lib.call("kmoe_gather_rows", ptr(x2d), ptr(row_token), n_rows, ptr(n_rows_dev), d, ptr(out),
              _lib.DTYPE_FP8_E4M3 if fp8 else _lib.DTYPE_BF16, ptr(scale), _stream(x2d))
    return out, scale


class PackedWeights(NamedTuple):
    w13: torch.Tensor
    w3: torch.Tensor
    s13: Optional[torch.Tensor]
    s3: Optional[torch.Tensor]
    E: int
    d: int
    F: int
    fp8: bool


def pack_weights(w1, w2, w3, fp8=False) -> PackedWeights:
    """Derived kernel layout of the reference expert weights w1,w2 (E,d,F), w3 (E,F,d)."""
    _need_gpu(w1, w2, w3)
    E, d, F = w1.shape
    if w2.shape != (E, d, F) or w3.shape != (E, F, d):
        raise ValueError("kmoe.pack_weights: w1/w2 must be (E,d,F) and w3 (E,F,d)")
    if w1.dtype not in (torch.float32, _BF16):
        raise ValueError(f"kmoe.pack_weights: unsupported weight dtype {w1.dtype}")
    dt = w1.dtype
    w1, w2, w3 = _contig(w1, dt), _contig(w2, dt), _contig(w3, dt)
    lib = _lib.load()
    pdt = _lib.DTYPE_FP8_E4M3 if fp8 else _lib.DTYPE_BF16
    wdt = _lib.DTYPE_F32 if dt == torch.float32 else _lib.DTYPE_BF16
    Fp = lib.kmoe_padded_ff(F)
    dp = (d + 255) // 256 * 256
    dev = w1.device
    w13p = torch.empty(lib.kmoe_packed_w13_bytes(E, d, F, pdt), device=dev, dtype=torch.uint8)
    w3p = torch.empty(lib.kmoe_packed_w3_bytes(E, d, F, pdt), device=dev, dtype=torch.uint8)
    s13 = torch.empty(E * 2 * Fp, device=dev, dtype=torch.float32) if fp8 else None
    s3 = torch.empty(E * dp, device=dev, dtype=torch.float32) if fp8 else None
    _lib.call("kmoe_pack_weights", ptr(w1), ptr(w2), ptr(w3), wdt, E, d, F, pdt, ptr(w13p), ptr(s13), ptr(w3p),
              ptr(s3), _stream(w1))
    return PackedWeights(w13p, w3p, s13, s3, E, d, F, fp8)


def gemm_gate_up(xperm, xscale, offsets, pw: PackedWeights, max_rows, save_gu=False):
    """h = SwiGLU gate/up of the permuted rows.  save_gu (fp8 training forward) also
    returns the descaled pre-activation gate/up values (max_rows, 2*F_pad) bf16 in the
    packed order: returns (h, gu)."""
    lib = _lib.load()
    Fp = lib.kmoe_padded_ff(pw.F)
    h = torch.empty(max(max_rows, 1), Fp, device=xperm.device, dtype=_BF16)
    if save_gu:
        if not pw.fp8:
            raise ValueError("kmoe.gemm_gate_up: save_gu is for fp8 rows (bf16: gemm_gate_up_rows)")
        gu = torch.empty(max(max_rows, 1), 2 * Fp, device=xperm.device, dtype=_BF16)
        with _Stage("gemm_gate_up"):
            _lib.call("kmoe_gemm_gate_up_fp8_gu", ptr(xperm), ptr(xscale), ptr(offsets), pw.E, pw.d, pw.F, max_rows,
                      ptr(pw.w13), ptr(pw.s13), ptr(h), ptr(gu), _stream(xperm))
        return h, gu
    with _Stage("gemm_gate_up"):
        _lib.call("kmoe_gemm_gate_up", ptr(xperm), ptr(xscale),
              _lib.DTYPE_FP8_E4M3 if pw.fp8 else _lib.DTYPE_BF16, ptr(offsets), pw.E, pw.d, pw.F, max_rows,
              ptr(pw.w13), ptr(pw.s13), ptr(h), _stream(xperm))
    return h


def gemm_gate_up_rows(x2d, row_index, row_token, offsets, pw: PackedWeights, max_rows, save_gu=False,
                      rscale=None):
    """gate_up GEMM whose A rows are x2d[row_index[row_token[r]]] (x2d[row_token[r]]
    without row_index): the dispatch gather fused into the GEMM's loads (bf16).
    save_gu (training) also returns the pre-activation gate/up values (max_rows,
    2*F_pad) in the packed order: returns (h, gu).
    rscale (T,) f32: row r's gate/up values are scaled by rscale[row_token[r]] (the
    RMSNorm scale; pw packed from norm-folded w1/w2)."""
    if pw.fp8:
        raise ValueError("kmoe.gemm_gate_up_rows: bf16 weights only (fp8 reads quantised permuted rows)")
    _need_gpu(x2d, row_token, offsets)
    x2d = _contig(x2d, _BF16)
    lib = _lib.load()
    Fp = lib.kmoe_padded_ff(pw.F)
    h = torch.empty(max(max_rows, 1), Fp, device=x2d.device, dtype=_BF16)
    if rscale is not None:
        if save_gu:
            raise ValueError("kmoe.gemm_gate_up_rows: rscale is a forward-only (inference) path")
        with _Stage("gemm_gate_up"):
            _lib.call("kmoe_gemm_gate_up_rows_scaled", ptr(x2d), ptr(row_index), x2d.shape[0], ptr(row_token),
                      ptr(offsets), pw.E, pw.d, pw.F, max_rows, ptr(pw.w13), ptr(rscale), ptr(h), _stream(x2d))
        return h
    if save_gu:
        gu = torch.empty(max(max_rows, 1), 2 * Fp, device=x2d.device, dtype=_BF16)
        with _Stage("gemm_gate_up"):
            _lib.call("kmoe_gemm_gate_up_rows_gu", ptr(x2d), ptr(row_index), x2d.shape[0], ptr(row_token),
                      ptr(offsets), pw.E, pw.d, pw.F, max_rows, ptr(pw.w13), ptr(h), ptr(gu), _stream(x2d))
        return h, gu
    with _Stage("gemm_gate_up"):
        _lib.call("kmoe_gemm_gate_up_rows", ptr(x2d), ptr(row_index), x2d.shape[0], ptr(row_token), ptr(offsets),
                  pw.E, pw.d, pw.F, max_rows, ptr(pw.w13), ptr(h), _stream(x2d))
    return h


def gemm_down(h, hscale, offsets, pw: PackedWeights, max_rows):
    y = torch.empty(max(max_rows, 1), pw.d, device=h.device, dtype=_BF16)
    with _Stage("gemm_down"):
        _lib.call("kmoe_gemm_down", ptr(h), ptr(hscale), _lib.DTYPE_FP8_E4M3 if pw.fp8 else _lib.DTYPE_BF16,
              ptr(offsets), pw.E, pw.d, pw.F, max_rows, ptr(pw.w3), ptr(pw.s3), ptr(y), _stream(h))
    return y


def quant_rows_fp8(m, n_rows_dev=None):
    rows, cols = m.shape
    q = torch.empty(rows, cols, device=m.device, dtype=torch.uint8)
    s = torch.empty(rows, device=m.device, dtype=torch.float32)
    with _Stage("quant_h"):
        _lib.call("kmoe_quant_rows_fp8", ptr(m), rows, ptr(n_rows_dev), cols, ptr(q), ptr(s), _stream(m))
    return q, s


def dequant_rows_fp8(q, scale, n_rows_dev=None):
    """bf16(e4m3(q) * scale[:, None]) of fp8 rows (rows past *n_rows_dev not written):
    the operand the fp8 GEMM took, for the straight-through backward."""
    _need_gpu(q, scale)
    rows, cols = q.shape
    out = torch.empty(rows, cols, device=q.device, dtype=_BF16)
    with _Stage("fp8_dequant"):
        _lib.call("kmoe_dequant_rows_fp8", ptr(q), ptr(scale), rows, ptr(n_rows_dev), cols, ptr(out), _stream(q))
    return out


def fake_quant_cols_e4m3(w):
    """w (E, K, N) fake-quantised per output column of each expert exactly as the fp8
    weight packing quantises it, dequantised to bf16 (the weights the fp8 GEMMs
    multiplied)."""
    _need_gpu(w)
    if w.dtype not in (torch.float32, _BF16):
        raise ValueError(f"kmoe.fake_quant_cols_e4m3: unsupported weight dtype {w.dtype}")
    w = _contig(w.detach(), w.dtype)
    E, K, N = w.shape
    out = torch.empty(E, K, N, device=w.device, dtype=_BF16)
    _lib.call("kmoe_fake_quant_e4m3_cols", ptr(w), _lib.DTYPE_F32 if w.dtype == torch.float32 else _lib.DTYPE_BF16,
              E, K, N, ptr(out), _stream(w))
    return out


class PlainPacked(NamedTuple):
    """Packed weights of non-gated experts (silu(x w1) w2): w1t (rows f of w1^T), w2t (rows n of w2^T)."""
    w1t: torch.Tensor
    w2t: torch.Tensor
    E: int
    d: int
    F: int
    fp8: bool = False


def pack_weights_plain(w1, w2) -> PlainPacked:
    """Derived kernel layout of non-gated expert weights w1 (E,d,F), w2 (E,F,d) (moe.py:187-191)."""
    _need_gpu(w1, w2)
    E, d, F = w1.shape
    if w2.shape != (E, F, d):
        raise ValueError("kmoe.pack_weights_plain: w1 must be (E,d,F) and w2 (E,F,d)")
    if w1.dtype not in (torch.float32, _BF16):
        raise ValueError(f"kmoe.pack_weights_plain: unsupported weight dtype {w1.dtype}")
    dt = w1.dtype
    w1, w2 = _contig(w1, dt), _contig(w2, dt)
    lib = _lib.load()
    dev = w1.device
    w1t = torch.empty(lib.kmoe_packed_w1t_bytes(E, d, F), device=dev, dtype=torch.uint8)
    w2t = torch.empty(lib.kmoe_packed_w3_bytes(E, d, F, _lib.DTYPE_BF16), device=dev, dtype=torch.uint8)
    _lib.call("kmoe_pack_weights_plain", ptr(w1), ptr(w2), _lib.DTYPE_F32 if dt == torch.float32 else _lib.DTYPE_BF16,
              E, d, F, ptr(w1t), ptr(w2t), _stream(w1))
    return PlainPacked(w1t, w2t, E, d, F)


def plain_ffn(xperm, offsets, pp: PlainPacked, max_rows):
    """Non-gated experts on the permuted rows (moe.py:281-283): p = x w1, h = silu(p),
    y = h w2.  Returns (yperm (max_rows, d), h, p) bf16."""
    E, d, F = pp.E, pp.d, pp.F
    lib = _lib.load()
    Fp = lib.kmoe_padded_ff(F)
    dev = xperm.device
    s = _stream(xperm)
    rows = max(max_rows, 1)
    p = torch.empty(rows, Fp, device=dev, dtype=_BF16)
    h = torch.empty(rows, Fp, device=dev, dtype=_BF16)
    y = torch.empty(rows, d, device=dev, dtype=_BF16)
    with _Stage("gemm_gate_up"):
        _lib.call("kmoe_gemm_grouped", ptr(xperm), ptr(offsets), E, d, max_rows, ptr(pp.w1t), (F + 255) // 256 * 256,
                  Fp, ptr(p), Fp, Fp, s)
    with _Stage("silu"):
        _lib.call("kmoe_silu_rows", ptr(p), max_rows, ptr(offsets[E:]), F, ptr(h), s)
    with _Stage("gemm_down"):
        _lib.call("kmoe_gemm_grouped", ptr(h), ptr(offsets), E, Fp, max_rows, ptr(pp.w2t), (d + 255) // 256 * 256, d,
                  ptr(y), d, d, s)
    return y, h, p


def grouped_ffn(xperm, xscale, offsets, pw: PackedWeights, max_rows):
    """gate_up -> (fp8: per-row requant of h) -> down.  Returns yperm (max_rows, d) bf16."""
    if isinstance(pw, PlainPacked):
        return plain_ffn(xperm, offsets, pw, max_rows)[0]
    h = gemm_gate_up(xperm, xscale, offsets, pw, max_rows)
    if pw.fp8:
        hq, hs = quant_rows_fp8(h, offsets[pw.E:])
        return gemm_down(hq, hs, offsets, pw, max_rows)
    return gemm_down(h, None, offsets, pw, max_rows)


def combine(yperm, src_row, src_w, T_out, out_map=None, scale=None, out_dtype=_BF16, residual=None,
            keep_mask=None, keep_scale=1.0):
    """y[o] = scale[s] * sum_j src_w[s,j] * yperm[src_row[s,j]] (moe.py:285-292, 132-158),
    plus residual[o] ((T_out, d), cast to out_dtype) when given (layers.py:187).
    keep_mask ((T_out, d) bool, with a residual): the residual dropout, the sum times
    keep_scale = 1/(1-p) where kept and 0 elsewhere (layers.py:190)."""
    fan = src_row.shape[1]
    d = yperm.shape[1]
    y = torch.empty(T_out, d, device=yperm.device, dtype=out_dtype)
    ydt = _lib.DTYPE_F32 if out_dtype == torch.float32 else _lib.DTYPE_BF16
    if residual is not None:
        residual = _contig(residual, out_dtype)
        if residual.shape != (T_out, d):
            raise ValueError(f"kmoe.combine: residual shape {tuple(residual.shape)} != {(T_out, d)}")
    if keep_mask is not None:
        if residual is None:
            raise ValueError("kmoe.combine: a dropout keep mask needs the residual")
        if keep_mask.shape != (T_out, d) or keep_mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"kmoe.combine: keep_mask must be bool/uint8 {(T_out, d)}, got "
                             f"{keep_mask.dtype} {tuple(keep_mask.shape)}")
        keep_mask = keep_mask.contiguous()
        with _Stage("combine"):
            _lib.call("kmoe_combine_residual_dropout", ptr(yperm), d, ptr(src_row), ptr(src_w), fan, ptr(out_map),
                      ptr(scale), ptr(residual), ptr(keep_mask), float(keep_scale), T_out, ptr(y), ydt,
                      _stream(yperm))
        return y
    with _Stage("combine"):
        _lib.call("kmoe_combine_residual", ptr(yperm), d, ptr(src_row), ptr(src_w), fan, ptr(out_map), ptr(scale),
                  ptr(residual), T_out, ptr(y), ydt, _stream(yperm))
    return y


def stage_timing() -> bool:
    """Whether a per-stage event recorder is installed."""
    return _STAGE_EVENTS is not None


def moe_forward(x2d, w_in, w_out, k, bias, pw: PackedWeights, capacity, out_dtype, residual=None, rms_eps=None,
                aux=None):
    """The token-choice layer forward without gradients in one native call (bf16 gated
    experts): (y (T, d), counts (E,) int32, aux (3,) f32 or None), the results of router,
    dispatch, the two expert products and combine.
    rms_eps: of RMSNorm(x), the norm weight folded into w_in and pw.  aux = (w_lb, w_z): also the
    aux losses of aux_loss().  residual (T, d): added in the combine."""
    _need_gpu(x2d, w_in, w_out)
    x2d = _contig(x2d, _BF16)
    w_in = _contig(w_in, _BF16)
    w_out = _contig(w_out, _BF16)
    T, d = x2d.shape
    E = w_out.shape[0]
    if w_in.shape != (_lib.ROUTER_HIDDEN, d) or w_out.shape[1] != _lib.ROUTER_HIDDEN:
        raise ValueError(f"kmoe.router: weight shapes {tuple(w_in.shape)}, {tuple(w_out.shape)} "
                         f"do not match d={d}, hidden={_lib.ROUTER_HIDDEN}")
    if (pw.E, pw.d) != (E, d) or pw.fp8:
        raise ValueError(f"kmoe.moe_forward: packed weights of {pw.E} experts, d={pw.d} (fp8={pw.fp8}) for a router "
                         f"of {E} experts, d={d}")
    if rms_eps is not None and not rms_eps >= 0.0:  # negative means "no norm" to the native call
        raise _lib.KmoeError("kmoe_moe_forward", _lib.KMOE_ERR_SHAPE, f"rms_eps {rms_eps} must be >= 0")
    dev = x2d.device
    bias = _contig(bias, torch.float32)
    y = torch.empty(T, d, device=dev, dtype=out_dtype)
    if residual is not None:
        residual = _contig(residual, out_dtype)
        if residual.shape != (T, d):
            raise ValueError(f"kmoe.combine: residual shape {tuple(residual.shape)} != {(T, d)}")
    counts = torch.empty(E, device=dev, dtype=torch.int32)
    aux_out = None
    w_lb = w_z = 0.0
    if aux is not None:
        w_lb, w_z = aux
        aux_out = torch.empty(3, device=dev, dtype=torch.float32)
    wsb = (_lib._LIB or _lib.load()).kmoe_moe_forward_workspace_bytes(T, d, E, k, pw.F)
    ws = torch.empty(wsb, device=dev, dtype=torch.uint8)
    _lib.call("kmoe_moe_forward", ptr(x2d), T, d, ptr(w_in), ptr(w_out), E, ptr(bias), k, ptr(pw.w13), ptr(pw.w3), pw.F,
              int(capacity), -1.0 if rms_eps is None else float(rms_eps), ptr(residual), ptr(y),
              _lib.DTYPE_F32 if out_dtype == torch.float32 else _lib.DTYPE_BF16, ptr(counts), ptr(aux_out), float(w_lb),
              float(w_z), ptr(ws), wsb, _stream(x2d))
    return y, counts, aux_out


class ECSelectOut(NamedTuple):
    idx: torch.Tensor        # (B,E,C) int64
    w: torch.Tensor          # (B,E,C) f32
    row_token: torch.Tensor  # (E*B*C,) int32
    offsets: torch.Tensor    # (E+1,) int32
    src_row: torch.Tensor    # (B*S, E) int32
    src_w: torch.Tensor      # (B*S, E) f32


def ec_select(logits, B, S, E, C, descending=True) -> ECSelectOut:
    """Expert-choice top-C per (sequence, expert) (moe.py:494-530).

    descending=True gives the reference's topk order; False the same selection in
    ascending token order (no sort: enough for a layer forward)."""
    _need_gpu(logits)
    logits = _contig(logits, torch.float32)
    dev = logits.device
    idx = torch.empty(B, E, C, device=dev, dtype=torch.int64)
    w = torch.empty(B, E, C, device=dev, dtype=torch.float32)
    row_token = torch.empty(E * B * C, device=dev, dtype=torch.int32)
    offsets = torch.empty(E + 1, device=dev, dtype=torch.int32)
    src_row = torch.empty(B * S, E, device=dev, dtype=torch.int32)
    src_w = torch.empty(B * S, E, device=dev, dtype=torch.float32)
    ws_bytes = _lib.load().kmoe_ec_workspace_bytes(B, S, E)
    ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)  # the logits transposed per expert
    with _Stage("ec_select"):
        _lib.call("kmoe_ec_select", ptr(logits), B, S, E, C, 1 if descending else 0, ptr(idx), ptr(w),
                  ptr(row_token), ptr(offsets), ptr(src_row), ptr(src_w), ptr(ws), ws_bytes, _stream(logits))
    return ECSelectOut(idx, w, row_token, offsets, src_row, src_w)


def ec_dlogits(logits, B, S, E, src_row, src_w, dw, dl):
    """Adds the expert-choice selection's logit gradient (kmoe_ec_dlogits) to dl (B*S, E)."""
    _need_gpu(logits, src_row, src_w, dw, dl)
    with _Stage("bwd_router"):
        _lib.call("kmoe_ec_dlogits", ptr(_contig(logits, torch.float32)), B, S, E, ptr(src_row), ptr(src_w),
                  ptr(_contig(dw, torch.float32)), ptr(dl), _stream(logits))
    return dl


class ModSelectOut(NamedTuple):
    logits: torch.Tensor      # (B,S) f32
    sel_idx: torch.Tensor     # (B,keep) int64 ascending
    sel_w: torch.Tensor       # (B,keep) f32 softmax over kept
    token_rows: torch.Tensor  # (B*keep,) int32
    out_map: torch.Tensor     # (B*S,) int32


def mod_select(x3d, w_mod, keep, logits=None) -> ModSelectOut:
    """Mixture-of-Depths top-keep per sequence (mod.py:67-122).  With `logits` ((B, S)
    f32, e.g. rmsnorm's mod_logits) the selection runs on them and x3d is not read."""
    _need_gpu(x3d, w_mod)
    B, S, d = x3d.shape
    dev = x3d.device
    stream = _stream(x3d)
    if logits is not None:
        logits = _contig(logits, torch.float32).view(B, S)
        x3d = w_mod = None
    else:
        x3d = _contig(x3d, _BF16)
        w_mod = _contig(w_mod, _BF16).reshape(-1)
        logits = torch.empty(B, S, device=dev, dtype=torch.float32)
    sel_idx = torch.empty(B, keep, device=dev, dtype=torch.int64)
    sel_w = torch.empty(B, keep, device=dev, dtype=torch.float32)
    token_rows = torch.empty(B * keep, device=dev, dtype=torch.int32)
    out_map = torch.empty(B * S, device=dev, dtype=torch.int32)
    with _Stage("mod_select"):
        _lib.call("kmoe_mod_select", ptr(x3d), B, S, d, ptr(w_mod), keep, ptr(logits), ptr(sel_idx), ptr(sel_w),
              ptr(token_rows), ptr(out_map), None, 0, stream)
    return ModSelectOut(logits, sel_idx, sel_w, token_rows, out_map)


def _fdt(t):
    if t.dtype == torch.float32:
        return _lib.DTYPE_F32
    if t.dtype == _BF16:
        return _lib.DTYPE_BF16
    raise ValueError(f"kmoe: unsupported dtype {t.dtype}")


class NormOut(NamedTuple):
    n: torch.Tensor                       # (T, d) bf16 normalised rows
    rrms: torch.Tensor                    # (T,) f32 1/sqrt(mean(x^2) + eps)
    mod_logits: Optional[torch.Tensor]    # (T,) f32 n . w_mod (with w_mod)


def rmsnorm(x2d, weight, eps, w_mod=None) -> NormOut:
    """RMSNorm (embeddings.py:167-195) of the rows of x2d (bf16 or f32) with weight (d,);
    with w_mod (d,) also the MoD router logits of the normalised rows (mod.py:93)."""
    _need_gpu(x2d, weight)
    if x2d.dtype not in (torch.float32, _BF16):
        x2d = x2d.float()
    x2d = x2d.contiguous()
    weight = weight.detach()
    if weight.dtype not in (torch.float32, _BF16):
        weight = weight.float()
    weight = weight.contiguous()
    T, d = x2d.shape
    n = torch.empty(T, d, device=x2d.device, dtype=_BF16)
    rrms = torch.empty(T, device=x2d.device, dtype=torch.float32)
    ml = None
    if w_mod is not None:
        w_mod = _contig(w_mod.detach(), _BF16).reshape(-1)
        ml = torch.empty(T, device=x2d.device, dtype=torch.float32)
    with _Stage("rmsnorm"):
        _lib.call("kmoe_rmsnorm", ptr(x2d), _fdt(x2d), ptr(weight), _fdt(weight), float(eps), T, d, ptr(n), ptr(rrms),
                  ptr(w_mod), ptr(ml), _stream(x2d))
    return NormOut(n, rrms, ml)


def rmsnorm_bwd(dn, x2d, weight, rrms, dres=None, dw_dtype=None):
    """Backward of rmsnorm: (dx in x2d's dtype (+ dres), dweight (d,))."""
    T, d = x2d.shape
    dn = _contig(dn, _BF16)
    weight = weight.detach().contiguous()
    if dres is not None:
        dres = _contig(dres, x2d.dtype)
    dw_dtype = weight.dtype if dw_dtype is None else dw_dtype
    dx = torch.empty(T, d, device=x2d.device, dtype=x2d.dtype)
    dwt = torch.empty(d, device=x2d.device, dtype=dw_dtype)
    lib = _lib.load()
    wsb = lib.kmoe_rmsnorm_bwd_workspace_bytes(T, d)
    ws = torch.empty(max(wsb, 4), device=x2d.device, dtype=torch.uint8)
    with _Stage("bwd_rmsnorm"):
        _lib.call("kmoe_rmsnorm_bwd", ptr(dn), ptr(x2d), _fdt(x2d), ptr(weight), _fdt(weight), ptr(rrms), ptr(dres), T,
                  d, ptr(dx), ptr(dwt), _fdt(dwt), ptr(ws), wsb, _stream(x2d))
    return dx, dwt

# ---------------------------------------------------------------- routing of logits
class RouteSpec(NamedTuple):
    """How logits become experts and weights (kmoe_route_topk): `scores` "softmax" or
    "sigmoid"; `groups` equal runs of experts of which the best `topk_groups` stay, a group
    being worth the sum of its best `group_top` (1 or 2) choices; `renorm` divides the
    weights by their sum; `scale` multiplies them."""
    scores: str = "softmax"
    groups: int = 1
    topk_groups: int = 1
    group_top: int = 2
    renorm: bool = True
    scale: float = 1.0


class RouteOut(NamedTuple):
    idx: torch.Tensor                        # (T, k) int64
    w: torch.Tensor                          # (T, k) f32
    block_counts: Optional[torch.Tensor] = None  # router-block histograms of idx (hist=True)


def _scores(name) -> int:
    try:
        return _lib.SCORES[name]
    except (KeyError, TypeError):
        raise ValueError(f"kmoe.route_topk: scores {name!r} is none of {sorted(_lib.SCORES)}") from None


def _route_logits(logits, who):
    _need_gpu(logits)
    if logits.dim() != 2:
        raise ValueError(f"kmoe.{who}: logits must be (tokens, experts), got {tuple(logits.shape)}")
    return _contig(logits, torch.float32)


def route_topk(logits, k, scores="softmax", bias=None, groups=1, topk_groups=1, group_top=2, renorm=True, scale=1.0,
               hist=False) -> RouteOut:
    """Experts and weights of logits (T, E): the k largest scores + bias (E,) among the
    experts of the best topk_groups of `groups` groups, and those experts' scores (without
    the bias), renormalised and times `scale`.  A logit of -inf masks its expert: it is
    picked only when too few others are left, with weight 0.  Equal choices: lowest index
    first; choices are compared in 64 bits.  hist: also the histograms that
    dispatch(block_counts=...) takes.  Not differentiable: kmoe.route_topk is."""
    sc = _scores(scores)
    logits = _route_logits(logits, "route_topk")
    T, E = logits.shape
    if bias is not None:
        if bias.shape != (E,) or bias.device != logits.device:
            raise ValueError(f"kmoe.route_topk: bias must be ({E},) on {logits.device}, got {tuple(bias.shape)} on "
                             f"{bias.device}")
        bias = _contig(bias.detach(), torch.float32)
    dev = logits.device
    idx = torch.empty(T, int(k), device=dev, dtype=torch.int64)
    w = torch.empty(T, int(k), device=dev, dtype=torch.float32)
    with _device(dev), _Stage("route"):
        bc = torch.empty(-(-T // router_block_tokens(T)), E, device=dev, dtype=torch.int32) if hist and T > 0 else None
        _lib.call("kmoe_route_topk", ptr(logits), T, E, int(k), sc, ptr(bias), int(groups), int(topk_groups),
                  int(group_top), int(bool(renorm)), float(scale), ptr(idx), ptr(w), ptr(bc), _stream(logits))
    return RouteOut(idx, w, bc)


def route_topk_bwd(logits, idx, dw, scores="softmax", renorm=True, scale=1.0, dlogits=None):
    """Gradient of route_topk's weights: dw (T, k) to the logits' (T, E) f32, added to
    `dlogits` when given.  idx: route_topk's, so a token's experts are distinct."""
    sc = _scores(scores)
    logits = _route_logits(logits, "route_topk_bwd")
    T, E = logits.shape
    _one_gpu("route_topk_bwd", logits, idx, dw, dlogits)
    k = idx.shape[-1]
    if idx.shape != (T, k) or dw.shape != (T, k):
        raise ValueError(f"kmoe.route_topk_bwd: idx and dw must be ({T}, k), got {tuple(idx.shape)}, {tuple(dw.shape)}")
    add = dlogits is not None
    if add and (dlogits.shape != (T, E) or dlogits.dtype != torch.float32 or not dlogits.is_contiguous()):
        raise ValueError(f"kmoe.route_topk_bwd: dlogits must be contiguous f32 ({T}, {E})")
    if not add:
        dlogits = torch.empty(T, E, device=logits.device, dtype=torch.float32)
    with _device(logits.device), _Stage("bwd_router"):
        _lib.call("kmoe_route_topk_bwd", ptr(logits), ptr(_contig(idx, torch.int64)), ptr(_contig(dw, torch.float32)), T, E,
                  k, sc, int(bool(renorm)), float(scale), int(add), ptr(dlogits), _stream(logits))
    return dlogits


# ---------------------------------------------------------------- microscaled rows and experts
MX_FORMATS = {"e4m3": _lib.DTYPE_FP8_E4M3, "e2m1": _lib.DTYPE_FP4_E2M1}
# activation format of each kind of 4-bit experts
MX_EXPERTS = {"w4a8": "e4m3", "w4a4": "e2m1"}


def _mx_fmt(fmt) -> int:
    try:
        return MX_FORMATS[fmt]
    except (KeyError, TypeError):
        raise ValueError(f"kmoe: microscaled element type {fmt!r} is none of {sorted(MX_FORMATS)}") from None


class MXRows(NamedTuple):
    """Rows in blocks of 32 values that share a power-of-two scale.  q (rows, Kp) e4m3 codes
    or (rows, Kp / 2) e2m1 pairs, the first in the low half, Kp = K rounded up to 128;
    scale (rows, K rounded up to 512, / 32), byte c for 2^(c - 127), 255 for a block of NaN; bytes
    past Kp / 32 are not used."""
    q: torch.Tensor
    scale: torch.Tensor
    K: int
    fmt: str


def _mx_rows(rows, K, fmt, dev) -> MXRows:
    kp = (K + 127) // 128 * 128
    return MXRows(torch.empty(rows, kp if fmt == "e4m3" else kp // 2, device=dev, dtype=torch.uint8),
                  torch.empty(rows, (K + 511) // 512 * 16, device=dev, dtype=torch.uint8), K, fmt)


def _coded(r: MXRows, who) -> int:
    """The element type code of coded rows that are laid out as the kernels read them."""
    code = _mx_fmt(r.fmt)
    kp = (r.K + 127) // 128 * 128
    if (r.q.dim() != 2 or r.q.shape[1] != (kp if r.fmt == "e4m3" else kp // 2)
            or r.scale.shape != (r.q.shape[0], (r.K + 511) // 512 * 16) or r.scale.device != r.q.device
            or any(t.element_size() != 1 or not t.is_contiguous() or t.data_ptr() % 16 for t in r[:2])):
        raise ValueError(f"kmoe.{who}: q {tuple(r.q.shape)} {r.q.dtype}, scale {tuple(r.scale.shape)} {r.scale.dtype} are "
                         f"not the contiguous, 16-byte aligned codes and scales of {r.fmt} rows of {r.K} values")
    return code


def _table(t, n, who, name):
    """An int32 table of at least n entries as the kernels read it."""
    if t.dtype != torch.int32 or not t.is_contiguous() or t.numel() < n:
        raise ValueError(f"kmoe.{who}: {name} must be contiguous int32 of {n} entries, got {t.dtype} {tuple(t.shape)}")


def quant_rows_mx(m, fmt="e4m3", row_index=None, n_rows_dev=None) -> MXRows:
    """Microscaled codes of the bf16 rows of m (n, K), K a multiple of 32, or of its rows
    row_index (int32; -1: zeros).  Rows past *n_rows_dev (int32, on the GPU) are left unwritten."""
    code = _mx_fmt(fmt)
    if n_rows_dev is not None:
        _table(n_rows_dev, 1, "quant_rows_mx", "n_rows_dev")
    _one_gpu("quant_rows_mx", m, row_index, n_rows_dev)
    if m.dim() != 2:
        raise ValueError(f"kmoe.quant_rows_mx: a matrix is needed, got {tuple(m.shape)}")
    m = _contig(m, _BF16)
    if row_index is not None:
        row_index = _contig(row_index, torch.int32)
    rows = m.shape[0] if row_index is None else row_index.numel()
    out = _mx_rows(rows, m.shape[1], fmt, m.device)
    with _device(m.device), _Stage("quant_x"):
        _lib.call("kmoe_quant_rows_mx", ptr(m), ptr(row_index), rows, ptr(n_rows_dev), m.shape[1], code, ptr(out.q),
                  ptr(out.scale), _stream(m))
    return out


def dequant_rows_mx(r: MXRows, row_index=None, n_rows_dev=None):
    """The values (n, K) bf16 of coded rows, or of rows row_index (int32; -1: zeros)."""
    code = _coded(r, "dequant_rows_mx")
    if n_rows_dev is not None:
        _table(n_rows_dev, 1, "dequant_rows_mx", "n_rows_dev")
    _one_gpu("dequant_rows_mx", r.q, row_index, n_rows_dev)
    if row_index is not None:
        row_index = _contig(row_index, torch.int32)
    rows = r.q.shape[0] if row_index is None else row_index.numel()
    out = torch.empty(rows, r.K, device=r.q.device, dtype=_BF16)
    with _device(r.q.device), _Stage("mx_dequant"):
        _lib.call("kmoe_dequant_rows_mx", ptr(r.q), ptr(r.scale), ptr(row_index), rows, ptr(n_rows_dev), r.K, code,
                  ptr(out), _stream(r.q))
    return out


def fake_quant_mx_cols(w):
    """The bf16 values that w (E, K, N) stands for in e2m1 blocks of 32 along K, as
    pack_weights_mx packs it."""
    _need_gpu(w)
    if w.dtype not in (torch.float32, _BF16) or w.dim() != 3:
        raise ValueError(f"kmoe.fake_quant_mx_cols: bf16 or f32 (E, K, N) weights are needed, got {w.dtype} "
                         f"{tuple(w.shape)}")
    w = _contig(w.detach(), w.dtype)
    E, K, N = w.shape
    out = torch.empty(E, K, N, device=w.device, dtype=_BF16)
    with _device(w.device):
        _lib.call("kmoe_fake_quant_mx_cols", ptr(w), _fdt(w), E, K, N, ptr(out), _stream(w))
    return out


class PackedWeightsMX(NamedTuple):
    """4-bit expert weights in the products' operand order (kmoe_pack_weights_mx)."""
    w13: torch.Tensor
    s13: torch.Tensor
    w3: torch.Tensor
    s3: torch.Tensor
    E: int
    d: int
    F: int


def pack_weights_mx(w1, w2, w3) -> PackedWeightsMX:
    """e2m1 blocks along K of the expert weights w1, w2 (E,d,F), w3 (E,F,d), packed."""
    _one_gpu("pack_weights_mx", w1, w2, w3)
    E, d, F = w1.shape
    if w2.shape != (E, d, F) or w3.shape != (E, F, d):
        raise ValueError("kmoe.pack_weights_mx: w1/w2 must be (E,d,F) and w3 (E,F,d)")
    dt = w1.dtype
    if dt not in (torch.float32, _BF16):
        raise ValueError(f"kmoe.pack_weights_mx: unsupported weight dtype {dt}")
    w1, w2, w3 = (_contig(w, dt) for w in (w1, w2, w3))
    lib = _lib.load()
    dev = w1.device
    bufs = [torch.empty(lib.kmoe_packed_mx_bytes(E, d, F, i), device=dev, dtype=torch.uint8) for i in range(4)]
    with _device(dev):
        _lib.call("kmoe_pack_weights_mx", ptr(w1), ptr(w2), ptr(w3), _fdt(w1), E, d, F, *(ptr(b) for b in bufs), _stream(w1))
    return PackedWeightsMX(*bufs, E, d, F)


def gemm_gate_up_mx(x: MXRows, row_token, offsets, pw: PackedWeightsMX, max_rows, save_gu=False):
    """Coded rows of silu(x w1) * (x w2) in x's format: permuted row r is x's row
    row_token[r] (row r without row_token).  save_gu (training): (h, gu), gu the bf16
    pre-activation gate / up values (max_rows, 2 F_pad) in the backward's column order."""
    code = _coded(x, "gemm_gate_up_mx")
    _table(offsets, pw.E + 1, "gemm_gate_up_mx", "offsets")
    if row_token is not None:
        _table(row_token, max_rows, "gemm_gate_up_mx", "row_token")
    _one_gpu("gemm_gate_up_mx", x.q, row_token, offsets, pw.w13)
    if x.K != pw.d:
        raise ValueError(f"kmoe.gemm_gate_up_mx: rows of {x.K} values for weights of d={pw.d}")
    if row_token is None and x.q.shape[0] < max_rows:
        raise ValueError(f"kmoe.gemm_gate_up_mx: {x.q.shape[0]} permuted rows, max_rows {max_rows}")
    fp = (pw.F + 127) // 128 * 128
    h = _mx_rows(max(max_rows, 1), pw.F, x.fmt, x.q.device)
    gu = torch.empty(max(max_rows, 1), 2 * fp, device=x.q.device, dtype=_BF16) if save_gu else None
    with _device(x.q.device), _Stage("gemm_gate_up"):
        _lib.call("kmoe_gemm_gate_up_mx", ptr(x.q), ptr(x.scale), code, x.q.shape[0], ptr(row_token),
                  ptr(offsets), pw.E, pw.d, pw.F, max_rows, ptr(pw.w13), ptr(pw.s13), ptr(h.q), ptr(h.scale), ptr(gu),
                  _stream(x.q))
    return (h, gu) if save_gu else h


def gemm_down_mx(h: MXRows, offsets, pw: PackedWeightsMX, max_rows):
    """y (max_rows, d) bf16 = h w3 of the coded rows of each expert."""
    code = _coded(h, "gemm_down_mx")
    _table(offsets, pw.E + 1, "gemm_down_mx", "offsets")
    _one_gpu("gemm_down_mx", h.q, offsets, pw.w3)
    if h.K != pw.F or h.q.shape[0] < max_rows:
        raise ValueError(f"kmoe.gemm_down_mx: rows {tuple(h.q.shape)} of {h.K} values, F={pw.F}, max_rows {max_rows}")
    y = torch.empty(max(max_rows, 1), pw.d, device=h.q.device, dtype=_BF16)
    with _device(h.q.device), _Stage("gemm_down"):
        _lib.call("kmoe_gemm_down_mx", ptr(h.q), ptr(h.scale), code, ptr(offsets), pw.E, pw.d, pw.F, max_rows,
                  ptr(pw.w3), ptr(pw.s3), ptr(y), _stream(h.q))
    return y


@functools.lru_cache(maxsize=1024)
def _mx_workspace(T, d, E, k, F, fmt, coded) -> int:
    return _lib.load().kmoe_mx_experts_workspace_bytes(T, d, E, k, F, fmt, int(coded))


class RoutedOut(NamedTuple):
    """What a one-call pass over routed tokens reports of its dispatch."""
    counts: torch.Tensor        # (E,) int32 routed counts
    aux: Optional[torch.Tensor]  # (3,) f32 aux losses, when asked for


def mx_experts(x2d, idx, w, pw: PackedWeightsMX, fmt, capacity=0, row_index=None, coded: Optional[MXRows] = None,
               block_counts=None, aux=None, T_out=None, out_map=None, scale=None, out_dtype=_BF16, residual=None):
    """Routed tokens through the 4-bit experts in one native call, as dispatch, quant_rows_mx,
    gemm_gate_up_mx, gemm_down_mx and combine do it: (y (T_out, d), counts (E,) int32, aux
    (3,) f32 or None).  fmt: element type of the activations; coded: their codes, if the
    caller has them; aux = (partials, w_lb, w_z): as for dispatch."""
    code = _mx_fmt(fmt)
    _one_gpu("mx_experts", x2d, idx, w, row_index, residual, out_map, scale, block_counts, pw.w13,
             None if coded is None else coded.q)
    x2d = _contig(x2d, _BF16)
    idx = _contig(idx, torch.int64)
    if w.dtype not in (torch.float32, _BF16):
        w = w.float()
    w = w.contiguous()
    T, k = idx.shape
    d = x2d.shape[1]
    if w.shape != (T, k) or pw.d != d or (row_index is None and x2d.shape[0] != T):
        raise ValueError(f"kmoe.mx_experts: x {tuple(x2d.shape)}, idx {(T, k)}, w {tuple(w.shape)}, weights of d={pw.d}")
    xq = xs = None
    if coded is not None:
        if coded.fmt != fmt or coded.K != d or coded.q.shape[0] != T or row_index is not None:
            raise ValueError(f"kmoe.mx_experts: coded rows {tuple(coded.q.shape)} ({coded.fmt}, K={coded.K}) for T={T}, "
                             f"d={d}, {fmt}")
        _coded(coded, "mx_experts")
        xq, xs = coded.q, coded.scale
    if row_index is not None:
        row_index = _contig(row_index, torch.int32)
        if row_index.numel() != T:
            raise ValueError(f"kmoe.mx_experts: row_index of {row_index.numel()} rows for {T} tokens")
    T_out = T if T_out is None else T_out
    if out_map is not None:
        _table(out_map, T_out, "mx_experts", "out_map")
    if scale is not None and (scale.dtype != torch.float32 or not scale.is_contiguous() or scale.numel() < T):
        raise ValueError(f"kmoe.mx_experts: scale must be contiguous f32 of {T} tokens, got {scale.dtype} "
                         f"{tuple(scale.shape)}")
    dev = x2d.device
    y = torch.empty(T_out, d, device=dev, dtype=out_dtype)
    if residual is not None:
        residual = _contig(residual, out_dtype)
        if residual.shape != (T_out, d):
            raise ValueError(f"kmoe.mx_experts: residual shape {tuple(residual.shape)} != {(T_out, d)}")
    if T == 0:
        y.zero_() if residual is None else y.copy_(residual)
        return y, torch.zeros(pw.E, device=dev, dtype=torch.int32), None
    counts = torch.empty(pw.E, device=dev, dtype=torch.int32)
    partials = aux_out = None
    w_lb = w_z = 0.0
    if aux is not None:
        partials, w_lb, w_z = aux
        aux_out = torch.empty(3, device=dev, dtype=torch.float32)
    lib = _lib._LIB or _lib.load()
    with _device(dev):
        if block_counts is not None and (block_counts.dtype != torch.int32 or not block_counts.is_contiguous() or
                                         block_counts.numel() != -(-T // lib.kmoe_router_block_tokens(T)) * pw.E):
            raise ValueError("kmoe.mx_experts: block_counts must be the router's per-block histograms (int32)")
        wsb = _mx_workspace(T, d, pw.E, k, pw.F, code, coded is not None)
        ws = torch.empty(max(wsb, 4), device=dev, dtype=torch.uint8)
        _lib.call("kmoe_mx_experts", ptr(x2d), ptr(row_index), T, d, code, ptr(xq), ptr(xs), ptr(idx), ptr(w),
                  _lib.DTYPE_F32 if w.dtype == torch.float32 else _lib.DTYPE_BF16, k, pw.E, int(capacity), ptr(block_counts),
                  ptr(partials), float(w_lb), float(w_z), ptr(aux_out), ptr(pw.w13), ptr(pw.s13), ptr(pw.w3), ptr(pw.s3),
                  pw.F, ptr(out_map), ptr(scale), ptr(residual), T_out, ptr(y),
                  _lib.DTYPE_F32 if out_dtype == torch.float32 else _lib.DTYPE_BF16, ptr(counts), ptr(ws), wsb, _stream(x2d))
    return y, counts, aux_out


class AddNormOut(NamedTuple):
    h: torch.Tensor                # (T, d) x + delta, in x's type
    n: torch.Tensor                # (T, d) bf16 RMSNorm of h
    rrms: torch.Tensor             # (T,) f32 1/sqrt(mean(h^2) + eps)
    q: Optional[torch.Tensor]      # codes and scales of n (quant), as MXRows has them
    scale: Optional[torch.Tensor]


def add_rmsnorm(x2d, delta, weight, eps, quant=None) -> AddNormOut:
    """Residual add and RMSNorm in one pass: h = x + delta (delta None: x itself),
    n = bf16(weight * h / sqrt(mean(h^2) + eps)) and, with quant "e4m3" / "e2m1", n's
    microscaled rows (those of quant_rows_mx(n)).  x2d, delta (T, d) bf16 or f32; an f32
    delta makes h f32.  Not differentiable: kmoe.add_rms_norm is."""
    code = _lib.DTYPE_BF16 if quant is None else _mx_fmt(quant)
    _one_gpu("add_rmsnorm", x2d, delta, weight)
    T, d = x2d.shape
    if weight.shape != (d,) or (delta is not None and delta.shape != (T, d)):
        raise ValueError(f"kmoe.add_rmsnorm: x {(T, d)}, delta {None if delta is None else tuple(delta.shape)}, weight "
                         f"{tuple(weight.shape)}")
    dt = x2d.dtype if x2d.dtype in (torch.float32, _BF16) else torch.float32
    if delta is not None:
        if delta.dtype != _BF16:
            dt = torch.float32
            delta = _contig(delta, torch.float32)
        else:
            delta = delta.contiguous()
    x2d = _contig(x2d, dt)
    weight = weight.detach()
    weight = _contig(weight, weight.dtype if weight.dtype in (torch.float32, _BF16) else torch.float32)
    dev = x2d.device
    h = x2d if delta is None else torch.empty_like(x2d)
    n = torch.empty(T, d, device=dev, dtype=_BF16)
    rrms = torch.empty(T, device=dev, dtype=torch.float32)
    rows = _mx_rows(T, d, quant, dev) if quant is not None else None
    q, scale = (None, None) if rows is None else rows[:2]
    with _device(dev), _Stage("rmsnorm"):
        _lib.call("kmoe_add_rmsnorm", ptr(x2d), _fdt(x2d), ptr(delta), _lib.DTYPE_BF16 if delta is None else _fdt(delta),
                  ptr(weight), _fdt(weight), float(eps), T, d, ptr(h), ptr(n), ptr(rrms), code, ptr(q), ptr(scale),
                  _stream(x2d))
    return AddNormOut(h, n, rrms, q, scale)


def add_rmsnorm_bwd(dn, h, weight, rrms, dh=None, bf16=False, dw_dtype=None):
    """Backward of add_rmsnorm from dn and dh (None: zero), the gradients of n and h (T, d):
    (dx in h's type, dx rounded to bf16 or None, dweight).  dx is the gradient of x and of
    delta; bf16 asks for the rounding of an f32 one, for the input that is bf16."""
    T, d = h.shape
    if dn.shape != (T, d) or (dh is not None and dh.shape != (T, d)) or weight.shape != (d,) or rrms.shape != (T,):
        raise ValueError(f"kmoe.add_rmsnorm_bwd: h {(T, d)}, dn {tuple(dn.shape)}, dh "
                         f"{None if dh is None else tuple(dh.shape)}, weight {tuple(weight.shape)}, rrms {tuple(rrms.shape)}")
    if rrms.dtype != torch.float32:
        raise ValueError(f"kmoe.add_rmsnorm_bwd: rrms must be the forward's f32, got {rrms.dtype}")
    _one_gpu("add_rmsnorm_bwd", h, dn, weight, rrms, dh)
    dn, h, rrms = _contig(dn, _BF16), h.contiguous(), rrms.contiguous()
    weight = weight.detach()
    dw_dtype = weight.dtype if dw_dtype is None else dw_dtype
    weight = _contig(weight, weight.dtype if weight.dtype in (torch.float32, _BF16) else torch.float32)
    dh = _contig(dh, h.dtype)
    dev = h.device
    dx = torch.empty(T, d, device=dev, dtype=h.dtype)
    dx16 = torch.empty(T, d, device=dev, dtype=_BF16) if bf16 and h.dtype == torch.float32 else None
    dwt = torch.empty(d, device=dev, dtype=dw_dtype if dw_dtype in (torch.float32, _BF16) else torch.float32)
    lib = _lib._LIB or _lib.load()
    wsb = lib.kmoe_rmsnorm_bwd_workspace_bytes(T, d)
    ws = torch.empty(max(wsb, 4), device=dev, dtype=torch.uint8)
    with _device(dev), _Stage("bwd_rmsnorm"):
        _lib.call("kmoe_add_rmsnorm_bwd", ptr(dn), ptr(h), _fdt(h), ptr(weight), _fdt(weight), ptr(rrms), ptr(dh), T, d,
                  ptr(dx), ptr(dx16), ptr(dwt), _fdt(dwt), ptr(ws), wsb, _stream(h))
    return dx, dx16, dwt.to(dw_dtype)
