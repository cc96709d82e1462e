"""AdamW over all tensors of a parameter group in one launch, states in 32 or in 8 bits.

The step that a training program takes after the layers' backward.  A step writes the weights
outside of torch's operations and counts the change, so what the modules keep from their weights
(packed copies, casts) follows; replays of a captured step are not counted, as everywhere
(kmoe.weights_changed).
"""
from __future__ import annotations

import ctypes
from operator import is_ as _is
from typing import Optional

import torch

from . import _lib
from .ops import _device

BLOCK = 256   # values of an 8-bit state that share a scale
CHUNK = 8192  # values of a workgroup
# a tensor's row of the kernel's table: its address, those of its states, its size
_FIELDS = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master", "step")


class _Plan:
    """The tensors of a group of one type on one device, as the kernel's table has them."""

    def __init__(self, params, states, bits, has_master):
        dev = params[0].device
        self._apart(params, states)
        rows, base, owner = [], [0], []
        for i, (p, st) in enumerate(zip(params, states)):
            rows.append([*self._where(p, st), p.numel()])
            chunks = -(-p.numel() // CHUNK)
            base.append(base[-1] + chunks)
            owner.append(torch.full((chunks,), i, dtype=torch.int32))
        if base[-1] >= 1 << 31:
            raise ValueError("kmoe.AdamW: more than 2^31 chunks of values in one group")
        self.table = torch.tensor(rows, dtype=torch.int64).to(dev)
        self.owner = torch.cat(owner).to(dev)
        self.base = torch.tensor(base, dtype=torch.int32).to(dev)
        self.base_host = (ctypes.c_int32 * len(base))(*base)
        self.tickets = torch.zeros(len(rows), dtype=torch.int32, device=dev)
        self.grads = (ctypes.c_void_p * len(rows))()
        self.params, self.states = params, states
        self.has_master = has_master
        self.bits = bits
        self.dtype = _lib.DTYPE_F32 if params[0].dtype == torch.float32 else _lib.DTYPE_BF16
        self.device = dev
        self.kind = params[0].dtype
        self.shapes = [p.shape for p in params]
        self.at = [(p, p.data_ptr(), p.shape, st, [(k, st[k], st[k].data_ptr()) for k in _FIELDS if k in st])
                   for p, st in zip(params, states)]

    @staticmethod
    def _apart(params, states):
        """Refuses tensors that share memory: workgroups write them side by side."""
        places = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), tuple(p.shape))
                        for p, st in zip(params, states) for t in (p, *(st[k] for k in _FIELDS if k in st)) if t.numel())
        for (_, end, a), (start, _, b) in zip(places, places[1:]):
            if start < end:
                raise ValueError(f"kmoe.AdamW: parameters {a} and {b} of one group, or states of theirs, share memory")

    @staticmethod
    def _where(p, st):
        return [p.data_ptr(), *(st[k].data_ptr() if k in st else 0 for k in _FIELDS)]

    def current(self) -> bool:
        """Whether the states hold the same tensors, each tensor is where it was and the parameters are what
        they were."""
        kind = self.kind
        for p, at, shape, st, held in self.at:
            if p.data_ptr() != at or p.shape != shape or p.dtype is not kind or not p.is_contiguous():
                return False
            for k, t, place in held:
                if st.get(k) is not t or t.data_ptr() != place:
                    return False
        return True


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) on the HIP kernel, for bf16 and f32 parameters on GPUs.

    state_bits 32: f32 moments, as torch.optim.AdamW has them.  8: one byte a value and one f32
    scale per 256 values; the first moment in e4m3, the second as the square root in unsigned
    codes of 4 exponent and 4 mantissa bits, a positive one never as zero.  master_weights (bf16
    parameters): the step works on an f32 copy of the weights, kept in the state, and the
    parameters are its rounding; without it, changes below half a bf16 step are lost.  When
    something else has written the parameter (as torch counts it), the copy is made anew where it
    does not round to it; a copied or unpickled optimizer keeps its copies' bits.

    lr may be a one-element f32 tensor on the parameters' GPU, read when the step runs: a captured
    step follows it.  The step count is on the GPU too, one per parameter; a parameter without a
    gradient is left alone.  A capture needs one eager step first, and gradients that stay where
    they are."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 master_weights=False):
        self._check(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))
        self._plans, self._stepped, self._states, self._held, self._seen = None, [], ([], []), [], {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      master_weights=bool(master_weights)))

    @staticmethod
    def _check(group):
        lr, (b1, b2) = group["lr"], group["betas"]
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"kmoe.AdamW: lr={lr}")
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0 and group["eps"] >= 0.0 and group["weight_decay"] >= 0.0):
            raise ValueError(f"kmoe.AdamW: betas {group['betas']} lie in [0, 1), eps {group['eps']} and weight_decay "
                             f"{group['weight_decay']} are not negative")
        if group["state_bits"] not in (32, 8):
            raise ValueError(f"kmoe.AdamW: state_bits={group['state_bits']} is neither 32 nor 8")

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        try:
            self._check(group)
            for p in group["params"]:
                self._check_param(p)
            if len(set(map(id, group["params"]))) < len(group["params"]):
                raise ValueError("kmoe.AdamW: a parameter stands twice in its group")
        except Exception:
            self.param_groups.pop()
            raise
        self._plans = None

    @staticmethod
    def _check_param(p):
        if p.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"kmoe.AdamW: parameters are bf16 or f32, got {p.dtype}")
        if not p.is_contiguous():
            raise ValueError(f"kmoe.AdamW: parameters are contiguous, got strides {p.stride()} of {tuple(p.shape)}")

    # _plans: the tables of the last step, _stepped: each group's parameters in them and the form of their
    # states, _states: the states that they were made from; _held: what captured steps read; _seen: version
    # of each parameter with an f32 copy after its last step
    def __setstate__(self, state):
        super().__setstate__(state)
        self._plans, self._stepped, self._states, self._seen = None, [], ([], []), {}
        self.__dict__.setdefault("_held", [])  # (torch's load_state_dict comes here too: graphs stay)

    def __getstate__(self):
        return {k: v for k, v in super().__getstate__().items() if k not in ("_plans", "_stepped", "_states", "_held", "_seen")}

    # ---------------------------------------------------------------- states
    def _new_state(self, p, group):
        st = {"step": torch.zeros(1, dtype=torch.int32, device=p.device)}
        if group["state_bits"] == 32:
            st["exp_avg"], st["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32) for _ in range(2))
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                st[k] = torch.zeros(p.numel(), dtype=torch.uint8, device=p.device)
                st[k + "_scale"] = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.float32, device=p.device)
        if group["master_weights"] and p.dtype == torch.bfloat16:
            st["master"] = p.detach().float()
        return st

    def _group_of(self, p):
        for g in self.param_groups:
            if any(q is p for q in g["params"]):
                return g
        raise ValueError("kmoe.AdamW: not a parameter of this optimizer")

    def _check_state(self, p, group, st):
        want = self._new_state(torch.empty(p.shape, dtype=p.dtype, device="meta"), group)
        odd = [k for k in _FIELDS if k in st and k not in want]
        if odd:
            raise ValueError(f"kmoe.AdamW: the state {', '.join(odd)} of a parameter {tuple(p.shape)} has no place in a group with "
                             f"state_bits {group['state_bits']} and master_weights {group['master_weights']}")
        for k, v in want.items():
            t = st.get(k)
            if (not isinstance(t, torch.Tensor) or t.dtype != v.dtype or t.numel() != v.numel() or t.device != p.device
                    or not t.is_contiguous()):
                raise ValueError(f"kmoe.AdamW: the state {k} of a parameter {tuple(p.shape)} is contiguous {v.dtype} of "
                                 f"{v.numel()} values on {p.device}, got "
                                 f"{(t.dtype, tuple(t.shape), str(t.device)) if isinstance(t, torch.Tensor) else t}")

    def set_state(self, p, step: int, **tensors) -> None:
        """Takes `tensors` (exp_avg, exp_avg_sq; in 8 bits also exp_avg_scale, exp_avg_sq_scale; with
        master weights master, else a copy of p) as p's state after `step` steps: the tensors
        themselves, written by later steps."""
        group = self._group_of(p)
        st = dict(tensors)
        st["step"] = torch.full((1,), int(step), dtype=torch.int32, device=p.device)
        if "master" not in st and group["master_weights"] and p.dtype == torch.bfloat16:
            st["master"] = p.detach().float()
        self._check_state(p, group, st)
        self.state[p] = st
        self._seen[p] = p._version
        self._plans = None

    def state_values(self, p, dtype=torch.float32):
        """(first moment, square root of the second) of p as bf16 or f32: in 8 bits the values that the
        codes stand for."""
        self._group_of(p)
        st = self.state.get(p)
        if not st:
            raise ValueError(f"kmoe.AdamW: a parameter {tuple(p.shape)} has no state before its first step")
        if dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"kmoe.AdamW: state values are bf16 or f32, not {dtype}")
        if "exp_avg_scale" not in st:
            return st["exp_avg"].to(dtype).view(p.shape), st["exp_avg_sq"].sqrt().to(dtype).view(p.shape)
        if not p.is_cuda:
            raise ValueError("kmoe.AdamW: parameters must be on a GPU (the HIP kernel is the only implementation)")
        m, root = (torch.empty(p.shape, dtype=dtype, device=p.device) for _ in range(2))
        with _device(p.device):
            _lib.call("kmoe_adamw_values", *(st[k].data_ptr() for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq",
                                                                       "exp_avg_sq_scale")), p.numel(),
                      _lib.DTYPE_F32 if dtype == torch.float32 else _lib.DTYPE_BF16, m.data_ptr(), root.data_ptr(),
                      _lib.stream_ptr(p.device))
        return m, root

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but the states keep the types they were saved in (torch casts them to their
        parameter's); what is refused leaves the optimizer as it was."""
        before = self.state, self.param_groups, self._plans, self._stepped, self._states, self._seen
        super().load_state_dict(state_dict)
        try:
            saved, states = state_dict["state"], {}
            params = [p for g in self.param_groups for p in g["params"]]
            names = [i for g in state_dict["param_groups"] for i in g["params"]]
            for group in self.param_groups:
                lacks = [k for k in ("lr", "betas", "eps", "weight_decay", "state_bits", "master_weights") if k not in group]
                if lacks:
                    raise ValueError(f"kmoe.AdamW: a parameter group of the state dict has no {', '.join(lacks)}")
                self._check(group)
            for i, p in zip(names, params):
                if i in saved:
                    st = {k: v.detach().to(p.device, copy=True).contiguous() if isinstance(v, torch.Tensor) else v
                          for k, v in saved[i].items()}
                    self._check_state(p, self._group_of(p), st)
                    states[p] = st
        except Exception:
            self.state, self.param_groups, self._plans, self._stepped, self._states, self._seen = before
            raise
        self.state.update(states)
        self._seen.update((p, p._version) for p in states)

    # ---------------------------------------------------------------- the step
    def _to_step(self, group):
        """The group's parameters that have had a gradient."""
        return [p for p in group["params"] if p.grad is not None or p in self.state]

    def _plan(self) -> None:
        """The tables of the parameters that have had a gradient."""
        plans, stepped = [], []
        for group in self.param_groups:
            kinds = {}
            stepped.append((group, self._to_step(group), group["state_bits"], group["master_weights"]))
            for p in stepped[-1][1]:
                if not p.is_cuda:
                    raise ValueError("kmoe.AdamW: parameters must be on a GPU (the HIP kernel is the only implementation)")
                self._check_param(p)
                if not self.state.get(p):
                    self.state[p] = self._new_state(p, group)
                    self._seen[p] = p._version
                else:
                    self._check_state(p, group, self.state[p])
                kinds.setdefault((p.device, p.dtype, "master" in self.state[p]), []).append(p)
                # (a state of another form than the group's has been refused)
            for (_, _, master), ps in kinds.items():
                plans.append((group, _Plan(ps, [self.state[p] for p in ps], group["state_bits"], master)))
        self._plans, self._stepped, self._states = plans, stepped, (list(self.state), list(self.state.values()))

    def _stale(self) -> bool:
        if self._plans is None or len(self._stepped) != len(self.param_groups):
            return True
        for group, (known, ps, bits, master) in zip(self.param_groups, self._stepped):
            now = self._to_step(group)
            if (group is not known or group["state_bits"] != bits or group["master_weights"] != master or len(now) != len(ps)
                    or not all(map(_is, now, ps))):
                return True
        # (the whole state entry by entry: a parameter's own would be looked up by its hash, which costs more)
        keys, states = self._states
        if len(self.state) != len(keys) or not all(map(_is, self.state, keys)) or not all(map(_is, self.state.values(), states)):
            return True
        return not all(plan.current() for _, plan in self._plans)

    @torch.no_grad()
    def step(self, closure=None) -> Optional[torch.Tensor]:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        if self._stale():
            if capturing:
                raise RuntimeError("kmoe.AdamW: a capture needs the states and tables of an eager step before it: take one, "
                                   "and keep the parameters where they are")
            self._plan()
        for group, plan in self._plans:
            lr, (b1, b2) = group["lr"], group["betas"]
            lr_dev, kept, moved = None, [], []
            if isinstance(lr, torch.Tensor):
                if lr.device == plan.device:
                    if lr.dtype != torch.float32 or lr.numel() != 1:
                        raise ValueError(f"kmoe.AdamW: lr is one f32 value, got {lr.dtype} {tuple(lr.shape)}")
                    lr_dev, lr = lr.data_ptr(), 0.0
                else:
                    lr = float(lr)
            kind, dev, shapes = plan.kind, plan.device, plan.shapes
            for i, p in enumerate(plan.params):
                g = p.grad
                if g is None:
                    plan.grads[i] = None
                    continue
                if g.dtype is not kind or g.shape != shapes[i] or g.device != dev or g.is_sparse:
                    raise ValueError(f"kmoe.AdamW: gradients are dense and of their parameter's type, device and shape, got "
                                     f"{g.dtype} {tuple(g.shape)} on {g.device}")
                if not g.is_contiguous():
                    g = g.contiguous()
                    kept.append(g)  # until the launch
                plan.grads[i] = g.data_ptr()
                moved.append(p)
                if plan.has_master and self._seen.get(p) != p._version:
                    if capturing:
                        raise RuntimeError("kmoe.AdamW: a parameter was written since the last step; take an eager step, which "
                                           "makes its f32 copy anew, before the capture")
                    # (anew where it does not round to the parameter: what was not written keeps its bits)
                    master = plan.states[i]["master"]
                    master.copy_(torch.where(master.to(p.dtype) == p, master, p.float()))
            if not any(p.numel() for p in moved):
                continue
            if capturing and not any(a is plan and b is group["lr"] for a, b, _ in self._held):
                # the replays read its tables and a rate on the GPU, and write the parameters as they lie now
                self._held.append((plan, group["lr"], [p.detach() for p in plan.params]))
            with _device(plan.device):
                _lib.call("kmoe_adamw", plan.table.data_ptr(), plan.owner.data_ptr(), plan.base.data_ptr(),
                          plan.base_host, len(plan.params), plan.grads, plan.dtype, plan.bits,
                          int(plan.has_master), float(lr), lr_dev, b1, b2, float(group["eps"]),
                          float(group["weight_decay"]), plan.tickets.data_ptr(), _lib.stream_ptr(plan.device))
            torch.autograd.graph.increment_version(moved)
            if plan.has_master:
                for p in moved:
                    self._seen[p] = p._version
        return loss
