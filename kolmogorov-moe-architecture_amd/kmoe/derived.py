"""Values made from weights (packed copies, casts, folds), kept until a weight changes.

What torch counts is seen: a write by an operation (an optimizer's step, copy_), a parameter that
is replaced, a .data that is assigned.  What it does not count is not: a write through .data or
a view of it, by a replayed graph, or by code outside of torch; `weights_changed` is for those.

In a capture nothing runs, so what is made there is not kept: it has no contents before a replay.
What was made before and is used in a capture lives as long as its module, since the replays
read it, also when later calls have made another.  A training step's replays make everything
anew, as weights move between them.
"""
from __future__ import annotations

import torch
from torch.multiprocessing.reductions import StorageWeakRef


def _state(tensors, flags):
    s = [flags]  # (one list and one comparison: this runs in every call)
    for t in tensors:
        s += (t._version, t.data_ptr(), t.untyped_storage()._cdata)
    return s


class Sources:
    """The tensors that a value was made from: their addresses, version counters and storages.  An
    address and a counter alone say nothing, as the allocator gives a freed weight's place to
    the next one and counters start at zero; the weak references hold on to no memory, but to the
    storages' identities.  Equal to nothing once copied or pickled with its module, whose
    copy has other weights."""
    __slots__ = ("_at", "_refs")

    def __init__(self, tensors, flags=()):
        self._at = _state(tensors, flags)
        self._refs = tuple(StorageWeakRef(t.untyped_storage()) for t in tensors)

    def same(self, tensors, flags=()) -> bool:
        return _state(tensors, flags) == self._at

    def __reduce__(self):
        return _gone, ()

    def __deepcopy__(self, memo):
        return _gone()


def _gone() -> Sources:
    return Sources((), None)


def capturing(t) -> bool:
    """Whether work on t's device is being captured into a graph (the default stream, 0, never is, and costs
    less to tell)."""
    i = t.get_device()
    return i >= 0 and torch._C._cuda_getCurrentRawStream(i) != 0 and torch.cuda.is_current_stream_capturing()


class _Held(list):
    """Values that graphs read; a module's copy has no such graphs."""

    def __reduce__(self):
        return _Held, ()

    def __deepcopy__(self, memo):
        return _Held()


def derived(owner: dict, name: str, tensors, make, flags=(), training=False):
    """What make() made from the tensors (and the flags), kept in owner[name] (a module's __dict__)
    until one of them changes.  training: of a pass whose weights move, see above."""
    entry = owner.get(name)
    if entry is not None and isinstance(entry[0], Sources) and entry[0].same(tensors, flags):
        if not capturing(tensors[0]):
            return entry[1]
        if not training:
            held = owner.setdefault("_held", _Held())
            if not any(v is entry[1] for v in held):
                held.append(entry[1])
            return entry[1]
    with torch.no_grad():
        value = make()
    if not capturing(tensors[0]):
        owner[name] = (Sources(tensors, flags), value)
    return value


_ENTRIES = ("_packed", "_bwd_cache", "_bf16_cache", "_fused_cache")
FREE = {}  # entries of functions that take weights and belong to no module


def weights_changed(module) -> None:
    """Forget what was made from the weights of `module` and the modules in it: its next call makes
    it again.  For writes that torch does not count: through .data, by replays of a captured
    optimizer step, by other code on the memory."""
    FREE.pop("grouped_swiglu_forward", None)
    for m in module.modules():
        for name in _ENTRIES:
            if m.__dict__.get(name) is not None:
                setattr(m, name, None)
