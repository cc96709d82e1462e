"""What is made from weights and kept (packed weights, casts) is made again when they change.  The
packing itself is a stand-in here: no kernel is launched."""
import copy
import pickle

import numpy as np
import pytest
import torch
from torch import nn

import kmoe
from kmoe import kernels, ops

E, D, F = 2, 64, 8


@pytest.fixture
def packs(monkeypatch):
    """Packing that returns the weights' sum, and counts."""
    made = []

    def pack(*ws, **kw):
        made.append(float(sum(w.double().sum() for w in ws if w is not None)))
        return made[-1]
    for name in ("pack_weights", "pack_weights_mx"):
        monkeypatch.setattr(ops, name, pack)
    monkeypatch.setattr(kmoe.backward, "pack_bwd_weights", pack)
    monkeypatch.setattr(ops, "fake_quant_mx_cols", lambda w: w)
    return made


def at_one_address(n):
    """Tensors of storages of their own at one address: what the allocator makes of a weight that is
    freed before the next is made."""
    memory = np.zeros((E, D, F), dtype=np.float32)
    return [torch.from_numpy(memory) for _ in range(n)], memory


@pytest.mark.parametrize("mx", [None, "w4a8"])
def test_kept_until_a_weight_is_written(packs, mx):
    ex = kmoe.GroupedExperts(E, D, F)
    ex.mx = mx
    first = ex.packed()
    assert ex.packed() == first and len(packs) == 1
    with torch.no_grad():
        ex.w1.add_(1.0)
    assert ex.packed() == pytest.approx(first + ex.w1.numel()) and len(packs) == 2
    ex.use_fp8, ex.mx = mx is None, None
    ex.packed()
    assert len(packs) == 3


@pytest.mark.parametrize("mx", [None, "w4a8"])
@pytest.mark.parametrize("get", ["packed", "bwd_packed"])
@pytest.mark.parametrize("how", ["parameter", "data"])
def test_another_weight_at_the_same_address(packs, mx, get, how):
    ex = kmoe.GroupedExperts(E, D, F)
    ex.mx = mx
    tensors, memory = at_one_address(3)
    ex.w1 = nn.Parameter(tensors[0])
    assert tensors[1].data_ptr() == ex.w1.data_ptr()
    rest = float((ex.w2.double().sum() + ex.w3.double().sum()).detach())
    assert getattr(ex, get)() == pytest.approx(rest)
    for value, t in ((1.0, tensors[1]), (2.0, tensors[2])):
        memory[:] = value
        if how == "parameter":
            ex.w1 = nn.Parameter(t)
        else:
            ex.w1.data = t
        assert ex.w1._version == 0
        assert getattr(ex, get)() == pytest.approx(rest + value * memory.size)


def test_routers_casts_and_free_functions(packs):
    tensors = [torch.from_numpy(m) for m in [np.zeros((128, D), dtype=np.float32)] * 2]
    r = kmoe.Router(kmoe.AdvancedMoEConfig(d_model=D, n_experts=4, d_ff_expert=F))
    r.router[0].weight = nn.Parameter(tensors[0])
    assert not r._kernel_weights()[0].any()
    tensors[1].fill_(1.0)
    r.router[0].weight = nn.Parameter(tensors[1].detach())
    assert bool((r._kernel_weights()[0] == 1.0).all())
    ws, memory = at_one_address(2)
    zero = torch.zeros(E, D, F)
    assert kernels._packed(ws[0], zero, zero.transpose(1, 2)) == 0.0
    memory[:] = 1.0
    assert kernels._packed(ws[1], zero, zero.transpose(1, 2)) == memory.size


def test_copies_pack_for_themselves(packs):
    ex = kmoe.GroupedExperts(E, D, F)
    ex.packed(), ex.bwd_packed()
    for other in (copy.deepcopy(ex), pickle.loads(pickle.dumps(ex))):
        n = len(packs)
        other.packed(), other.bwd_packed()
        assert len(packs) == n + 2
    ex.packed()
    assert len(packs) == 6


def test_entries_of_modules_pickled_before(packs):
    """An entry keyed by addresses and versions, as modules once held it, is not taken."""
    ex = kmoe.GroupedExperts(E, D, F)
    ex._packed = (tuple((w.data_ptr(), w._version) for w in ex._weights()), "old")
    assert ex.packed() != "old"


def test_weights_changed(packs):
    """Writes that torch does not count are seen once the caller says so."""
    layer = kmoe.MoELayer(kmoe.AdvancedMoEConfig(d_model=D, n_experts=E, moe_top_k=1, d_ff_expert=F, moe_mx="w4a4"))
    ex = layer.grouped_experts
    before, back, cast = ex.packed(), layer._bwd_weights(), layer.router._kernel_weights()[0].clone()
    for p in layer.parameters():
        p.data.mul_(2.0)
    assert ex.packed() == before  # not counted
    kmoe.weights_changed(layer)
    assert ex.packed() == pytest.approx(2 * before) and layer._bwd_weights() == pytest.approx(2 * back)
    assert torch.equal(layer.router._kernel_weights()[0], 2 * cast)


def test_freed_weights_are_not_held():
    """The key keeps no weight's memory."""
    from kmoe.derived import Sources
    t = torch.zeros(1000)
    storage = torch.multiprocessing.reductions.StorageWeakRef(t.untyped_storage())
    s = Sources((t,))
    assert s.same((t,)) and not storage.expired()
    del t
    assert storage.expired() and not s.same((torch.zeros(1000),))


def test_captures(packs, monkeypatch):
    """What is made in a capture is not kept; what a capture uses outlives its replacement; a training
    pass in a capture makes it anew.  (A capture is a stand-in here.)"""
    from kmoe import backward, derived
    state = dict(capturing=False)
    for m in (derived, backward):
        monkeypatch.setattr(m, "capturing", lambda t: state["capturing"])
    ex = kmoe.GroupedExperts(E, D, F)
    state["capturing"] = True
    ex.packed()
    assert ex._packed is None and len(packs) == 1
    state["capturing"] = False
    kept = ex.packed()
    assert ex._packed[1] is kept and len(packs) == 2
    state["capturing"] = True
    assert ex.packed() is kept and ex.packed() is kept and len(packs) == 2
    ex.packed(training=True), ex.bwd_packed()
    assert len(packs) == 4 and ex._packed[1] is kept
    state["capturing"] = False
    with torch.no_grad():
        ex.w1.add_(1.0)
    assert ex.packed() is not kept and [v for v in ex._held if v is kept] == [kept]
    other = copy.deepcopy(ex)
    assert not other._held
    # constants of shapes
    monkeypatch.setattr(backward, "_ONES", {})
    monkeypatch.setattr(backward, "_IN_GRAPHS", set())
    state["capturing"] = True
    assert backward._ones(3, 2, "cpu") is not backward._ones(3, 2, "cpu")
    state["capturing"] = False
    t = backward._ones(3, 2, "cpu")
    state["capturing"] = True
    assert backward._ones(3, 2, "cpu") is t
    state["capturing"] = False
    for n in range(40):
        backward._ones(4 + n, 2, "cpu")
    assert backward._ones(3, 2, "cpu") is t and len(backward._ONES) < 20
