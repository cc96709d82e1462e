"""kmoe.AdamW without a GPU: refusals, states, state dicts, and the ABI's checks."""
import ctypes

import pytest
import torch

import kmoe
from kmoe import _lib

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first


def _param(*shape, dtype=torch.bfloat16):
    return torch.nn.Parameter(torch.zeros(*shape, dtype=dtype))


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-9),
                                dict(weight_decay=-0.1), dict(state_bits=4), dict(state_bits=16), dict(lr=float("nan"))])
def test_refuses_hyperparameters(kw):
    with pytest.raises(ValueError, match="kmoe.AdamW"):
        kmoe.AdamW([_param(4)], **kw)


def test_refuses_parameters():
    with pytest.raises(ValueError, match="bf16 or f32"):
        kmoe.AdamW([_param(4, dtype=torch.float16)])
    with pytest.raises(ValueError, match="contiguous"):
        kmoe.AdamW([torch.nn.Parameter(torch.zeros(4, 6).t())])
    opt = kmoe.AdamW([_param(4)])
    with pytest.raises(ValueError, match="bf16 or f32"):
        opt.add_param_group({"params": [_param(4, dtype=torch.float64)]})
    p = _param(4)
    p.grad = torch.zeros_like(p)
    with pytest.raises(ValueError, match="on a GPU"):
        kmoe.AdamW([p]).step()


@pytest.mark.parametrize("bits", [8, 32])
def test_set_state_is_checked(bits):
    p = _param(3, 100)
    opt = kmoe.AdamW([p], state_bits=bits)
    f32 = lambda n: torch.zeros(n)
    good = (dict(exp_avg=f32(300), exp_avg_sq=f32(300)) if bits == 32 else
            dict(exp_avg=torch.zeros(300, dtype=torch.uint8), exp_avg_scale=f32(2),
                 exp_avg_sq=torch.zeros(300, dtype=torch.uint8), exp_avg_sq_scale=f32(2)))
    opt.set_state(p, 3, **good)
    assert int(opt.state[p]["step"]) == 3
    for k in good:
        for bad in (None, good[k][:-1], good[k].double()):
            with pytest.raises(ValueError, match=k):
                opt.set_state(p, 3, **{**good, k: bad})
    with pytest.raises(ValueError, match="not a parameter"):
        opt.set_state(_param(3, 100), 3, **good)


@pytest.mark.parametrize("bits", [8, 32])
def test_state_dict_keeps_types(bits):
    """torch's own load casts a state to its parameter's type; these keep theirs."""
    def make():
        p, q = _param(3, 100), _param(7)
        return p, q, kmoe.AdamW([p, q], state_bits=bits, master_weights=True)

    p, q, opt = make()
    for t in (p, q):
        st = opt._new_state(t, opt.param_groups[0])
        opt.set_state(t, 5, **{k: (v.random_(0, 200) if v.dtype == torch.uint8 else v.normal_()) for k, v in st.items()
                               if k != "step"})
    p2, q2, opt2 = make()
    opt2.load_state_dict(opt.state_dict())
    for a, b in ((p, p2), (q, q2)):
        assert set(opt.state[a]) == set(opt2.state[b])
        for k, v in opt.state[a].items():
            w = opt2.state[b][k]
            assert w.dtype == v.dtype and torch.equal(w, v) and w.data_ptr() != v.data_ptr(), k
    _, _, other = make()
    other.param_groups[0]["state_bits"] = 40 - bits
    sd = opt.state_dict()
    sd["param_groups"][0]["state_bits"] = 40 - bits
    with pytest.raises(ValueError, match="the state"):
        other.load_state_dict(sd)


def test_pickled_optimizer_keeps_its_states():
    import copy
    p = _param(5)
    opt = kmoe.AdamW([p], state_bits=32)
    opt.set_state(p, 2, exp_avg=torch.ones(5), exp_avg_sq=torch.ones(5))
    c = copy.deepcopy(opt)
    (q,) = c.param_groups[0]["params"]
    assert int(c.state[q]["step"]) == 2 and c._plans is None


def test_abi_refuses():
    lib = _lib.load()
    base = (ctypes.c_int32 * 2)(0, 1)
    grads = (ctypes.c_void_p * 1)(0x1000)
    good = [FAKE, FAKE, FAKE, base, 1, grads, _lib.DTYPE_BF16, 32, 0, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, FAKE, None]

    def call(**at):
        a = list(good)
        for k, v in at.items():
            a[int(k[1:])] = v
        return lib.kmoe_adamw(*a)
    for i in (0, 1, 2, 3, 5, 15):
        assert call(**{f"a{i}": None}) == -1
    assert call(a4=-1) == -2 and call(a4=0) == 0
    assert call(a6=_lib.DTYPE_FP8_E4M3) == -3
    assert call(a7=16) == -6
    assert call(a6=_lib.DTYPE_F32, a8=1) == -6
    assert call(a11=1.0) == -2 and call(a12=-0.5) == -2 and call(a13=-1.0) == -2 and call(a14=-1.0) == -2
    assert call(a3=(ctypes.c_int32 * 2)(2, 1)) == -2
    assert call(a5=(ctypes.c_void_p * 1)(None)) == 0  # nothing has a gradient: nothing runs


# ---------------------------------------------------------------- what a step is given
class OnGpu(torch.nn.Parameter):
    """A parameter that says it is on a GPU, for the host's part of a step."""
    is_cuda = True


@pytest.fixture
def steps(monkeypatch):
    """The tensors that each native call of a step gets: [(address of p, of its first moment, values, of its
    gradient), ...] of those with a gradient.  Nothing runs."""
    import contextlib

    from kmoe import optim
    calls = []

    def call(name, table, owner, base, base_host, n, grads, *rest):
        rows = torch.frombuffer((ctypes.c_int64 * (8 * n)).from_address(table), dtype=torch.int64).view(n, 8).tolist()
        calls.append([(r[0], r[1], r[7], g) for r, g in zip(rows, list(grads)[:n]) if g])
    monkeypatch.setattr(optim._lib, "call", call)
    monkeypatch.setattr(optim._lib, "stream_ptr", lambda d=None: 0)
    monkeypatch.setattr(optim, "_device", lambda d: contextlib.nullcontext())
    return calls


def _on_gpu(*sizes, dtype=torch.float32):
    ps = [OnGpu(torch.randn(n).to(dtype)) for n in sizes]
    for p in ps:
        p.grad = torch.ones_like(p.detach())
    return ps


def _want(opt, *ps):
    return [(p.data_ptr(), opt.state[p]["exp_avg"].data_ptr(), p.numel(), p.grad.data_ptr()) for p in ps]


def test_a_step_takes_the_present_states(steps):
    """States that a program clears or replaces, whole or a tensor of them."""
    a, b = _on_gpu(5, 300)
    opt = kmoe.AdamW([a, b])
    opt.step()
    plans = opt._plans
    opt.step()
    assert opt._plans is plans and steps[0] == steps[1] == _want(opt, a, b)  # made once
    old = opt.state[a]
    opt.state.clear()
    opt.step()
    assert opt.state[a] is not old and steps[-1] == _want(opt, a, b) and set(opt.state_dict()["state"]) == {0, 1}
    import collections
    opt.state = collections.defaultdict(dict)
    opt.step()
    assert steps[-1] == _want(opt, a, b)
    opt.state[b] = {k: v.clone() for k, v in opt.state[b].items()}
    opt.step()
    assert steps[-1] == _want(opt, a, b)
    opt.state[b]["exp_avg"] = torch.ones(300)
    opt.step()
    assert steps[-1] == _want(opt, a, b)
    opt.state[b]["exp_avg"] = torch.ones(299)
    with pytest.raises(ValueError, match="the state exp_avg"):
        opt.step()


def test_a_step_takes_the_present_parameters(steps):
    """Parameters that a program replaces in their group, or gives other memory."""
    a, b, c = _on_gpu(5, 300, 300)
    opt = kmoe.AdamW([a, b])
    opt.step()
    opt.param_groups[0]["params"][1] = c
    opt.step()
    assert steps[-1] == _want(opt, a, c)
    opt.param_groups[0]["params"] = [c, a]
    opt.step()
    assert steps[-1] == _want(opt, c, a)
    n = len(steps)
    for shorter in (lambda t: t[:3], lambda t: t.view(15, 20).t()):
        (q,) = _on_gpu(300)
        opt = kmoe.AdamW([q])
        opt.step()
        q.grad = None
        q.data = shorter(q.data)  # the same address
        q.grad = torch.ones_like(q.detach())
        with pytest.raises(ValueError, match="kmoe.AdamW"):
            opt.step()
    assert len(steps) == n + 2  # (the first step of each)


def test_a_parameter_without_a_state_or_gradient_is_left(steps):
    a, b = _on_gpu(5, 300)
    opt = kmoe.AdamW([a, b])
    opt.step()
    del opt.state[b]
    b.grad = None
    opt.step()
    assert steps[-1] == _want(opt, a) and b not in opt.state
    b.grad = torch.ones(300)
    opt.step()
    assert steps[-1] == _want(opt, a, b)


def test_a_refused_parameter_stays_refused(steps):
    a, b = _on_gpu(5, 300)
    b.grad = None
    opt = kmoe.AdamW([a, b])
    opt.step()
    b.is_cuda = False
    b.grad = torch.ones(300)
    for _ in range(2):
        with pytest.raises(ValueError, match="on a GPU"):
            opt.step()
    assert len(steps) == 1


@pytest.mark.parametrize("how", ["deepcopy", "pickle", "state_dict", "weights_after"])
def test_master_weights_outlive_a_copy(steps, how):
    """The f32 copies of a copied, unpickled or reloaded optimizer keep the bits that bf16 lacks; what was
    written since is taken over."""
    import copy
    import io
    (p,) = _on_gpu(5, dtype=torch.bfloat16)
    opt = kmoe.AdamW([p], master_weights=True)
    opt.step()
    fine = torch.tensor([1.0010, -2.003, 0.5, 3.01, 0.0])
    opt.state[p]["master"].copy_(fine)
    with torch.no_grad():
        p.copy_(fine)
    opt._seen[p] = p._version  # as after a step
    if how == "deepcopy":
        opt = copy.deepcopy(opt)
    elif how == "pickle":
        buf = io.BytesIO()
        torch.save(opt, buf)
        buf.seek(0)
        opt = torch.load(buf, weights_only=False)
    else:
        (q,) = _on_gpu(5, dtype=torch.bfloat16)
        other = kmoe.AdamW([q], master_weights=True)
        with torch.no_grad():
            if how == "state_dict":
                q.copy_(p)
                other.load_state_dict(opt.state_dict())
            else:  # the weights after the states
                other.load_state_dict(opt.state_dict())
                q.copy_(p)
        opt = other
    (q,) = opt.param_groups[0]["params"]
    if not getattr(q, "is_cuda"):
        q = OnGpu(q.detach())
        st = opt.state.pop(opt.param_groups[0]["params"][0])
        opt.param_groups[0]["params"][0] = q
        opt.state[q] = st
    q.grad = torch.ones_like(q.detach())
    opt.step()
    assert torch.equal(opt.state[q]["master"], fine)
    with torch.no_grad():
        q[3] = 7.0
        q[4] = float("nan")
    opt.step()
    got = opt.state[q]["master"]
    assert torch.equal(got[:3], fine[:3]) and float(got[3]) == 7.0 and bool(got[4].isnan())


@pytest.mark.parametrize("group,match", [
    (dict(params=[_param(4, dtype=torch.float16)]), "bf16 or f32"), (dict(params=[_param(4), torch.nn.Parameter(torch.zeros(4, 6).t())]), "contiguous"),
    (dict(params=[_param(4)], state_bits=4), "state_bits"), (dict(params=[_param(4)], betas=(0.9, 1.0)), "betas"),
    (dict(params=[_param(4)], lr=-1.0), "lr=-1"), (dict(params=[_param(4)], lr=float("nan")), "lr=nan")])
def test_a_refused_group_does_not_join(group, match):
    opt = kmoe.AdamW([_param(4)])
    good = opt.param_groups[0]
    for _ in range(2):
        with pytest.raises(ValueError, match=match):
            opt.add_param_group(dict(group))
        assert len(opt.param_groups) == 1 and opt.param_groups[0] is good
    opt.add_param_group({"params": [_param(4)], "lr": torch.tensor(0.1)})
    assert len(opt.param_groups) == 2


@pytest.mark.filterwarnings("ignore:optimizer contains")
def test_parameters_that_share_memory_are_refused(steps):
    """Their values would be stepped by two workgroups at once."""
    p = _param(40)
    with pytest.raises(ValueError, match="twice"):
        kmoe.AdamW([p, p])
    opt = kmoe.AdamW([_param(4)])
    with pytest.raises(ValueError, match="twice"):
        opt.add_param_group({"params": [p, _param(3), p]})
    assert len(opt.param_groups) == 1
    buf = torch.zeros(100)
    for cut in ((0, 40, 39, 100), (0, 100, 40, 60), (50, 60, 0, 51)):
        ps = [OnGpu(buf[cut[0]:cut[1]]), OnGpu(buf[cut[2]:cut[3]])]
        for q in ps:
            q.grad = torch.ones_like(q.detach())
        opt = kmoe.AdamW(ps)
        for _ in range(2):
            with pytest.raises(ValueError, match="share memory"):
                opt.step()
        n = len(steps)
        kmoe.AdamW([{"params": [q]} for q in ps]).step()  # groups are stepped one after the other
        assert len(steps) == n + 2
    a, b = _on_gpu(5, 300)
    opt = kmoe.AdamW([a, b])
    m = torch.zeros(305)
    for q, at in ((a, m[:5]), (b, m[4:304])):
        opt.set_state(q, 1, exp_avg=at, exp_avg_sq=torch.zeros(q.numel()))
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    n = len(steps)
    ps = [OnGpu(buf[:40]), OnGpu(buf[:0]), OnGpu(buf[40:]), OnGpu(torch.zeros(0))]
    for q in ps:
        q.grad = torch.ones_like(q.detach())
    kmoe.AdamW(ps).step()
    assert len(steps) == n + 1


def test_what_captured_steps_read_outlives_a_load(steps, monkeypatch):
    """Loading a state dict takes states and tables away from later steps, not from the graphs of earlier ones."""
    a, b = _on_gpu(5, 300)
    opt = kmoe.AdamW([a, b])
    opt.step()
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_available", lambda: True)
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        opt.step()
    (plan,) = [p for _, p in opt._plans]
    held = list(opt._held)
    assert any(x is plan for x in held[0])
    opt.load_state_dict(opt.state_dict())
    assert len(opt._held) == len(held) and all(x is y for x, y in zip(opt._held, held))
    opt.step()
    assert all(p is not plan for _, p in opt._plans) and steps[-1] == _want(opt, a, b)


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_state_dict_changes_nothing(bits):
    """One of another form, or of torch's own AdamW."""
    ps = [_param(3, 100), _param(7)]
    opt = kmoe.AdamW(ps, lr=0.5, state_bits=bits)
    for p in ps:
        st = opt._new_state(p, opt.param_groups[0])
        opt.set_state(p, 5, **{k: v for k, v in st.items() if k != "step"})
    states, groups = [opt.state[p] for p in ps], opt.param_groups
    qs = [torch.nn.Parameter(p.detach().float()) for p in ps]
    other = torch.optim.AdamW(qs, lr=0.25)
    for q in qs:
        q.grad = torch.ones_like(q)
    other.step()
    wrong = kmoe.AdamW([_param(3, 100), _param(8)], state_bits=bits)
    for p in wrong.param_groups[0]["params"]:
        st = wrong._new_state(p, wrong.param_groups[0])
        wrong.set_state(p, 5, **{k: v for k, v in st.items() if k != "step"})
    bad = opt.state_dict()
    bad["state"] = {0: bad["state"][0], 1: {**bad["state"][1], "exp_avg": None}}
    number = opt.state_dict()
    number["state"] = {**number["state"], 1: {**number["state"][1], "step": 5}}
    for sd, match in ((other.state_dict(), "state_bits"), (wrong.state_dict(), "the state exp_avg"), (bad, "the state exp_avg"),
                      (number, "the state step")):
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(sd)
        assert opt.param_groups is groups and groups[0]["lr"] == 0.5 and set(opt.state) == set(ps)
        assert all(opt.state[p] is st and st["exp_avg"].dtype == (torch.uint8 if bits == 8 else torch.float32)
                   for p, st in zip(ps, states))


def test_values_of_no_state():
    p = _param(5)
    opt = kmoe.AdamW([p])
    with pytest.raises(ValueError, match="no state"):
        opt.state_values(p)
    with pytest.raises(ValueError, match="not a parameter"):
        opt.state_values(_param(5))
    assert not opt.state


def test_states_of_another_form_are_refused(steps):
    """Entries that the kernel would take for another form of states than the group's; a program's own entries
    are left alone."""
    f32 = lambda n: torch.zeros(n)
    for bits, extra in ((32, dict(exp_avg_scale=f32(1))), (32, dict(exp_avg_sq_scale=f32(2))), (32, dict(master=f32(300))),
                        (8, dict(master=f32(300)))):
        (p,) = _on_gpu(300, dtype=torch.bfloat16)
        opt = kmoe.AdamW([p], state_bits=bits)
        good = {k: v for k, v in opt._new_state(p, opt.param_groups[0]).items() if k != "step"}
        with pytest.raises(ValueError, match="has no"):
            opt.set_state(p, 1, **good, **extra)
        assert p not in opt.state
        opt.step()
        opt.state[p] = {**opt.state[p], **extra}
        with pytest.raises(ValueError, match="has no"):
            opt.step()
        sd = opt.state_dict()
        other = kmoe.AdamW([_param(300)], state_bits=bits)
        with pytest.raises(ValueError, match="has no"):
            other.load_state_dict(sd)
        assert not other.state
    for key, value in (("state_bits", 8), ("master_weights", True)):
        (p,) = _on_gpu(300, dtype=torch.bfloat16)
        opt = kmoe.AdamW([p])
        opt.step()
        opt.param_groups[0][key] = value
        with pytest.raises(ValueError, match="the state"):
            opt.step()
    a, b = _on_gpu(5, 300)
    opt = kmoe.AdamW([a, b])
    opt.step()
    opt.state[a]["note"], opt.state[b]["mean"] = "mine", torch.ones(7)
    opt.step()
    plans = opt._plans
    opt.state[b]["mean"] = torch.zeros(9)
    opt.step()
    assert opt._plans is plans and steps[-1] == _want(opt, a, b)
    other = kmoe.AdamW(_on_gpu(5, 300))
    other.load_state_dict(opt.state_dict())
    q, r = other.param_groups[0]["params"]
    assert other.state[q]["note"] == "mine" and torch.equal(other.state[r]["mean"], torch.zeros(9))
