"""kmoe.AdamW on the GPU against its formulas in 64 bits, and its 8-bit codes bit for bit against
the same formulas in separate f32 operations."""
import copy

import pytest
import torch

import kmoe

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of f32, relative to the value
HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _decode(st, n):
    """(m, v) in f64 that the states stand for."""
    if "exp_avg_scale" not in st:
        return st["exp_avg"].double().view(-1).cpu(), st["exp_avg_sq"].double().view(-1).cpu()
    rep = lambda s: s.cpu().double().repeat_interleave(256)[:n]
    m = st["exp_avg"].cpu().view(torch.float8_e4m3fn).double() * rep(st["exp_avg_scale"])
    c = st["exp_avg_sq"].cpu().int()
    root = torch.where(c >= 16, (16 + c % 16).double() * torch.exp2((c // 16 - 19).double()), c.double() * 2.0 ** -18)
    return m, (root * rep(st["exp_avg_sq_scale"])) ** 2


def _codes32(m, v, g, b1, b2):
    """The codes and scales after one step, in f32 operations one by one, on the CPU.  m, v: f32."""
    m = b1 * m + (1.0 - b1) * g
    v = b2 * v + ((1.0 - b2) * g) * g
    # (from 64 bits, whose rounding to f32 is that of the exact root; the CPU's f32 root is not always)
    root = torch.sqrt(v.double()).float()
    blocks = lambda t: torch.nn.functional.pad(t, (0, -t.numel() % 256)).view(-1, 256)
    bm, br = blocks(m), blocks(root)
    sm, sv = bm.abs().amax(1) * (1.0 / 448.0), br.amax(1) * (1.0 / 1.9375)
    sm = torch.where(sm >= 2.0 ** -100, sm, 0.0)
    inv = lambda s: torch.where(s > 0, 1.0 / torch.where(s > 0, s, 1.0), 0.0)[:, None]
    qm = (bm * inv(sm)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    q = (br * inv(sv)).clamp(max=1.9375)
    e = torch.where(q > 0, torch.frexp(q).exponent - 1, -14).clamp(min=-14)
    qv = torch.round(torch.ldexp(q, 4 - e)).int() + (e + 14) * 16
    qv = torch.where((qv == 0) & (br > 0), 1, qv).to(torch.uint8)
    n = m.numel()
    return qm.view(-1)[:n], sm, qv.view(-1)[:n], sv


def _tensors(dev, shapes, dtype, seed=0, gstd=1e-3):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter(torch.randn(*s, generator=g).mul(0.02).to(dtype).to(dev)) for s in shapes]
    gs = [torch.randn(*s, generator=g).mul(gstd).to(dtype).to(dev) for s in shapes]
    return ps, gs


def _check_step(p_old, m, v, g, t, hp, p, st, dtype, bits, master=None):
    """p and the states after step t from (p_old, m, v, g) in f64, within the sum of the roundings."""
    b1, b2 = hp["betas"]
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    den = (v1 / (1 - b2 ** t)).sqrt() + hp["eps"]
    step = hp["lr"] / (1 - b1 ** t)
    want = p_old * (1 - hp["lr"] * hp["weight_decay"]) - step * m1 / den
    # m: constant, product and sum round, relative to the terms; v the same with a product more;
    # the update: its factor, root, product with 1/sqrt(1 - b2^t), sum with eps, reciprocal (a
    # whole step), two products; the weight: its factor, product and sum
    am = b1 * m.abs() + (1 - b1) * g.abs()
    e_m, e_v = 3 * U * am, 4 * U * v1
    e_p = 3 * U * p_old.abs() + 2 * U * want.abs() + step / den * (e_m + (2 + 1 + 1 + 1 + 2 + 2 + 2) * U * am)
    if dtype == torch.bfloat16 and master is None:
        e_p = e_p + 2.0 ** -8 * want.abs()
    got = (p if master is None else master).detach().double().view(-1).cpu()
    assert bool(((got - want).abs() <= e_p * 1.001 + 1e-38).all()), float(((got - want).abs() - e_p).max())
    if master is not None:
        assert torch.equal(p.detach().view(-1).cpu(), master.view(-1).cpu().to(torch.bfloat16))
    gm, gv = _decode(st, m.numel())
    if bits == 32:
        assert bool(((gm - m1).abs() <= e_m + 1e-45).all()) and bool(((gv - v1).abs() <= e_v + 1e-45).all())
    else:
        rep = lambda s: s.cpu().double().repeat_interleave(256)[:m.numel()]
        # half a step of the code (relative, or of the smallest exponent), the never-zero rule of the
        # root, and f32's: the scale, its reciprocal and the product round
        root, sm, sv = v1.sqrt(), rep(st["exp_avg_scale"]), rep(st["exp_avg_sq_scale"])
        assert bool(((gm - m1).abs() <= 2.0 ** -4 * m1.abs() + 2.0 ** -10 * sm + e_m + 4 * U * m1.abs()).all())
        assert bool(((gv.sqrt() - root).abs() <= 2.0 ** -5 * root + 2.0 ** -18 * sv + 8 * U * root).all())
        assert bool(((gv > 0) | (v1 == 0)).all())


SHAPES = [(1,), (255,), (256,), (257,), (3, 5, 7), (64, 130), (8192,), (8193,), (40, 1000), (0,), (2, 9000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True], ids=["", "master"])
def test_steps(dev, dtype, bits, master):
    ps, gs = _tensors(dev, SHAPES, dtype)
    opt = kmoe.AdamW(ps, state_bits=bits, master_weights=master, **HYPER)
    has = master and dtype == torch.bfloat16
    cur = [(p.detach().double().view(-1).cpu(), torch.zeros(p.numel(), dtype=torch.float64),
            torch.zeros(p.numel(), dtype=torch.float64)) for p in ps]
    for t in range(1, 5):
        for p, g in zip(ps, gs):
            p.grad = g * t
        before = [(p.detach().double().view(-1).cpu() if not (has and t > 1) else
                   opt.state[p]["master"].double().view(-1).cpu()) for p in ps]
        opt.step()
        for i, p in enumerate(ps):
            st = opt.state[p]
            if p.numel():
                assert int(st["step"]) == t
            _check_step(before[i], cur[i][1], cur[i][2], p.grad.double().view(-1).cpu(), t, HYPER, p, st, dtype, bits,
                        st.get("master"))
            cur[i] = (None, *_decode(st, p.numel()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_codes_bit_for_bit(dev, dtype):
    n = 100003
    gen = torch.Generator().manual_seed(1)
    (p,), _ = _tensors(dev, [(n,)], dtype)
    opt = kmoe.AdamW([p], state_bits=8, **HYPER)
    m, v = torch.zeros(n), torch.zeros(n)
    for t in range(6):
        # magnitudes over many powers of two, some zeros, a block of zeros
        g = torch.randn(n, generator=gen) * torch.exp2(torch.randint(-30, 4, (n,), generator=gen).float())
        g[torch.rand(n, generator=gen) < 0.1] = 0.0
        g[512:768] = 0.0
        p.grad = g.to(dtype).to(dev)
        opt.step()
        cm, sm, cv, sv = _codes32(m, v, p.grad.float().cpu(), *HYPER["betas"])
        st = {k: x.cpu() for k, x in opt.state[p].items()}
        assert torch.equal(st["exp_avg_scale"], sm) and torch.equal(st["exp_avg_sq_scale"], sv)
        assert torch.equal(st["exp_avg"], cm) and torch.equal(st["exp_avg_sq"], cv)
        m, r = (x.cpu() for x in opt.state_values(p))
        v = r * r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_values_of_codes(dev, dtype):
    """Every code's number, from the definition."""
    p = torch.nn.Parameter(torch.zeros(515, device=dev))
    opt = kmoe.AdamW([p], state_bits=8)
    codes = (torch.arange(515) % 256).to(torch.uint8)
    scale = torch.tensor([2.0, 0.75, 0.3])
    opt.set_state(p, 0, exp_avg=codes.to(dev), exp_avg_scale=scale.to(dev), exp_avg_sq=codes.to(dev),
                  exp_avg_sq_scale=scale.to(dev))
    m, root = (t.cpu() for t in opt.state_values(p, dtype))
    rep = scale.repeat_interleave(256)[:515]
    want = torch.tensor([(16 + c % 16) * 2.0 ** (c // 16 - 19) if c >= 16 else c * 2.0 ** -18 for c in codes.tolist()])
    assert torch.equal(root, (want * rep).to(dtype))
    assert torch.equal(m.nan_to_num(9.0), (codes.view(torch.float8_e4m3fn).float() * rep).to(dtype).nan_to_num(9.0))
    q = torch.nn.Parameter(torch.zeros(4, 3, device=dev))
    opt = kmoe.AdamW([q])
    q.grad = torch.ones_like(q)
    opt.step()
    assert all(t.shape == q.shape and t.dtype == dtype for t in opt.state_values(q, dtype))


@pytest.mark.parametrize("bits", [32, 8])
def test_no_gradient_leaves_a_tensor(dev, bits):
    ps, gs = _tensors(dev, [(300,), (400,), (500,)], torch.bfloat16)
    opt = kmoe.AdamW(ps, state_bits=bits, **HYPER)
    ps[0].grad, ps[2].grad = gs[0], gs[2]
    opt.step()
    opt.step()
    assert ps[1] not in opt.state and [int(opt.state[p]["step"]) for p in (ps[0], ps[2])] == [2, 2]
    old = ps[0].detach().clone()
    ps[0].grad, ps[1].grad = None, gs[1]
    opt.step()
    assert torch.equal(ps[0], old) and [int(opt.state[p]["step"]) for p in ps] == [2, 1, 3]


def test_many_tensors_and_groups(dev):
    """More tensors than one launch holds, in two groups, as one tensor each would do it."""
    n = 600
    ps, gs = _tensors(dev, [(1 + 37 * i % 900,) for i in range(n)], torch.bfloat16)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt = kmoe.AdamW([{"params": ps[:250], "lr": 1e-3}, {"params": ps[250:], "weight_decay": 0.0}], state_bits=8, **HYPER)
    for p, g in zip(ps, gs):
        p.grad = g
    opt.step()
    for i in (0, 1, 249, 250, 400, 599):
        one = kmoe.AdamW([qs[i]], state_bits=8, **{**HYPER, **({"lr": 1e-3} if i < 250 else {"weight_decay": 0.0})})
        qs[i].grad = gs[i]
        one.step()
        assert torch.equal(ps[i], qs[i])
    assert all(int(opt.state[p]["step"]) == 1 for p in ps)


def test_misaligned_and_strided(dev):
    """Parameters inside one buffer at odd places, a gradient that is not contiguous."""
    buf = torch.randn(5000, device=dev).to(torch.bfloat16)
    p = torch.nn.Parameter(buf[3:3 + 40 * 30].view(40, 30))
    guard = buf.clone()
    q = torch.nn.Parameter(p.detach().clone())
    g = torch.randn(30, 40, device=dev).to(torch.bfloat16).t()
    for bits in (32, 8):
        a, b = kmoe.AdamW([p], state_bits=bits, **HYPER), kmoe.AdamW([q], state_bits=bits, **HYPER)
        p.grad, q.grad = g, g.contiguous()
        a.step()
        b.step()
        assert torch.equal(p, q)
    assert torch.equal(buf[:3], guard[:3]) and torch.equal(buf[3 + 1200:], guard[3 + 1200:])


def test_infinite_gradient_shows(dev):
    p = torch.nn.Parameter(torch.ones(1000, device=dev))
    opt = kmoe.AdamW([p], state_bits=8, **HYPER)
    p.grad = torch.full((1000,), 1e-3, device=dev)
    opt.step()
    p.grad[300] = float("inf")
    opt.step()
    m, v = opt.state_values(p)
    bad = torch.zeros(1000, dtype=torch.bool, device=dev)
    bad[256:512] = True
    assert torch.equal(m.isnan(), bad) and torch.equal(v.isnan(), bad)
    assert bool(torch.isfinite(p[~bad]).all())


def test_versions_and_master(dev):
    """A step counts as a change of the weights; a write of them by others renews the f32 copy."""
    ps, gs = _tensors(dev, [(100,)], torch.bfloat16)
    opt = kmoe.AdamW(ps, master_weights=True, **HYPER)
    ps[0].grad = gs[0]
    v0 = ps[0]._version
    opt.step()
    assert ps[0]._version > v0
    with torch.no_grad():
        ps[0].fill_(2.0)
    opt.step()
    m = opt.state[ps[0]]["master"]
    assert bool(((m - 2.0).abs() < 0.1).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(dev, bits):
    """Replays count, follow a learning rate on the GPU, and are the eager steps bit for bit."""
    ps, gs = _tensors(dev, [(5000,), (33, 77)], torch.bfloat16)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    lr = torch.tensor(1e-2, device=dev)
    lr2 = lr.clone()
    hp = {k: v for k, v in HYPER.items() if k != "lr"}
    a, b = kmoe.AdamW(ps, lr=lr, state_bits=bits, **hp), kmoe.AdamW(qs, lr=lr2, state_bits=bits, **hp)
    for p, q, g in zip(ps, qs, gs):
        p.grad, q.grad = g.clone(), g.clone()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            a.step()
    a.step()
    b.step()
    with torch.cuda.graph(graph):
        a.step()
    for t in range(2, 6):
        for p, q in zip(ps, qs):
            p.grad.mul_(-1.5)
            q.grad.mul_(-1.5)
        lr.mul_(0.5)
        lr2.mul_(0.5)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and int(a.state[p]["step"]) == int(b.state[q]["step"]) == t
    # another plan (a third tensor) does not take the captured one's tables away
    extra = torch.nn.Parameter(torch.zeros(10, device=dev))
    a.add_param_group({"params": [extra]})
    extra.grad = torch.ones_like(extra)
    a.step()
    b.step()
    graph.replay()
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_state_dict_resumes(dev):
    ps, gs = _tensors(dev, [(1000,)], torch.bfloat16)
    opt = kmoe.AdamW(ps, state_bits=8, master_weights=True, **HYPER)
    ps[0].grad = gs[0]
    opt.step()
    sd, w = copy.deepcopy(opt.state_dict()), ps[0].detach().clone()
    opt.step()
    q = torch.nn.Parameter(w)
    other = kmoe.AdamW([q], state_bits=8, master_weights=True, **HYPER)
    other.load_state_dict(sd)
    q.grad = gs[0]
    other.step()
    assert torch.equal(q, ps[0]) and torch.equal(other.state[q]["master"], opt.state[ps[0]]["master"])


def test_against_torch(dev):
    """torch.optim.AdamW in f64 on the same gradients, 20 steps."""
    ps, _ = _tensors(dev, [(4000,)], torch.float32)
    r = torch.nn.Parameter(ps[0].detach().double())
    a, b = kmoe.AdamW(ps, **HYPER), torch.optim.AdamW([r], **HYPER)
    gen = torch.Generator().manual_seed(2)
    for _ in range(20):
        g = torch.randn(4000, generator=gen).to(dev)
        ps[0].grad, r.grad = g, g.double()
        a.step()
        b.step()
    # a step moves a weight by at most about lr (1 + wd |p|) and is off by some 20 roundings of f32
    assert float((ps[0].double() - r).abs().max()) <= 20 * (20 * U * 1e-2 * 3 + 4 * U * 0.3)


def test_refusals(dev):
    p = torch.nn.Parameter(torch.zeros(4, device=dev))
    opt = kmoe.AdamW([p], lr=torch.zeros(2, device=dev))
    p.grad = torch.zeros(4, device=dev)
    with pytest.raises(ValueError, match="one f32 value"):
        opt.step()
    q = torch.nn.Parameter(torch.zeros(4, device=dev, dtype=torch.bfloat16))
    opt = kmoe.AdamW([q])
    q.grad = torch.zeros(4, device=dev, dtype=torch.bfloat16).to_sparse()
    with pytest.raises(ValueError, match="dense"):
        opt.step()


def test_replaced_states_and_parameters(dev):
    """A cleared state starts anew, a replaced parameter is stepped, a parameter of fewer values in the same
    place is refused."""
    ps, gs = _tensors(dev, [(300,), (1000,), (1000,)], torch.float32)
    p, q, r = ps
    for t, g in zip(ps, gs):
        t.grad = g
    start = [t.detach().clone() for t in ps]
    opt = kmoe.AdamW([p, q], **HYPER)
    opt.step()
    first = [t.detach().clone() for t in ps]
    opt.step()
    opt.state.clear()
    with torch.no_grad():
        for t, s in zip(ps, start):
            t.copy_(s)
    opt.step()
    assert torch.equal(p, first[0]) and torch.equal(q, first[1]) and int(opt.state[p]["step"]) == 1
    opt.param_groups[0]["params"][1] = r
    with torch.no_grad():
        r.copy_(start[1])
    r.grad = q.grad
    opt.step()
    assert torch.equal(r, first[1]) and torch.equal(q, first[1]) and int(opt.state[p]["step"]) == 2
    guard = r.detach().clone()
    r.grad = None
    r.data = r.data[:400]
    r.grad = gs[0].new_ones(400)
    with pytest.raises(ValueError, match="the state"):
        opt.step()
    assert torch.equal(r.data.as_strided((1000,), (1,)), guard)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copied_optimizer_goes_on(dev, bits):
    """Steps of a copy with f32 weights are the original's, bit for bit."""
    ps, gs = _tensors(dev, [(300,), (40, 25)], torch.bfloat16)
    opt = kmoe.AdamW(ps, state_bits=bits, master_weights=True, **HYPER)
    for t in range(3):
        for p, g in zip(ps, gs):
            p.grad = g * (t + 1)
        opt.step()
    qs, other = copy.deepcopy((ps, opt))
    assert all(a is b for a, b in zip(qs, other.param_groups[0]["params"]))
    for t in range(3):
        for p, q, g in zip(ps, qs, gs):
            p.grad, q.grad = g * -t, g * -t
        opt.step()
        other.step()
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and torch.equal(opt.state[p]["master"], other.state[q]["master"])
            assert not torch.equal(opt.state[p]["master"], p.detach().float())


def test_groups_of_empty_parameters(dev):
    """Nothing to step is no error."""
    e, p = torch.nn.Parameter(torch.zeros(0, 5, device=dev)), torch.nn.Parameter(torch.ones(3, device=dev))
    e.grad, p.grad = torch.zeros_like(e), torch.ones_like(p)
    for bits in (32, 8):
        opt = kmoe.AdamW([{"params": [e]}, {"params": [p]}], state_bits=bits, **HYPER)
        opt.step()
        opt.step()
        assert int(opt.state[p]["step"]) == 2 and all(t.numel() == 0 for t in opt.state_values(e))


def test_a_captured_step_keeps_its_learning_rate(dev):
    """A rate on the GPU that the program drops or replaces after the capture is not read from freed memory."""
    (p,), (g,) = _tensors(dev, [(300,)], torch.float32)
    q = torch.nn.Parameter(p.detach().clone())
    p.grad, q.grad = g, g.clone()
    hp = {k: v for k, v in HYPER.items() if k != "lr"}
    opt = kmoe.AdamW([{"params": [p], "lr": torch.full((), 1e-2, device=dev)}], **hp)
    eager = kmoe.AdamW([q], lr=1e-2, **hp)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    other = [torch.full((), 7.0, device=dev) for _ in range(64)]  # where the old one was, if it was freed
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for _ in range(3):
        eager.step()
    assert torch.equal(p, q) and len(other) == 64


def test_a_captured_step_keeps_its_memory(dev):
    """Replays after a parameter or its states were given other memory write what they were captured with, not
    what has come there since."""
    (p,), (g,) = _tensors(dev, [(3000,)], torch.float32)
    p.grad = g
    opt = kmoe.AdamW([p], **HYPER)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    p.data = p.data.clone()
    opt.state[p] = {k: v.clone() for k, v in opt.state[p].items()}
    opt.step()  # with tables of its own
    kept = p.detach().clone()
    other = [torch.full((3000,), 7.0, device=dev) for _ in range(64)]
    step = int(opt.state[p]["step"])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(p, kept) and int(opt.state[p]["step"]) == step
    assert all(bool((t == 7.0).all()) for t in other)


def test_replays_after_a_load(dev):
    """A step captured before load_state_dict still writes the parameters, with the states that it was captured with."""
    (p,), (g,) = _tensors(dev, [(3000,)], torch.float32)
    q = torch.nn.Parameter(p.detach().clone())
    p.grad, q.grad = g, g.clone()
    opt, eager = kmoe.AdamW([p], **HYPER), kmoe.AdamW([q], **HYPER)
    opt.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.load_state_dict(opt.state_dict())
    other = [torch.full((n,), 7.0, device=dev) for n in (1, 16, 3000) * 30]
    for _ in range(2):
        graph.replay()
        eager.step()
    torch.cuda.synchronize()
    assert torch.equal(p, q) and all(bool((t == 7.0).all()) for t in other)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_past_32_bits(dev, bits):
    """More than 2^31 values: the first, the middle and the last ones are stepped as a small tensor of theirs is."""
    n, part = (1 << 31) + 1234 * 256 + 77, 256 * 40
    gen = torch.Generator(device=dev).manual_seed(3)
    p = torch.nn.Parameter(torch.empty(n, device=dev, dtype=torch.bfloat16).normal_(0.0, 0.02, generator=gen))
    p.grad = torch.empty(n, device=dev, dtype=torch.bfloat16).normal_(0.0, 1e-3, generator=gen)
    cuts = [slice(0, part), slice((1 << 31) - part, (1 << 31) + part), slice((n - part) // 256 * 256, n)]
    qs = [torch.nn.Parameter(p.detach()[c].clone()) for c in cuts]
    opt, small = kmoe.AdamW([p], state_bits=bits, **HYPER), kmoe.AdamW(qs, state_bits=bits, **HYPER)
    for t in range(2):
        for q, c in zip(qs, cuts):
            q.grad = p.grad[c].clone()
        opt.step()
        small.step()
    m, root = (opt.state_values(p, torch.bfloat16))
    for q, c in zip(qs, cuts):
        assert torch.equal(p.detach()[c], q.detach())
        assert all(torch.equal(a[c], b) for a, b in zip((m, root), small.state_values(q, torch.bfloat16)))
    assert int(opt.state[p]["step"]) == 2
