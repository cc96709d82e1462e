"""CPU tests of the routing, add-norm and microscaled entry points: sizes, refusals (no kernel
is launched), configuration checks, and the 64-bit restatements against differences."""
import ctypes

import pytest
import torch

import kmoe
from kmoe import _lib, ops
from oracle import mx_oracle as M

NULL, FAKE = None, ctypes.c_void_p(0x1000)  # FAKE is never read: validation fails first
E4, E2 = _lib.DTYPE_FP8_E4M3, _lib.DTYPE_FP4_E2M1


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def rc(lib, name, *args):
    return getattr(lib, name)(*args), lib.kmoe_last_error().decode()


def test_sizes(lib):
    assert lib.kmoe_mx_row_bytes(2048, E4) == 2048 and lib.kmoe_mx_row_bytes(192, E2) == 128
    assert lib.kmoe_mx_row_bytes(64, 0) == 0 and lib.kmoe_mx_row_bytes(0, E4) == 0
    assert lib.kmoe_mx_scale_bytes(2048) == 64 and lib.kmoe_mx_scale_bytes(96) == 16
    # half a byte a weight, one scale byte for 32
    assert lib.kmoe_packed_mx_bytes(16, 2048, 2816, 0) == 16 * 2 * 2816 * 2048 // 2
    assert lib.kmoe_packed_mx_bytes(16, 2048, 2816, 1) == 16 * 2 * 2816 * 2048 // 32
    assert lib.kmoe_packed_mx_bytes(2, 64, 100, 0) == 2 * 256 * 128 // 2
    assert lib.kmoe_packed_mx_bytes(2, 64, 100, 3) == 2 * 256 * 128 // 32
    assert lib.kmoe_packed_mx_bytes(2, 65, 100, 0) == 0 and lib.kmoe_packed_mx_bytes(65, 64, 100, 0) == 0


def test_route_refusals(lib):
    def call(T=4, E=16, k=2, scores=0, groups=1, keep=1, top=2, logits=FAKE):
        return rc(lib, "kmoe_route_topk", logits, T, E, k, scores, NULL, groups, keep, top, 1, 1.0, FAKE, FAKE, NULL, NULL)
    assert call(logits=NULL)[0] == -1
    assert call(E=65)[0] == -2 and call(E=0)[0] == -2 and call(T=-1)[0] == -2
    assert call(k=0)[0] == -2 and call(k=9)[0] == -2 and call(E=4, k=5)[0] == -2
    assert call(groups=3)[0] == -2 and call(groups=4, keep=5)[0] == -2 and call(groups=0)[0] == -2
    assert call(groups=4, keep=1, k=5)[0] == -2 and "kept groups" in call(groups=4, keep=1, k=5)[1]
    assert call(top=3)[0] == -2 and call(scores=2)[0] == -6
    assert call(T=0, logits=NULL)[0] == 0
    assert rc(lib, "kmoe_route_topk_bwd", FAKE, FAKE, NULL, 4, 16, 2, 0, 1, 1.0, 0, FAKE, NULL)[0] == -1
    assert rc(lib, "kmoe_route_topk_bwd", FAKE, FAKE, FAKE, 4, 16, 17, 0, 1, 1.0, 0, FAKE, NULL)[0] == -2


def test_add_norm_refusals(lib):
    def call(x=FAKE, xd=0, d=64, fmt=0, q=NULL, eps=1e-5, h=FAKE, delta=FAKE):
        return rc(lib, "kmoe_add_rmsnorm", x, xd, delta, 0, FAKE, 0, eps, 4, d, h, FAKE, FAKE, fmt, q, q, NULL)[0]
    assert call(x=NULL) == -1 and call(h=NULL) == -1
    assert call(xd=2) == -3 and call(fmt=1) == -3
    assert call(fmt=E4) == -1 and call(d=60) == -2 and call(fmt=E4, q=FAKE, d=40) == -2
    assert rc(lib, "kmoe_add_rmsnorm_bwd", FAKE, FAKE, 0, FAKE, 0, FAKE, FAKE, 4, 64, FAKE, FAKE, FAKE, 0, FAKE, 1 << 20,
              NULL)[0] == -3
    assert call(d=8200) == -6 and call(eps=-1.0) == -2 and call(eps=float("nan")) == -2


def test_mx_refusals(lib):
    assert rc(lib, "kmoe_quant_rows_mx", NULL, NULL, 4, NULL, 64, E4, FAKE, FAKE, NULL)[0] == -1
    assert rc(lib, "kmoe_quant_rows_mx", FAKE, NULL, 4, NULL, 64, 0, FAKE, FAKE, NULL)[0] == -3
    assert rc(lib, "kmoe_quant_rows_mx", FAKE, NULL, 4, NULL, 48, E4, FAKE, FAKE, NULL)[0] == -2
    assert rc(lib, "kmoe_quant_rows_mx", FAKE, NULL, 1 << 31, NULL, 64, E4, FAKE, FAKE, NULL)[0] == -2
    assert rc(lib, "kmoe_dequant_rows_mx", FAKE, FAKE, NULL, -1, NULL, 64, E4, FAKE, NULL)[0] == -2
    assert rc(lib, "kmoe_fake_quant_mx_cols", FAKE, E4, 2, 64, 64, FAKE, NULL)[0] == -3
    assert rc(lib, "kmoe_fake_quant_mx_cols", FAKE, 0, 2, 0, 64, FAKE, NULL)[0] == -2
    assert rc(lib, "kmoe_pack_weights_mx", FAKE, FAKE, FAKE, 0, 2, 60, 64, FAKE, FAKE, FAKE, FAKE, NULL)[0] == -2
    assert rc(lib, "kmoe_pack_weights_mx", FAKE, FAKE, FAKE, 0, 2, 64, 64, FAKE, NULL, FAKE, FAKE, NULL)[0] == -1

    def gate_up(fmt=E4, n_x=10, tok=FAKE, E=2, d=64, F=64, rows=4, hq=FAKE):
        return rc(lib, "kmoe_gemm_gate_up_mx", FAKE, FAKE, fmt, n_x, tok, FAKE, E, d, F, rows, FAKE, FAKE, hq, FAKE, NULL, NULL)
    assert gate_up(fmt=0)[0] == -3 and gate_up(E=65)[0] == -2 and gate_up(d=96)[0] == -2 and gate_up(F=0)[0] == -2
    assert gate_up(hq=NULL)[0] == -1 and gate_up(n_x=0)[0] == -2 and gate_up(rows=-1)[0] == -2
    # 2 GiB of gathered rows: the load window's end
    code, msg = gate_up(n_x=1 << 20, d=2048)
    assert code == -2 and "too large" in msg
    # more workgroups than a launch takes
    assert gate_up(rows=(1 << 31) - 1, F=1 << 15)[0] == -2
    assert rc(lib, "kmoe_gemm_down_mx", FAKE, FAKE, E4, FAKE, 2, 64, 64, 4, FAKE, FAKE, NULL, NULL)[0] == -1
    assert rc(lib, "kmoe_gemm_down_mx", FAKE, FAKE, E4, FAKE, 2, 64, 1 << 24, 4, FAKE, FAKE, FAKE, NULL)[0] == -2


def cfg(**kw):
    return kmoe.AdvancedMoEConfig(d_model=128, n_experts=16, d_ff_expert=64, **kw)


def test_configuration_checks():
    with pytest.raises(ValueError, match="moe_mx"):
        kmoe.MoELayer(cfg(moe_mx="w4"))
    with pytest.raises(ValueError, match="exclude"):
        kmoe.MoELayer(cfg(moe_mx="w4a8", moe_fp8=True))
    with pytest.raises(NotImplementedError):
        kmoe.MoELayer(cfg(moe_mx="w4a8", ffn_activation="gelu"))
    with pytest.raises(ValueError, match="groups"):
        kmoe.Router(cfg(moe_router_groups=3))
    with pytest.raises(ValueError, match="kept groups"):
        kmoe.Router(cfg(moe_router_groups=16, moe_top_k=2))
    with pytest.raises(ValueError, match="scores"):
        kmoe.Router(cfg(moe_router_scores="relu"))
    with pytest.raises(ValueError, match="balanced"):
        kmoe.Router(cfg(moe_balanced_routing=True, moe_balance_bias=True))
    with pytest.raises(ValueError, match="token choice"):
        kmoe.MoELayer(cfg(moe_routing="expert_choice", moe_router_scores="sigmoid"))
    assert kmoe.Router(cfg()).spec is None
    assert kmoe.MoELayer(cfg(moe_mx="w4a4")).grouped_experts.mx_act == "e2m1"


def test_balance_bias_keeps_its_type():
    r = kmoe.Router(cfg(moe_balance_bias=True))
    r.balance_bias.fill_(1.0 + 2.0 ** -20)
    r = r.to(torch.bfloat16)
    assert r.router[0].weight.dtype == torch.bfloat16
    assert r.balance_bias.dtype == torch.float32 and float(r.balance_bias[0]) == 1.0 + 2.0 ** -20
    assert r.state_dict()["balance_bias"] is not None
    with torch.device("meta"):
        m = kmoe.Router(cfg(moe_balance_bias=True))
    m = m.to_empty(device="cpu").to(torch.bfloat16)
    assert m.balance_bias.dtype == torch.float32 and not m.balance_bias.is_meta


def test_modules_without_the_new_attributes():
    """Modules pickled before these attributes were there act as they did."""
    ex, router = kmoe.GroupedExperts(2, 64, 64), kmoe.Router(kmoe.AdvancedMoEConfig(d_model=64, n_experts=4))
    ex.__dict__.pop("mx", None)
    router.__dict__.pop("spec", None)
    router._buffers.pop("balance_bias")
    assert ex.mx is None and ex.mx_act is None and router.spec is None
    router.to(torch.bfloat16)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.route_topk(torch.zeros(2, 4), 1), lambda: ops.quant_rows_mx(x),
                 lambda: ops.fake_quant_mx_cols(x[None]), lambda: ops.add_rmsnorm(x, x, torch.ones(64), 1e-5)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_coded_rows_and_tables_are_checked():
    """Codes, scales and tables that the kernels would read past: refused by their layout, on
    any device."""
    u8 = torch.uint8
    good = ops.MXRows(torch.zeros(4, 128, dtype=u8), torch.zeros(4, 16, dtype=u8), 64, "e4m3")
    pw = ops.PackedWeightsMX(*(torch.zeros(1, dtype=u8) for _ in range(4)), 2, 64, 64)
    off, row = torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    bad = [good._replace(q=torch.zeros(4, 256, dtype=u8)[:, :128]), good._replace(q=torch.zeros(4, 64, dtype=u8)),
           good._replace(K=192), good._replace(fmt="e2m1"), good._replace(scale=torch.zeros(3, 16, dtype=u8)),
           good._replace(scale=torch.zeros(4, 4, dtype=u8)), good._replace(scale=torch.zeros(4, 32, dtype=u8)[:, :16]),
           good._replace(q=good.q.to(torch.int32)), good._replace(q=torch.zeros(128, 4, dtype=u8).t()),
           good._replace(q=torch.zeros(4 * 128 + 8, dtype=u8)[8:].view(4, 128))]
    for r in bad:
        for call in (lambda: ops.dequant_rows_mx(r), lambda: ops.gemm_gate_up_mx(r, None, off, pw, 4),
                     lambda: ops.gemm_down_mx(r, off, pw, 4)):
            with pytest.raises(ValueError, match="contiguous, 16-byte aligned codes"):
                call()
    for o, r in ((off[:2], row), (off.long(), row), (off, row[:3]), (off, row.long()), (off, row.repeat(2)[::2])):
        with pytest.raises(ValueError, match="contiguous int32"):
            ops.gemm_gate_up_mx(good, r, o, pw, 4)
    with pytest.raises(ValueError, match="contiguous int32"):
        ops.gemm_down_mx(good, off[:2], pw, 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.gemm_down_mx(good, off, pw, 4)


def test_capture_beside_an_eager_graph_is_refused(monkeypatch):
    """The rule alone, on stand-ins for leaves: refused while a graph recorded on the default
    stream lives, not for graphs of other leaves, of another stream, or gone."""
    from types import SimpleNamespace

    from kmoe import backward

    def leaf(**kw):
        return SimpleNamespace(**{**dict(requires_grad=True, is_leaf=True, is_cuda=True), **kw})
    state = dict(capturing=False, stream=0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(ops, "_stream", lambda t: state["stream"])

    def record(*leaves, **kw):
        state.update(dict(capturing=False, stream=0), **kw)
        ctx = SimpleNamespace()
        backward.leaves_of(ctx, *leaves)
        return ctx
    a, b, c = leaf(), leaf(), leaf(is_leaf=False)
    first, second = record(a, None, c), record(a)
    del first
    with pytest.raises(RuntimeError, match="still alive"):
        record(b, a, capturing=True)
    record(b, c, capturing=True)
    del second
    record(a, capturing=True)
    side = record(b, stream=7)
    record(b, capturing=True)
    assert not vars(side)


# ---- the restatements themselves
def test_elements_against_torch_casts():
    v = torch.cat([torch.linspace(-500, 500, 20001), torch.logspace(-12, 9, 5000, base=2.0)]).double()
    want = v.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()
    assert torch.equal(M.elements(v, "e4m3").abs(), want.abs())
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    near = M.elements(v, "e2m1").abs()
    dist = (v.abs()[:, None].clamp(max=6) - grid).abs().min(1).values
    assert torch.equal((near - v.abs().clamp(max=6)).abs(), dist)
    ties = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    assert M.elements(ties, "e2m1").tolist() == [0, 1, 1, 2, 2, 4, 4]


def test_values_are_a_fixed_point():
    v = torch.randn(40, 64, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    for fmt in ("e4m3", "e2m1"):
        q = M.quant(v, fmt)[0]
        assert torch.equal(M.quant(q, fmt)[0], q)


def test_straight_through_formula_against_differences():
    """With the quantisers' steps held fixed (each a constant added to its input) the experts are
    a smooth function whose gradient the straight-through one is."""
    g = torch.Generator().manual_seed(1)
    x, w1, w2, w3 = (0.3 * torch.randn(*s, dtype=torch.float64, generator=g) for s in ((3, 32), (32, 8), (32, 8), (8, 32)))
    dy = torch.randn(3, 32, dtype=torch.float64, generator=g)
    leaves = [t.clone().requires_grad_(True) for t in (x, w1, w2, w3)]
    grads = torch.autograd.grad(M.swiglu_rows(*leaves, "e4m3"), leaves, dy)
    off = [M.quant(x, "e4m3")[0] - x] + [M.q_cols(w[None])[0] - w for w in (w1, w2, w3)]
    h0 = torch.nn.functional.silu((x + off[0]) @ (w1 + off[1])) * ((x + off[0]) @ (w2 + off[2]))
    hoff = M.quant(h0, "e4m3")[0] - h0

    def f(x, w1, w2, w3):
        h = torch.nn.functional.silu((x + off[0]) @ (w1 + off[1])) * ((x + off[0]) @ (w2 + off[2])) + hoff
        return ((h @ (w3 + off[3])) * dy).sum()
    base = [x, w1, w2, w3]
    for i, gr in enumerate(grads):
        for at in ((0, 0), (1, 5), (2, 7)):
            d = torch.zeros_like(base[i])
            d[at] = 1e-5
            num = (f(*[b + d if j == i else b for j, b in enumerate(base)])
                   - f(*[b - d if j == i else b for j, b in enumerate(base)])) / 2e-5
            assert abs(float(num - gr[at])) <= 1e-7 * (1 + abs(float(num)))


def test_route_restatement_against_torch():
    lg = torch.randn(50, 12, generator=torch.Generator().manual_seed(2))
    idx, w = M.route(lg, 3)
    v, i = torch.topk(torch.softmax(lg.double(), -1), 3)
    assert torch.equal(idx, i) and torch.allclose(w, v / v.sum(-1, keepdim=True), rtol=1e-12)
    idx, w = M.route(lg, 2, kind="sigmoid", groups=4, topk_groups=1, group_top=1, renorm=False, scale=2.0)
    s = torch.sigmoid(lg.double()).view(50, 4, 3)
    best = s.amax(-1).argmax(-1)
    v, i = s[torch.arange(50), best].topk(2)
    assert torch.equal(idx, best[:, None] * 3 + i) and torch.allclose(w, 2 * v, rtol=1e-12)


def test_shapes_types_and_places_of_arguments():
    """What the kernels would read past or misread is refused before anything else, on any device."""
    h, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64)
    r = torch.ones(4)
    for kw in (dict(weight=torch.ones(32)), dict(rrms=torch.ones(3)), dict(rrms=torch.ones(4, 1)), dict(rrms=r.double()),
               dict(dn=h[:2]), dict(dh=h[:, :32])):
        a = {**dict(dn=h, h=h, weight=w, rrms=r), **kw}
        with pytest.raises(ValueError, match="add_rmsnorm_bwd"):
            ops.add_rmsnorm_bwd(**a)
    rows = ops.MXRows(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 16, dtype=torch.uint8), 64, "e4m3")
    for n in (torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(ValueError, match="n_rows_dev"):
            ops.quant_rows_mx(h, n_rows_dev=n)
        with pytest.raises(ValueError, match="n_rows_dev"):
            ops.dequant_rows_mx(rows, n_rows_dev=n)


class _On:
    """A tensor's stand-in on a device of that name."""

    def __init__(self, name):
        self.device, self.is_cuda = torch.device(name), name != "cpu"

    def get_device(self):
        return self.device.index if self.is_cuda else -1


def test_tensors_of_one_call_are_on_one_gpu():
    ops._one_gpu("f", _On("cuda:0"), None, _On("cuda:0"))
    for other in ("cpu", "cuda:1"):
        with pytest.raises(ValueError, match="one GPU"):
            ops._one_gpu("f", _On("cuda:0"), None, _On(other))
    with pytest.raises(ValueError, match="GPU"):
        ops._one_gpu("f", _On("cpu"), _On("cuda:0"))
