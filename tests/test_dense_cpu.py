"""The dense operators without a GPU: refusals of arguments, in Python and at the C ABI."""
import ctypes

import pytest
import torch

import kmoe
from kmoe import _lib

BF = torch.bfloat16
FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x1008)


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def ad(n=2, r=8, K=64, N=72):
    return kmoe.Adapters(z(n, r, K), z(n, N, r), torch.ones(n))


IDS = torch.zeros(4, dtype=torch.int32)


@pytest.mark.parametrize("args,kw,match", [
    ((z(4, 64), z(72, 64), z(72, 64), z(64, 72), "swish"), {}, "activation"),
    ((z(4, 64), z(72, 64), z(72, 64), z(64, 72), ["silu"]), {}, "activation"),
    ((z(4, 64), z(72, 64), z(72, 56), z(64, 72)), {}, "w_up"),
    ((z(4, 64), z(72, 64), z(72, 64), z(72, 64)), {}, "w_down"),
    ((z(4, 56), z(72, 64), z(72, 64), z(64, 72)), {}, "x "),
    ((z(4, 64).int(), z(72, 64), z(72, 64), z(64, 72)), {}, "floating point"),
    ((z(4, 60), z(72, 60), z(72, 60), z(60, 72)), {}, "multiples of 8"),
    ((z(4, 64), z(70, 64), z(70, 64), z(64, 70)), {}, "multiples of 8"),
    ((z(4, 64), z(72, 64, dtype=torch.float16), z(72, 64), z(64, 72)), {}, "bf16 or f32"),
    ((z(4, 64), z(72, 64), z(72, 64), z(64, 72)), {}, "on a GPU"),
    ((z(4, 64), z(72, 64), z(72, 64), z(64, 72)), dict(adapters=kmoe.FFNAdapters(gate=ad(N=64)), ids=IDS), "gate adapters"),
    ((z(4, 64), z(72, 64), z(72, 64), z(64, 72)), dict(adapters=kmoe.FFNAdapters(gate=ad()), ids=IDS), "on a GPU"),
])
def test_ffn_refusals(args, kw, match):
    with pytest.raises(ValueError, match=match):
        kmoe.gated_ffn(*args, **kw)


def test_adapter_refusals():
    x, w = z(4, 64), z(72, 64)
    bad = [ad()._replace(a=z(2, 8, 72)), ad()._replace(b=z(2, 64, 8)), ad()._replace(b=z(3, 72, 8)), ad()._replace(b=z(2, 72, 16)),
           ad(r=136), ad(r=0), ad(n=0), ad()._replace(a=z(8, 64))]
    for a in bad:
        with pytest.raises(ValueError, match="adapted_linear: a must be"):
            kmoe.adapted_linear(x, w, a, IDS)
    with pytest.raises(ValueError, match="scale must be"):
        kmoe.adapted_linear(x, w, ad()._replace(scale=torch.ones(3)), IDS)
    with pytest.raises(ValueError, match="no gradient"):
        kmoe.adapted_linear(x, w, ad()._replace(scale=torch.ones(2, requires_grad=True)), IDS)
    with pytest.raises(ValueError, match="on a GPU"):
        kmoe.adapted_linear(x, w, ad(), IDS)
    from kmoe.dense import _ids
    with pytest.raises(ValueError, match="need ids"):
        _ids(None, x, 2, "adapted_linear")
    with pytest.raises(ValueError, match="one for each row"):
        _ids(IDS[:3], x, 2, "adapted_linear")
    with pytest.raises(ValueError, match="int32 or int64"):
        _ids(IDS.float(), x, 2, "adapted_linear")
    assert _ids(torch.tensor([1 << 32, -5, 0, 1]), x, 2, "adapted_linear").tolist() == [2, -1, 0, 1]


def test_module():
    with pytest.raises(ValueError, match="multiples of 8"):
        kmoe.GatedFFN(60, 72)
    with pytest.raises(ValueError, match="activation"):
        kmoe.GatedFFN(64, 72, "tanh")
    m = kmoe.GatedFFN(64, 72)
    assert [tuple(p.shape) for p in m.parameters()] == [(72, 64), (72, 64), (64, 72)]
    c = kmoe.get_test_config()
    assert kmoe.MoELayer(c).shared is None
    c.moe_shared_d_ff = 704
    layer = kmoe.MoELayer(c)
    assert layer.shared is layer.shared_expert and layer.shared.d_ff == 704
    import pickle
    old = kmoe.MoELayer(kmoe.get_test_config())
    del old.__dict__["shared_expert"]  # as a layer pickled before there were any
    assert pickle.loads(pickle.dumps(old)).shared is None
    c.ffn_activation = "silu"
    with pytest.raises(NotImplementedError, match="swiglu"):
        kmoe.MoELayer(c)


def _call(name, good):
    fn = getattr(_lib.load(), name)

    def call(**at):
        a = list(good)
        for k, v in at.items():
            a[int(k[1:])] = v
        return fn(*a)
    return call


def test_abi_gated_ffn():
    a = _lib.Adapter(0x1000, 0x1000, None, 8)
    ws = _lib.load().kmoe_gated_ffn_workspace_bytes(100, 64, 72, 8, 8)
    assert ws >= 100 * 72 * 2 + 3 * 100 * 8 * 2
    call = _call("kmoe_gated_ffn", [FAKE, 100, 64, 72, FAKE, FAKE, FAKE, 0, FAKE, 2, ctypes.byref(a), ctypes.byref(a),
                                    ctypes.byref(a), FAKE, FAKE, ws, None])
    assert call(a1=0) == 0
    for i in (0, 4, 5, 6, 8, 13, 14):
        assert call(**{f"a{i}": None}) == -1, i
    for i in (0, 4, 5, 6, 13, 14):
        assert call(**{f"a{i}": ODD}) == -2, i
    assert call(a1=-1) == -2 and call(a1=1 << 31) == -2 and call(a2=60) == -2 and call(a3=0) == -2
    assert call(a7=4) == -6 and call(a7=-1) == -6
    assert call(a9=0) == -2 and call(a15=ws - 1) == -4
    for r in (0, 4, 136):
        assert call(a10=ctypes.byref(_lib.Adapter(0x1000, 0x1000, None, r))) == -2
    assert call(a11=ctypes.byref(_lib.Adapter(0x1000, 0x1000, None, 16))) == -2  # not the gate's rank
    assert call(a12=ctypes.byref(_lib.Adapter(None, 0x1000, None, 8))) == -1
    assert call(a12=ctypes.byref(_lib.Adapter(0x1008, 0x1000, None, 8))) == -2


def test_abi_adapted_linear_backward():
    a = _lib.Adapter(0x1000, 0x1000, None, 8)
    ws = _lib.load().kmoe_adapted_linear_backward_workspace_bytes(100, 64, 72, 2, 8)
    assert ws >= 2 * (100 * 8 + 2 * 8 * 64 + 2 * 8 * 72)
    call = _call("kmoe_adapted_linear_backward", [FAKE, FAKE, 100, 64, FAKE, 72, FAKE, 2, ctypes.byref(a), FAKE, FAKE, FAKE,
                                                  FAKE, FAKE, ws, None])
    assert call(a2=0, a10=None, a11=None, a12=None) == 0
    for i in (0, 1, 4, 6, 8, 9):
        assert call(**{f"a{i}": None}) == -1, i
    for i in (0, 1, 4, 9, 10, 11, 12, 13):
        assert call(**{f"a{i}": ODD}) == -2, i
    assert call(a2=-1) == -2 and call(a3=4) == -2 and call(a5=0) == -2 and call(a7=0) == -2 and call(a7=32768) == -2
    assert call(a14=ws - 1) == -4 and call(a13=None) == -4
    for r in (0, 4, 136):
        assert call(a8=ctypes.byref(_lib.Adapter(0x1000, 0x1000, None, r))) == -2
    assert call(a8=ctypes.byref(_lib.Adapter(None, 0x1000, None, 8))) == -1


def test_abi_adapted_linear():
    a = _lib.Adapter(0x1000, 0x1000, None, 8)
    ws = _lib.load().kmoe_adapted_linear_workspace_bytes(100, 64, 72, 8)
    call = _call("kmoe_adapted_linear", [FAKE, 100, 64, FAKE, 72, FAKE, 2, ctypes.byref(a), FAKE, FAKE, ws, None])
    assert call(a1=0) == 0 and call(a10=ws - 1) == -4 and call(a9=None) == -4
    for i in (0, 3, 5, 8):
        assert call(**{f"a{i}": None}) == -1, i
    assert call(a2=4) == -2 and call(a4=-8) == -2 and call(a6=0) == -2 and call(a8=ODD) == -2


def test_abi_parts():
    call = _call("kmoe_dense_gate_up", [FAKE, 100, 64, FAKE, FAKE, 72, 0, FAKE, 0, FAKE, None])
    assert call(a1=0) == 0
    for i in (0, 3, 4, 7):
        assert call(**{f"a{i}": None}) == -1, i
    assert _lib.load().kmoe_dense_saved_bytes(17, 24) == 2 * 2 * 1536 and _lib.load().kmoe_dense_saved_bytes(0, 24) == 0
    assert call(a6=9) == -6 and call(a2=63) == -2 and call(a7=ODD) == -2 and call(a9=ODD) == -2 and call(a8=1) == -2
    call = _call("kmoe_dense_linear", [FAKE, 0, 100, 64, FAKE, 72, FAKE, None])
    assert call(a2=0) == 0
    for i in (0, 4, 6):
        assert call(**{f"a{i}": None}) == -1, i
    assert call(a3=0) == -2 and call(a5=71) == -2 and call(a6=ODD) == -2
    assert call(a3=1 << 22) == -2  # a tile's offsets are 32 bits
    assert call(a1=1, a2=_lib.LOST_ROWS + 1) == -2
    call = _call("kmoe_dense_dh", [FAKE, 100, 64, FAKE, 72, FAKE, FAKE, FAKE, 0, None])
    assert call(a1=0) == 0
    for i in (0, 3, 5, 6, 7):
        assert call(**{f"a{i}": None}) == -1, i
    assert call(a8=1) == -2
    call = _call("kmoe_dense_dx", [FAKE, None, 0, 100, 72, FAKE, None, 64, FAKE, None])
    assert call(a3=0) == 0
    for i in (0, 5, 8):
        assert call(**{f"a{i}": None}) == -1, i
    assert call(a1=FAKE) == -1 and call(a2=1) == -2
    call = _call("kmoe_dense_wgrad", [FAKE, FAKE, None, None, 101, 72, 64, FAKE, 0, None])
    for i in (0, 1, 7):
        assert call(**{f"a{i}": None}) == -1, i
    assert call(a2=FAKE) == -1 and call(a2=FAKE, a3=ODD) == -2
    assert call(a4=-1) == -2 and call(a5=4) == -2 and call(a6=0) == -2 and call(a8=2) == -3 and call(a7=ODD) == -2


def _partial_bytes(T, n, r, C, C2):
    """Bytes of the partial sums of a launch over the gradients of factors of C and C2 columns (0: none):
    columns in blocks of 128 an adapter, runs of rows up to 512 workgroups, of 256 to 65536 rows."""
    up = lambda a, b: -(-a // b)
    runs = min(up(512, n * (up(C, 128) + up(C2, 128))), up(T, 256))
    runs = max(runs, up(T, 65536), 1)
    return runs * n * r * (C + C2) * 4 if runs > 1 else 0


def test_adapter_gradients_fit_their_workspace():
    """With the gradients of both factors, or of either one alone, which may take more runs of rows."""
    import random
    lib, rng = _lib.load(), random.Random(3)
    piece = lambda b: -(-b // 256) * 256
    cases = [(257, 2048, 2048, 16, 16), (513, 2048, 5632, 5, 16), (2042, 2048, 2048, 16, 16), (4099, 2048, 5632, 16, 32),
             (1, 8, 8, 1, 8), (70000, 64, 72, 2, 8)]
    cases += [(rng.randint(1, 1 << rng.randint(1, 18)), 8 * rng.randint(1, 704), 8 * rng.randint(1, 704), rng.randint(1, 40),
               8 * rng.randint(1, 16)) for _ in range(5000)]
    for T, K, N, n, r in cases:
        have = lib.kmoe_adapted_linear_backward_workspace_bytes(T, K, N, n, r)
        have -= piece(4 * T * r) + piece(2 * n * r * K) + piece(2 * n * r * N)
        for C, C2 in ((K, N), (K, 0), (N, 0)):
            assert _partial_bytes(T, n, r, C, C2) <= have, (T, K, N, n, r, C, C2)


def test_odd_ranks_are_filled_up_inside_the_operator():
    """The factors reach the operator's own graph node as they are: another node of theirs, outside of it, would
    not be seen where a capture beside a live graph of the same leaves is refused."""
    from kmoe import dense
    given = kmoe.Adapters(z(2, 5, 64).requires_grad_(True), z(2, 72, 5).requires_grad_(True))
    got = dense._adapters(given, 64, 72, "adapted_linear", "")
    assert got.a is given.a and got.b is given.b
    a, b = (t.detach().normal_() for t in given[:2])
    held = dense._held(kmoe.Adapters(a, b))
    assert held.a.shape == (2, 8, 64) and held.b.shape == (2, 72, 8)
    assert torch.equal(held.a[:, :5], a) and torch.equal(held.b[..., :5], b)
    assert not bool(held.a[:, 5:].any()) and not bool(held.b[..., 5:].any())


def test_abi_refuses_launches_past_32_bits():
    """Grids of 2^32 threads and counters of 2^31 rows, before anything is launched."""
    a, lib = _lib.Adapter(0x1000, 0x1000, None, 8), _lib.load()
    big = 1 << 62
    call = _call("kmoe_adapted_linear", [FAKE, 1 << 27, 8, FAKE, 8, FAKE, 2, ctypes.byref(a), FAKE, FAKE, big, None])
    assert call() == -2 and call(a1=(1 << 31) - 1) == -2
    call = _call("kmoe_adapted_linear_backward", [FAKE, FAKE, 1 << 27, 8, FAKE, 8, FAKE, 2, ctypes.byref(a), FAKE, FAKE, FAKE, FAKE, FAKE,
                                                  big, None])
    assert call() == -2
    call = _call("kmoe_gated_ffn", [FAKE, 1 << 27, 8, 8, FAKE, FAKE, FAKE, 0, FAKE, 2, None, None, ctypes.byref(a), FAKE, FAKE, big, None])
    assert call() == -2
    call = _call("kmoe_dense_linear", [FAKE, 0, (1 << 31) - 1, 8, FAKE, 8, FAKE, None])
    assert call() == -2
    call = _call("kmoe_dense_wgrad", [FAKE, FAKE, None, None, (1 << 31) - 63, 8, 8, FAKE, 0, None])
    assert call() == -2
    n = 1 << 35
    assert lib.kmoe_adamw_values(FAKE, FAKE, FAKE, FAKE, n, 0, FAKE, FAKE, None) == -2
    base = (ctypes.c_int32 * 2)(0, 1 << 24)
    assert lib.kmoe_adamw(FAKE, FAKE, FAKE, base, 1, (ctypes.c_void_p * 1)(0x1000), 0, 32, 0, 1e-3, None, 0.9, 0.99, 1e-8, 0.0,
                          FAKE, None) == -2
