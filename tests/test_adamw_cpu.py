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
