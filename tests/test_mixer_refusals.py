"""Arguments that linear attention and block_norm refuse, on the CPU: Python's checks, the C ABI's status codes (given before
any device is asked for), and shapes without a GPU."""
import ctypes

import pytest
import torch

import sffft_b200 as sf
import sffft_b200.torch_ops as ops

B, H, HKV, L, D, DV = 2, 4, 2, 10, 16, 24


def la_args(**kw):
    a = dict(q=torch.zeros(B, H, L, D), k=torch.zeros(B, HKV, L, D), v=torch.zeros(B, HKV, L, DV), log_decay=torch.zeros(H))
    a.update(kw)
    return a


BAD_LA = {
    "k of another length": dict(k=torch.zeros(B, HKV, L + 1, D)),
    "v of other heads": dict(v=torch.zeros(B, H, L, DV)),
    "heads that do not divide": dict(k=torch.zeros(B, 3, L, D), v=torch.zeros(B, 3, L, DV)),
    "no heads": dict(k=torch.zeros(B, 0, L, D), v=torch.zeros(B, 0, L, DV)),
    "three axes": dict(q=torch.zeros(H, L, D)),
    "mixed types": dict(k=torch.zeros(B, HKV, L, D, dtype=torch.bfloat16)),
    "half precision": dict(q=torch.zeros(B, H, L, D, dtype=torch.float16)),
    "decay of another length": dict(log_decay=torch.zeros(H + 1)),
    "decay in bf16": dict(log_decay=torch.zeros(H, dtype=torch.bfloat16)),
    "decay that wants a gradient": dict(log_decay=torch.zeros(H, requires_grad=True)),
    "scale 0": dict(scale=0.0),
    "scale nan": dict(scale=float("nan")),
    "state of another shape": dict(initial_state=torch.zeros(B, H, DV, D)),
    "state in bf16": dict(initial_state=torch.zeros(B, H, D, DV, dtype=torch.bfloat16)),
    "lengths in int64": dict(lengths=torch.zeros(B, dtype=torch.int64)),
    "lengths of another batch": dict(lengths=torch.zeros(B + 1, dtype=torch.int32)),
    "CPU tensors": dict(),
}


@pytest.mark.parametrize("what", BAD_LA)
def test_linear_attention_refuses(what):
    with pytest.raises(ValueError):
        sf.linear_attention(**la_args(**BAD_LA[what]))
    with pytest.raises(ValueError):
        ops.linear_attention(**la_args(**BAD_LA[what]))
    with pytest.raises(ValueError):
        sf.linear_attention_backward(**la_args(**BAD_LA[what]), dy=torch.zeros(B, H, L, DV))


def step_args(**kw):
    a = dict(q=torch.zeros(B, H, D), k=torch.zeros(B, HKV, D), v=torch.zeros(B, HKV, DV), log_decay=torch.zeros(H),
             state=torch.zeros(5, H, D, DV))
    a.update(kw)
    return a


BAD_STEP = {
    "k of another size": dict(k=torch.zeros(B, HKV, D + 1)),
    "heads that do not divide": dict(k=torch.zeros(B, 3, D), v=torch.zeros(B, 3, DV)),
    "a state of another shape": dict(state=torch.zeros(5, H, DV, D)),
    "a state in bf16": dict(state=torch.zeros(5, H, D, DV, dtype=torch.bfloat16)),
    "a transposed state": dict(state=torch.zeros(5, H, DV, D).transpose(2, 3)),
    "slots that overlap": dict(state=torch.zeros(1, H, D, DV).expand(5, H, D, DV)),
    "too few slots": dict(state=torch.zeros(1, H, D, DV)),
    "slots in int64": dict(slots=torch.zeros(B, dtype=torch.int64)),
    "slots of another batch": dict(slots=torch.zeros(B + 1, dtype=torch.int32)),
    "scale inf": dict(scale=float("inf")),
    "CPU tensors": dict(),
}


@pytest.mark.parametrize("what", BAD_STEP)
def test_step_refuses(what):
    for f in (sf.linear_attention_step, ops.linear_attention_step):
        with pytest.raises(ValueError):
            f(**step_args(**BAD_STEP[what]))


def test_step_refuses_a_gradient():
    with pytest.raises(ValueError):
        ops.linear_attention_step(**step_args(q=torch.zeros(B, H, D, requires_grad=True)))


def bn_args(**kw):
    t = torch.zeros
    a = dict(x=t(3, 5, 32), y=t(3, 5, 32), gate=t(3, 5, 32), post_weight=t(32), weight=t(32))
    a.update(kw)
    return a


BAD_BN = {
    "nothing": dict(x=None, y=None),
    "x of another shape": dict(x=torch.zeros(3, 5, 31)),
    "x in bf16 beside y in fp32": dict(x=torch.zeros(3, 5, 32, dtype=torch.bfloat16)),
    "half precision": dict(y=torch.zeros(3, 5, 32, dtype=torch.float16)),
    "a gate of another shape": dict(gate=torch.zeros(5, 32)),
    "a gate of another type": dict(gate=torch.zeros(3, 5, 32, dtype=torch.bfloat16)),
    "a weight of another size": dict(weight=torch.zeros(31)),
    "weights of two types": dict(weight=torch.zeros(32, dtype=torch.bfloat16)),
    "groups that do not divide": dict(groups=5),
    "no groups": dict(groups=0),
    "another activation": dict(act="gelu"),
    "a gate without y": dict(y=None, post_weight=None),
    "only x": dict(y=None, gate=None, post_weight=None, weight=None),
    "another axis": dict(dim=0),
    "eps below 0": dict(eps=-1e-6),
    "scale nan": dict(scale=float("nan")),
    "CPU tensors": dict(),
}


@pytest.mark.parametrize("what", BAD_BN)
def test_block_norm_refuses(what):
    for f in (sf.block_norm, ops.block_norm):
        with pytest.raises(ValueError):
            f(**bn_args(**BAD_BN[what]))


def test_c_abi_statuses():
    lib = sf.lib()
    size = ctypes.c_size_t()
    def la(**kw):
        f = dict(B=1, H=2, Hkv=1, L=4, D=8, Dv=8, io=0, device=0, scale=1.0)
        f.update(kw)
        return ctypes.byref(sf.LinearAttentionDesc(*f.values()))
    call = lambda d, q=16, work=None: lib.sffft_linear_attention(d, q, 16, 16, 16, None, None, 16, None, work, 0, None)  # noqa: E731
    bad = [dict(H=0), dict(Hkv=0), dict(H=3, Hkv=2), dict(B=-1), dict(L=-1), dict(D=0), dict(Dv=0), dict(io=2), dict(device=-1),
           dict(scale=0.0), dict(scale=float("inf"))]
    for kw in bad:
        assert call(la(**kw)) == sf.ERR_INVALID_ARGUMENT, kw
        assert lib.sffft_linear_attention_workspace_bytes(la(**kw), 0, ctypes.byref(size)) == sf.ERR_INVALID_ARGUMENT
        g = ctypes.byref(sf.LinearAttentionGrads())
        assert lib.sffft_linear_attention_backward(la(**kw), g, *[16] * 4, None, None, 16, None, 16, 16, 16, None, None, 0,
                                                   None) == sf.ERR_INVALID_ARGUMENT
    assert call(None) == sf.ERR_INVALID_ARGUMENT
    assert call(la(), q=None) == sf.ERR_INVALID_ARGUMENT
    assert call(la(), work=8) == sf.ERR_INVALID_ARGUMENT
    assert lib.sffft_linear_attention(la(), 16, 16, 16, None, None, None, 16, None, None, 0, None) == sf.ERR_INVALID_ARGUMENT
    assert call(la(D=257)) == sf.ERR_UNSUPPORTED and call(la(Dv=4097)) == sf.ERR_UNSUPPORTED
    assert call(la(B=1 << 20, H=1 << 10, Hkv=1)) == sf.ERR_UNSUPPORTED
    assert lib.sffft_linear_attention_workspace_bytes(la(), 0, None) == sf.ERR_INVALID_ARGUMENT
    assert call(la(B=0)) == sf.OK
    g = ctypes.byref(sf.LinearAttentionGrads())
    assert lib.sffft_linear_attention_backward(la(Dv=257), g, *[16] * 4, None, None, 16, None, 16, 16, 16, None, None, 0,
                                               None) == sf.ERR_UNSUPPORTED
    assert lib.sffft_linear_attention_backward(la(), None, *[16] * 4, None, None, 16, None, 16, 16, 16, None, None, 0,
                                               None) == sf.ERR_INVALID_ARGUMENT

    def step(**kw):
        f = dict(B=2, H=2, Hkv=1, D=8, Dv=8, pool=2, io=0, device=0, scale=1.0)
        f.update(kw)
        return ctypes.byref(sf.LinearAttentionStepDesc(*f.values()))
    call = lambda d, slots=None, state=16: lib.sffft_linear_attention_step(d, 16, 16, 16, 16, state, slots, 16, None)  # noqa: E731
    for kw in (dict(H=0), dict(H=3, Hkv=2), dict(B=-1), dict(D=0), dict(pool=1), dict(pool=-1), dict(io=2), dict(scale=float("nan"))):
        assert call(step(**kw)) == sf.ERR_INVALID_ARGUMENT, kw
    assert call(step(), state=None) == sf.ERR_INVALID_ARGUMENT and call(None) == sf.ERR_INVALID_ARGUMENT
    assert call(step(), state=18) == sf.ERR_INVALID_ARGUMENT
    assert call(step(B=0, pool=0)) == sf.OK

    def bn(**kw):
        f = dict(rows=4, channels=8, inner=0, groups=1, io=0, res_io=0, weight_io=0, gate=0, act=0, scale=1.0, eps=1e-6, device=0)
        f.update(kw)
        return ctypes.byref(sf.BlockNormDesc(*f.values()))
    call = lambda d, x=16, y=16, gate=None, pw=16, w=16, h=16, n=16: lib.sffft_block_norm(d, x, y, gate, pw, w, h, n, None, None, None)  # noqa: E731
    for kw in (dict(rows=-1), dict(channels=0), dict(inner=-1), dict(inner=3), dict(groups=0), dict(groups=3), dict(io=2), dict(gate=3),
               dict(act=3), dict(scale=float("inf")), dict(eps=-1.0), dict(eps=float("nan")), dict(gate=1), dict(device=-1)):
        assert call(bn(**kw)) == sf.ERR_INVALID_ARGUMENT, kw
    assert call(None) == sf.ERR_INVALID_ARGUMENT
    assert call(bn(), gate=16) == sf.ERR_INVALID_ARGUMENT          # a gate that the descriptor does not name
    assert call(bn(), x=None, y=None) == sf.ERR_INVALID_ARGUMENT
    assert call(bn(), y=None) == sf.ERR_INVALID_ARGUMENT           # a weight for y without y
    assert call(bn(), y=None, pw=None, w=None) == sf.ERR_INVALID_ARGUMENT
    assert call(bn(), h=None) == sf.ERR_INVALID_ARGUMENT and call(bn(), n=None) == sf.ERR_INVALID_ARGUMENT
    assert call(bn(res_io=1)) == sf.ERR_UNSUPPORTED and call(bn(channels=8193)) == sf.ERR_UNSUPPORTED
    assert call(bn(rows=0)) == sf.OK
    back = lambda d, r1=16, r2=16, dh=16, dn=16, dx=16, work=256: lib.sffft_block_norm_backward(  # noqa: E731
        d, 16, 16, None, 16, 16, r1, r2, dh, dn, dx, 16, None, 16, 16, work, 0, None)
    for kw in (dict(r1=None), dict(r2=None), dict(dn=None), dict(dx=None), dict(work=16)):
        assert back(bn(), **kw) == sf.ERR_INVALID_ARGUMENT, kw
    assert lib.sffft_block_norm_workspace_bytes(bn(), None) == sf.ERR_INVALID_ARGUMENT


def test_c_abi_refuses_addresses_between_elements():
    lib = sf.lib()
    la = ctypes.byref(sf.LinearAttentionDesc(1, 2, 2, 4, 8, 8, sf.IO["bf16"], 0, 1.0))
    g = ctypes.byref(sf.LinearAttentionGrads())
    step = ctypes.byref(sf.LinearAttentionStepDesc(2, 2, 2, 8, 8, 2, sf.IO["bf16"], 0, 1.0))
    bn = ctypes.byref(sf.BlockNormDesc(4, 8, 0, 1, sf.IO["bf16"], sf.IO["fp32"], sf.IO["fp32"], 0, 0, 1.0, 1e-6, 0))

    def refused(f, *args, odd):   # each of the addresses in turn
        for i in odd:
            a = list(args)
            a[i] += 1 if a[i] else 257
            assert f(*a) == sf.ERR_INVALID_ARGUMENT, (f.__name__, i)

    refused(lib.sffft_linear_attention, la, 16, 16, 16, 16, 16, 16, 16, 32, 0, 0, None, odd=[*range(1, 9), 9])
    refused(lib.sffft_linear_attention_backward, la, g, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 32, 0, 0, None, odd=range(2, 14))
    refused(lib.sffft_linear_attention_step, step, 16, 16, 16, 16, 16, 16, 16, None, odd=range(1, 8))
    refused(lib.sffft_block_norm, bn, 16, 16, None, 16, 16, 16, 16, 16, 16, None, odd=[1, 2, 4, 5, 6, 7, 8, 9])
    refused(lib.sffft_block_norm_backward, bn, 16, 16, None, 16, 16, 16, 16, 16, 16, 16, 16, None, 16, 16, 256, 0, None,
            odd=[1, 2, 4, 5, 6, 7, 8, 9, 10, 11, 13, 14, 15])


def test_c_abi_refuses_a_state_in_its_own_place():
    lib = sf.lib()
    la = ctypes.byref(sf.LinearAttentionDesc(1, 2, 2, 4, 8, 8, 0, 0, 1.0))
    g = ctypes.byref(sf.LinearAttentionGrads())
    assert lib.sffft_linear_attention(la, 16, 16, 16, 16, None, 32, 16, 32, None, 0, None) == sf.ERR_INVALID_ARGUMENT
    assert lib.sffft_linear_attention_backward(la, g, 16, 16, 16, 16, None, 16, 16, 32, 16, 16, 16, 32, None, 0, None) == sf.ERR_INVALID_ARGUMENT


def test_backward_refuses_a_scale_without_a_reciprocal():
    la = ctypes.byref(sf.LinearAttentionDesc(1, 2, 2, 4, 8, 8, 0, 0, 1e-40))
    assert sf.lib().sffft_linear_attention_backward(la, ctypes.byref(sf.LinearAttentionGrads()), 16, 16, 16, 16, None, 16, 16, None, 16,
                                                    16, 16, None, None, 0, None) == sf.ERR_INVALID_ARGUMENT


def test_shapes_without_a_gpu():
    m = lambda *s, dtype=torch.bfloat16: torch.empty(s, device="meta", dtype=dtype)  # noqa: E731
    y, s = ops.linear_attention(m(B, H, L, D), m(B, HKV, L, D), m(B, HKV, L, DV), m(H, dtype=torch.float32))
    assert y.shape == (B, H, L, DV) and y.dtype == torch.bfloat16 and s.shape == (B, H, D, DV) and s.dtype == torch.float32
    q = m(B, L, H, D).transpose(1, 2)
    y, _ = ops.linear_attention(q, m(B, HKV, L, D), m(B, HKV, L, DV), m(H, dtype=torch.float32))
    assert y.transpose(1, 2).is_contiguous()
    y = ops.linear_attention_step(m(B, H, D), m(B, HKV, D), m(B, HKV, DV), m(H, dtype=torch.float32),
                                  m(5, H, D, DV, dtype=torch.float32))
    assert y.shape == (B, H, DV)
    x = m(3, 5, 32, dtype=torch.float32)
    h, n = ops.block_norm(x, m(3, 5, 32), m(32), m(32, dtype=torch.float32), m(32, dtype=torch.float32), groups=4)
    assert h.shape == (3, 5, 32) and h.dtype == torch.float32 and n.dtype == torch.bfloat16
    h, n = ops.block_norm(None, m(3, 5, 32), dim=1)
    assert h.dtype == torch.bfloat16 and n is None
