"""The joint between two blocks (norm, gate, residual scale, residual stream, norm) on the device: values and gradients
against the formulas in 64 bits for each of its parts, both layouts, odd sizes, strides, streams and graphs."""
import ctypes
import itertools

import pytest
import torch

import sffft_b200 as sf
import sffft_b200.torch_ops as ops
from tests import mixer_ref as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def make(shape, dim, dtype, res, gate="full", post=True, residual=True, pre=True, wtype=F32, seed=0, branch=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    C = shape[dim]
    t = dict(x=(2 * r(*shape)).to(res) if residual else None, y=r(*shape).to(dtype) if branch else None)
    t["gate"] = {"full": lambda: r(*shape).to(dtype), "channel": lambda: r(C).to(dtype), "none": lambda: None}[gate]()
    t["post_weight"] = (1 + 0.2 * r(C)).to(wtype) if post else None
    t["weight"] = (1 + 0.2 * r(C)).to(wtype) if pre else None
    return t, r(*shape).to(res if residual else dtype), r(*shape).to(dtype) if pre else None


def check(t, dh, dn, groups=1, act="silu", dim=-1, scale=0.5, eps=1e-5):
    lead = t["y"] if t["y"] is not None else t["x"]
    C, rows = lead.shape[dim], lead.numel() // lead.shape[dim]
    kw = dict(scale=scale, eps=eps, groups=groups, act=act, dim=dim)
    args = (t["x"], t["y"], t["gate"], t["post_weight"], t["weight"], scale, eps, groups, act, dim)
    want, mags = ref.norm(*args, dh, dn), ref.norm_magnitudes(*args, dh, dn)
    h, n, r1, r2 = sf.block_norm(**t, **kw, stats=True)
    got = {"n": n}
    if t["y"] is not None:
        got["h"] = h
    else:
        assert h is t["x"]
    plain = sf.block_norm(**t, **kw)
    assert all(a is b or torch.equal(a, b) for a, b in zip(plain, (h, n)))
    got.update(zip(("dx", "dy", "dgate", "dpw", "dw"), sf.block_norm_backward(dh, dn, **t, rstd_post=r1, rstd=r2, **kw)))
    got = {name: x for name, x in got.items() if x is not None}
    assert set(got) == set(want)
    for name, x in got.items():
        value = want[name]
        assert x.shape == value.shape, name
        off, tol = (x.double() - value).abs(), ref.norm_bound(name, value, mags[name], x.dtype, C, rows)
        bad = ~(off <= tol)
        assert not bad.any(), (name, off[bad].max().item(), (off / tol).max().item(), bad.nonzero()[0].tolist())
    return got


@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF, F32), (BF, BF)])
@pytest.mark.parametrize("gate,post,residual,pre", [c for c in itertools.product(("full", "channel", "none"), (True, False),
                                                                                 (True, False), (True, False))])
def test_every_part_present_or_absent(gate, post, residual, pre, dtype, res):
    res = res if residual else dtype
    for shape, dim in (((3, 5, 96), -1), ((2, 96, 36), 1)):
        t, dh, dn = make(shape, dim, dtype, res, gate, post, residual, pre)
        check(t, dh, dn, 4 if post else 1, dim=dim)


@pytest.mark.parametrize("dtype,res", [(F32, F32), (BF, F32), (BF, BF)])
@pytest.mark.parametrize("C", [1, 7, 8, 64, 100, 256, 257, 512, 768, 1000, 1024, 1030, 2048, 2052, 4096, 5000, 8192, 8191])
def test_channels(C, dtype, res):
    for rows in (1, 5):
        t, dh, dn = make((rows, C), -1, dtype, res, seed=C)
        check(t, dh, dn)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("C,groups", [(768, 12), (768, 3), (768, 2), (1024, 16), (96, 6), (320, 5), (64, 8), (4096, 4), (30, 10), (8192, 2)])
def test_groups(C, groups, dtype):
    t, dh, dn = make((9, C), -1, dtype, F32, seed=groups)
    check(t, dh, dn, groups)
    t, dh, dn = make((2, C, 8), 1, dtype, F32, seed=groups)
    check(t, dh, dn, groups, dim=1)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,C,L", [(1, 1, 1), (2, 40, 3), (1, 64, 31), (3, 100, 32), (2, 33, 33), (1, 768, 100), (2, 1030, 65), (5, 24, 1024)])
def test_channels_first(B, C, L, dtype):
    t, dh, dn = make((B, C, L), 1, dtype, F32, seed=L)
    check(t, dh, dn, dim=1)
    t, dh, dn = make((B, C, L), 1, dtype, dtype, "channel", seed=L)
    check(t, dh, dn, act="sigmoid", dim=1)


@pytest.mark.parametrize("act", ["none", "silu", "sigmoid"])
@pytest.mark.parametrize("wtype", [F32, BF])
def test_activations_and_types_of_weights(act, wtype):
    for gate in ("full", "channel"):
        t, dh, dn = make((2, 50, 128), -1, BF, F32, gate, wtype=wtype)
        got = check(t, dh, dn, act=act)
        assert got["dw"].dtype == wtype and got["dpw"].dtype == wtype and got["dgate"].dtype == BF


def test_many_rows():
    t, dh, dn = make((4, 2047, 256), -1, BF, F32)
    check(t, dh, dn, 4)
    t, dh, dn = make((4, 64, 2048), 1, BF, BF, "channel")
    check(t, dh, dn, 2, dim=1)


def test_norm_alone_before_a_block():
    for shape, dim in (((7, 768), -1), ((2, 64, 40), 1)):
        for dtype in (F32, BF):
            t, _, dn = make(shape, dim, dtype, dtype, "none", False, True, True, branch=False)
            check(t, None, dn, dim=dim)


def test_one_row_of_one_axis():
    t, dh, dn = make((96,), -1, F32, F32)
    check(t, dh, dn, 3)


def test_rows_of_zeros_large_and_small_values():
    t, dh, dn = make((6, 128), -1, F32, F32)
    t["y"][0] = 0
    t["x"][0] = 0
    t["y"][1] *= 1e15
    t["x"][2] *= 1e15
    t["y"][3] *= 1e-15
    check(t, dh, dn, 2)
    h, n = sf.block_norm(**t, scale=0.5, eps=1e-5, groups=2, act="silu")
    assert (h[0] == 0).all() and (n[0] == 0).all()


def test_gate_far_from_zero():
    t, dh, dn = make((3, 64), -1, F32, F32)
    t["gate"] = torch.linspace(-120, 120, 192, device="cuda").reshape(3, 64).contiguous()
    for act in ("silu", "sigmoid"):
        got = check(t, dh, dn, act=act)
        assert all(torch.isfinite(x).all() for x in got.values())


def test_strides():
    g = torch.Generator(device="cuda").manual_seed(0)
    buf = torch.randn((3, 20, 5 * 64 + 1), device="cuda", generator=g).to(BF)
    t, dh, dn = make((3, 20, 64), -1, BF, BF)
    want = check(t, dh, dn)
    views = dict(t)
    for i, name in enumerate(("x", "y", "gate")):
        views[name] = buf[..., 64 * i:64 * i + 64]        # rows at odd addresses, 321 values apart
        views[name].copy_(t[name])
    got = check(views, dh, dn)
    assert all((got[n].float() - want[n].float()).abs().max() <= 2.0 ** -6 * want[n].float().abs().max() for n in want)
    tr = dict(t)
    tr["y"] = t["y"].transpose(0, 1).contiguous().transpose(0, 1)       # rows not evenly spaced
    tr["gate"] = t["gate"].transpose(1, 2).contiguous().transpose(1, 2)  # channels not contiguous
    assert all(torch.equal(a, want[n]) for n, a in check(tr, dh.expand_as(dh), dn).items())
    one = dict(t)
    one["x"] = t["x"][:1].expand(3, 20, 64)
    check(one, dh, dn)


def test_no_rows():
    t, dh, dn = make((0, 64), -1, F32, F32, "channel")
    h, n = sf.block_norm(**t)
    assert h.shape == (0, 64) and n.shape == (0, 64)
    out = sf.block_norm_backward(dh, dn, **t, rstd_post=torch.empty((0, 1), device="cuda"), rstd=torch.empty(0, device="cuda"))
    assert out[0].shape == (0, 64) and all((w == 0).all() and w.shape == (64,) for w in out[2:])


def test_results_do_not_change_from_call_to_call():
    for shape, dim in (((3000, 512), -1), ((3, 256, 1000), 1)):
        t, dh, dn = make(shape, dim, BF, F32, "channel")
        a = check(t, dh, dn, 4, dim=dim)
        for _ in range(2):
            b = check(t, dh, dn, 4, dim=dim)
            assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.parametrize("shape,dim", [((2, 30, 64), -1), ((2, 64, 28), 1)])
def test_gradients_through_autograd_and_against_differences(shape, dim):
    t, dh, dn = make(shape, dim, F32, F32, seed=4)
    names = ("x", "y", "gate", "post_weight", "weight")
    kw = dict(scale=0.5, eps=1e-5, groups=2, act="silu", dim=dim)
    leaves = [t[n].clone().requires_grad_() for n in names]
    h, n = ops.block_norm(*leaves, **kw)
    grads = torch.autograd.grad([h, n], leaves, [dh, dn])
    direct = check(t, dh, dn, 2, dim=dim)
    assert all(torch.equal(a, direct[m]) for a, m in zip(grads, ("dx", "dy", "dgate", "dpw", "dw")))

    def loss(args):
        out = ref.norm(*args, 0.5, 1e-5, 2, "silu", dim)
        return (out["h"] * dh.double()).sum() + (out["n"] * dn.double()).sum()

    g = torch.Generator(device="cuda").manual_seed(5)
    args = [t[m].double() for m in names]
    for i, m in enumerate(names):
        way = torch.randn(t[m].shape, device="cuda", generator=g, dtype=torch.float64)
        e = 1e-4   # the difference's error is e^2 / 6 of the third derivative, whose scale is the first's
        d = (loss(args[:i] + [args[i] + e * way] + args[i + 1:]) - loss(args[:i] + [args[i] - e * way] + args[i + 1:])) / (2 * e)
        got = (grads[i].double() * way).sum()
        assert (d - got).abs() <= 1e-5 * (grads[i].double() * way).abs().sum(), m


def test_autograd_of_one_output_alone():
    t, dh, dn = make((5, 64), -1, F32, F32)
    leaves = {n: w.clone().requires_grad_() for n, w in t.items()}
    h, n = ops.block_norm(**leaves, act="silu")
    _, _, r1, r2 = sf.block_norm(**t, act="silu", stats=True)
    got = torch.autograd.grad(n.sum(), list(leaves.values()), retain_graph=True)
    want = sf.block_norm_backward(None, torch.ones_like(n), **t, rstd_post=r1, rstd=r2, act="silu")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad(h.sum(), [leaves["x"], leaves["y"]])
    assert torch.equal(got[0], torch.ones_like(h))
    w = t["weight"].clone().requires_grad_()
    x = t["x"].clone().requires_grad_()
    same, n = ops.block_norm(x, weight=w)
    assert same is x
    torch.autograd.grad((n * n).sum() + same.sum(), [x, w])


def test_streams_graphs_and_compile():
    t, dh, dn = make((2, 100, 768), -1, BF, F32)
    kw = dict(scale=0.5, groups=12, act="silu")
    want = sf.block_norm(**t, **kw)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = sf.block_norm(**t, **kw, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h, n, r1, r2 = sf.block_norm(**t, **kw, stats=True)
            outs.append((h, n) + sf.block_norm_backward(dh, dn, **t, rstd_post=r1, rstd=r2, **kw))
        graphs.append(g)
    t["x"].mul_(-1)
    torch.cuda.synchronize()
    for g, s in zip(graphs, (side, torch.cuda.Stream())):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    h, n, r1, r2 = sf.block_norm(**t, **kw, stats=True)
    now = (h, n) + sf.block_norm_backward(dh, dn, **t, rstd_post=r1, rstd=r2, **kw)
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, now))
    t["x"].mul_(-1)
    f = torch.compile(lambda x, y: ops.block_norm(x, y, t["gate"], t["post_weight"], t["weight"], **kw), fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(f(t["x"], t["y"]), want))


def test_training_step_under_compile():
    t, dh, dn = make((2, 40, 96), -1, BF, F32, "channel")
    names = ("x", "y", "gate", "post_weight", "weight")

    def loss(*a):
        h, n = ops.block_norm(*a, scale=0.5, groups=4, act="silu")
        return (h * dh).sum() + (n * dn).sum(dtype=torch.float32)

    grads = []
    for f in (loss, torch.compile(loss, fullgraph=True)):
        leaves = [t[n].clone().requires_grad_() for n in names]
        f(*leaves).backward()
        grads.append([x.grad for x in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    x, w = (t[n].clone().requires_grad_() for n in ("x", "weight"))
    g, = torch.autograd.grad(ops.block_norm(x, weight=w)[1].sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):     # no second derivative
        g.sum().backward()


@pytest.mark.parametrize("C,groups,dtype", [(96, 4, F32), (768, 12, BF), (1030, 1, BF), (8192, 2, F32)])
def test_results_in_the_place_of_x_and_y(C, groups, dtype):
    t, _, _ = make((9, C), -1, dtype, F32)
    kw = dict(scale=0.5, eps=1e-5, groups=groups, act="silu")
    h, n = sf.block_norm(**t, **kw)
    p = lambda x: x.data_ptr()  # noqa: E731
    x, y, gate, pw, w = t.values()
    desc = sf.BlockNormDesc(9, C, 0, groups, sf.IO["bf16" if dtype == BF else "fp32"], 0, 0, sf.GATE["full"], sf.ACT["silu"], 0.5, 1e-5,
                            x.device.index, C, C, C)
    assert sf.lib().sffft_block_norm(ctypes.byref(desc), p(x), p(y), p(gate), p(pw), p(w), p(x), p(y), None, None,
                                     torch.cuda.current_stream().cuda_stream) == sf.OK
    assert torch.equal(x, h) and torch.equal(y, n)


@pytest.mark.parametrize("C,groups", [(96, 96), (800, 200), (8191, 8191)])
def test_groups_of_a_few_channels(C, groups):
    t, dh, dn = make((5, C), -1, F32, F32, seed=groups)
    check(t, dh, dn, groups)


def test_groups_without_the_norm_of_y():
    for shape, dim in (((3, 5, 96), -1), ((2, 96, 36), 1)):
        t, dh, dn = make(shape, dim, BF, F32, post=False)
        kw = dict(scale=0.5, act="silu", dim=dim)
        for f in (sf.block_norm, ops.block_norm):
            assert all(torch.equal(a, b) for a, b in zip(f(**t, **kw, groups=8), f(**t, **kw)))
        r2 = sf.block_norm(**t, **kw, stats=True)[3]
        a, b = (sf.block_norm_backward(dh, dn, **t, rstd=r2, **kw, groups=g) for g in (8, 1))
        assert all(x is y or torch.equal(x, y) for x, y in zip(a, b))


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 values apart."""
    C, far = 96, (1 << 31) + 32
    buf = torch.empty(far + 3 * C, dtype=BF, device="cuda")
    t, dh, dn = make((2, C), -1, BF, BF)
    for i, name in enumerate(("x", "y", "gate")):
        view = torch.as_strided(buf, (2, C), (far, 1), i * C)
        view.copy_(t[name])
        t[name] = view
    check(t, dh, dn, 4)


def test_layouts_agree():
    """[B][C][L] and [B][L][C] give the same numbers, up to the order of the sums over channels."""
    t, dh, dn = make((2, 64, 48), 1, F32, F32)
    a = check(t, dh, dn, 4, dim=1)
    rows = {n: w if w is None or w.dim() == 1 else w.transpose(1, 2).contiguous() for n, w in t.items()}
    b = check(rows, dh.transpose(1, 2).contiguous(), dn.transpose(1, 2).contiguous(), 4)
    for n in a:
        x = a[n].transpose(1, 2) if a[n].dim() == 3 else a[n]
        assert (x - b[n]).abs().max() <= 1e-5 * b[n].abs().max(), n
