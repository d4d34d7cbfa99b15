"""Linear attention with a decay for each head on the device: values, states and gradients against the definition in 64
bits, at the sizes where a kernel changes its way; lengths, strides, streams, graphs and the single-token form."""
import pytest
import torch

import sffft_b200 as sf
import sffft_b200.torch_ops as ops
from tests import mixer_ref as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def decays(H, device, kind="mixed"):
    h = torch.arange(H, dtype=torch.float64)
    ld = torch.log1p(-torch.exp2(-(1 + 9 * h / max(1, H - 1))))     # lambda 1/2 ... 1 - 2^-10
    if kind == "edges":
        ld[0] = 0.0                                                  # no decay
        if H > 1:
            ld[1] = -float("inf")                                    # no memory
        if H > 2:
            ld[2] = -40.0                                            # lambda^m leaves fp32 within a few tokens
    return ld.float().to(device)


def make(B, H, Hkv, L, D, Dv, dtype, seed=0, token_major=False, state=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    def heads(n, d):
        return r(B, L, n, d).to(dtype).transpose(1, 2) if token_major else r(B, n, L, d).to(dtype)
    t = dict(q=heads(H, D), k=heads(Hkv, D), v=heads(Hkv, Dv), dy=heads(H, Dv))
    t["s0"] = r(B, H, D, Dv) if state else None
    t["ds"] = r(B, H, D, Dv) if state else None
    return t


def check(t, ld, scale, lengths=None, backward=True):
    q, k, v = t["q"], t["k"], t["v"]
    B, H, L, D = q.shape
    Dv = v.shape[3]
    want = ref.attention(q, k, v, ld, scale, t["s0"], lengths, t["dy"] if backward else None, t["ds"])
    got = dict(zip(("y", "state"), sf.linear_attention(q, k, v, ld, scale, t["s0"], lengths)))
    if backward:
        got.update(zip(("dq", "dk", "dv", "ds0"), sf.linear_attention_backward(q, k, v, ld, t["dy"], t["ds"], scale, t["s0"],
                                                                              lengths)))
    for name, x in got.items():
        if x is None:
            continue
        value, mag = want[name]
        assert x.shape == value.shape and x.dtype == (F32 if name in ("state", "ds0") else q.dtype)
        off = (x.double() - value).abs()
        tol = ref.attention_bound(name, value, mag, q.dtype, L, D, Dv, H // k.shape[1])
        assert torch.isfinite(x).all(), name
        bad = off > tol
        assert not bad.any(), (name, off[bad].max().item(), (off / tol).max().item(), bad.nonzero()[0].tolist())
    sf.linear_attention_check()
    return got


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("L", [1, 2, 31, 63, 64, 65, 127, 128, 129, 255, 257, 640, 1500])
def test_lengths_of_one_head(L, dtype):
    check(make(2, 3, 3, L, 64, 64, dtype, L), decays(3, "cuda"), 0.125)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D,Dv", [(1, 1), (3, 5), (8, 8), (16, 40), (40, 16), (64, 128), (128, 64), (72, 96), (96, 72), (128, 128),
                                  (100, 20), (130, 24), (24, 136), (256, 256), (65, 64)])
def test_head_sizes(D, Dv, dtype):
    check(make(1, 2, 2, 200, D, Dv, dtype, D), decays(2, "cuda"), D ** -0.5)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("H,Hkv", [(4, 1), (6, 2), (6, 3), (5, 5)])
@pytest.mark.parametrize("token_major", [False, True])
def test_shared_heads_and_order_of_axes(H, Hkv, token_major, dtype):
    t = make(2, H, Hkv, 333, 64, 64, dtype, H, token_major)
    got = check(t, decays(H, "cuda"), 0.125)
    if token_major and Hkv > 1:
        assert got["y"].transpose(1, 2).is_contiguous() and got["dk"].transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("state", [False, True])
def test_lengths_of_rows(state, dtype):
    L = 700
    t = make(8, 2, 1, L, 64, 128, dtype, 5, True, state)
    n = torch.tensor([L, 0, 1, 64, 129, 511, 256, L + 9], dtype=torch.int32, device="cuda")
    for name in ("q", "k", "v", "dy"):     # whatever lies behind a row's last token
        for b in range(8):
            t[name][b, :, min(int(n[b]), L):] = float("nan") if b % 2 else float("inf")
    got = check(t, decays(2, "cuda"), 0.3, n)
    for name in ("y", "dq", "dk", "dv"):
        for b in range(8):
            assert (got[name][b, :, min(int(n[b]), L):] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H", [(2, 90), (9, 20), (31, 6), (32, 8), (33, 6), (32, 20)])
def test_many_rows_of_many_lengths(B, H, dtype):
    """More blocks than run at once, which may take the longest rows first; some of one length."""
    L = 140
    t = make(B, H, 2, L, 64, 64, dtype, B, True)
    n = torch.randint(0, L + 1, (B,), device="cuda", dtype=torch.int32, generator=torch.Generator("cuda").manual_seed(B))
    n[1::4] = 77
    check(t, decays(H, "cuda"), 0.3, n)


@pytest.mark.parametrize("D,Dv", [(64, 64), (64, 128), (128, 64), (128, 128), (96, 72)])
@pytest.mark.parametrize("L", [2, 3, 130])
def test_states_of_bf16_rows_are_exact_to_32_bits(L, D, Dv):
    """Fast decay, so that a state is a sum of few terms lambda^m k v.  Each term is a product of 24 + 8 + 8 bits: lambda^m
    and its product with k are off by 2 and 1 half steps of fp32, the three bf16 parts of that leave less than one, and of
    the up to 3 * 16 additions (16 positions an instruction) of a row's last positions each truncates: 2^-23 of the
    magnitude.  Terms further back than 16 positions weigh less than e^-64.  64 * 2^-23 holds them all."""
    t = make(2, 3, 3, L, D, Dv, BF, L + D, state=False)
    ld = torch.tensor([-4.0, -4.7, -5.3], device="cuda")
    value, mag = ref.attention(t["q"], t["k"], t["v"], ld, 0.125)["state"]
    _, s = sf.linear_attention(t["q"], t["k"], t["v"], ld, 0.125)
    off = (s.double() - value).abs()
    # a tenth of that where it is the usual: two roundings to bf16 would leave 2^-17 = 64 * 2^-23 at the most, 2^-19 usually
    assert (off <= 64 * 2.0 ** -23 * mag).all()
    assert torch.linalg.norm(off) <= 4 * 2.0 ** -23 * torch.linalg.norm(value)
    ds = torch.zeros_like(s)
    value, mag = ref.attention(t["q"], t["k"], t["v"], ld, 0.125, ds, None, t["dy"], ds)["ds0"]
    d0 = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], ds, 0.125, ds)[3]
    off = (d0.double() - value).abs()
    assert (off <= 64 * 2.0 ** -23 * mag).all()
    assert torch.linalg.norm(off) <= 4 * 2.0 ** -23 * torch.linalg.norm(value)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_decays_at_the_ends_of_their_range(dtype):
    check(make(1, 4, 4, 400, 64, 64, dtype, 9), decays(4, "cuda", "edges"), 0.125)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("D", [64, 128])
def test_long_rows_of_few_heads_are_cut(D, dtype):
    n = torch.tensor([5000, 3210], dtype=torch.int32, device="cuda")
    check(make(2, 2, 2, 5000, D, D, dtype, 11), decays(2, "cuda"), D ** -0.5)
    check(make(2, 2, 1, 5000, D, D, dtype, 12), decays(2, "cuda"), D ** -0.5, n)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_many_heads(dtype):
    check(make(20, 16, 16, 130, 64, 64, dtype, 13, state=False), decays(16, "cuda"), 0.125)


def test_parts_of_a_fused_projection_and_odd_strides():
    L, H, D = 300, 3, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    ld = decays(H, "cuda")
    for width in (3 * H * D, 3 * H * D + 8, 3 * H * D + 1):     # the last one leaves rows at odd addresses
        buf = torch.randn((2, L, width), device="cuda", generator=g).to(BF)
        q, k, v = (buf[..., i * H * D:(i + 1) * H * D].view(2, L, H, D).transpose(1, 2) for i in range(3))
        t = dict(q=q, k=k, v=v, dy=torch.randn((2, H, L, D), device="cuda", generator=g).to(BF), s0=None, ds=None)
        check(t, ld, 0.125)
    t = make(1, H, H, L, D, D, BF, 3)
    t["q"] = torch.randn((1, H, D, L), device="cuda", generator=g).to(BF).transpose(2, 3)    # values not contiguous
    t["dy"] = torch.ones((), device="cuda", dtype=BF).expand(1, H, L, D)
    check(t, ld, 0.125)


def test_no_tokens_and_no_rows():
    ld = decays(2, "cuda")
    t = make(3, 2, 2, 0, 64, 64, BF)
    y, s = sf.linear_attention(t["q"], t["k"], t["v"], ld, 1.0, t["s0"])
    assert y.shape == (3, 2, 0, 64) and torch.equal(s, t["s0"])
    out = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 1.0, t["s0"])
    assert out[0].shape == (3, 2, 0, 64) and (out[3] - t["ds"]).abs().max() <= 2.0 ** -22 * t["ds"].abs().max()
    t = make(0, 2, 2, 5, 64, 64, BF)
    y, s = sf.linear_attention(t["q"], t["k"], t["v"], ld)
    assert y.shape == (0, 2, 5, 64) and s.shape == (0, 2, 64, 64)


def test_results_do_not_change_from_call_to_call():
    t = make(2, 4, 2, 3000, 64, 64, BF, 4, True)
    ld = decays(4, "cuda")
    n = torch.tensor([3000, 1234], dtype=torch.int32, device="cuda")
    a = sf.linear_attention(t["q"], t["k"], t["v"], ld, 0.125, t["s0"], n)
    b = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 0.125, t["s0"], n)
    for _ in range(3):
        assert all(torch.equal(x, z) for x, z in zip(a, sf.linear_attention(t["q"], t["k"], t["v"], ld, 0.125, t["s0"], n)))
        c = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 0.125, t["s0"], n)
        assert all(torch.equal(x, z) for x, z in zip(b, c))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_pieces_of_a_row_give_the_row(dtype):
    """A row in one call, and in pieces that hand on their state: states agree to the sums' rounding, y to its type's."""
    t = make(1, 3, 3, 900, 64, 64, dtype, 6, state=False)
    ld = decays(3, "cuda")
    q, k, v = t["q"], t["k"], t["v"]
    want = ref.attention(q, k, v, ld, 0.125)
    s, ys = None, []
    for a, b in ((0, 1), (1, 130), (130, 386), (386, 900)):
        y, s = sf.linear_attention(q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], ld, 0.125, s)
        ys.append(y)
    for name, x in (("y", torch.cat(ys, 2)), ("state", s)):
        value, mag = want[name]
        assert ((x.double() - value).abs() <= ref.attention_bound(name, value, mag, dtype, 900, 64, 64)).all(), name


def test_convolution_with_an_exponential_filter():
    """With D = Dv = 1 and q = k = 1 the operator is the framework's convolution with the filter lambda^n."""
    H, L = 6, 1024
    ld = decays(H, "cuda")
    u = torch.randn((2, H, L), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    k = torch.exp(ld.double()[:, None] * torch.arange(L, device="cuda")).float()
    conv = ops.causal_conv(u, k)
    one = torch.ones((2, H, L, 1), device="cuda")
    y, _ = ops.linear_attention(one, one, u[..., None].contiguous(), ld)
    # the convolution holds 5e-4 in relative L2; linear attention adds 1e-5 at most
    assert torch.linalg.norm(conv - y[..., 0]) <= 5.1e-4 * torch.linalg.norm(y)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_gradients_through_autograd_and_against_differences(dtype):
    """The loss <y, dy> + <S, ds> is linear in each of q, k, v and S_0, so a central difference of any width is exact."""
    B, H, Hkv, L, D, Dv = 2, 4, 2, 150, 64, 64
    t = make(B, H, Hkv, L, D, Dv, dtype, 8, True)
    ld = decays(H, "cuda")
    names = ("q", "k", "v", "s0")
    leaves = [t[n].clone().requires_grad_() for n in names]
    y, s = ops.linear_attention(*leaves[:3], ld, 0.125, leaves[3])
    grads = torch.autograd.grad([y, s], leaves, [t["dy"], t["ds"]])
    direct = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 0.125, t["s0"])
    assert all(torch.equal(a, b) for a, b in zip(grads, direct))

    def loss(args):
        out = ref.attention(*args[:3], ld, 0.125, args[3])
        return (out["y"][0] * t["dy"].double()).sum() + (out["state"][0] * t["ds"].double()).sum()

    g = torch.Generator(device="cuda").manual_seed(3)
    want = ref.attention(t["q"], t["k"], t["v"], ld, 0.125, t["s0"], None, t["dy"], t["ds"])
    for i, (n, grad) in enumerate(zip(names, grads)):
        way = torch.randn(t[n].shape, device="cuda", generator=g).double()
        args = [t[m].double() for m in names]
        up = loss(args[:i] + [args[i] + way] + args[i + 1:])
        down = loss(args[:i] + [args[i] - way] + args[i + 1:])
        value, mag = want[{"s0": "ds0"}.get(n, "d" + n)]
        tol = (ref.attention_bound({"s0": "ds0"}.get(n, "d" + n), value, mag, dtype, L, D, Dv, 2) * way.abs()).sum()
        assert ((up - down) / 2 - (grad.double() * way).sum()).abs() <= tol + 1e-9 * up.abs(), n


def test_autograd_of_one_output_alone():
    t = make(1, 2, 2, 100, 64, 64, F32, 2)
    ld = decays(2, "cuda")
    q, k, v = (t[n].clone().requires_grad_() for n in "qkv")
    y, s = ops.linear_attention(q, k, v, ld)
    y.sum().backward(retain_graph=True)
    want = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, torch.ones_like(t["dy"]))
    assert all(torch.equal(a.grad, b) for a, b in zip((q, k, v), want))
    gk, gv = torch.autograd.grad(s.sum(), [k, v])
    want = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, torch.zeros_like(t["dy"]), torch.ones_like(s))
    assert torch.equal(gk, want[1]) and torch.equal(gv, want[2])
    with pytest.raises(RuntimeError):     # no second derivative
        g, = torch.autograd.grad(ops.linear_attention(q, k, v, ld)[0].sum(), [q], create_graph=True)
        g.sum().backward()


def test_streams_graphs_and_compile():
    t = make(2, 4, 4, 2000, 64, 64, BF, 4, True)
    ld = decays(4, "cuda")
    args = (t["q"], t["k"], t["v"], ld, 0.125, t["s0"])
    want = sf.linear_attention(*args)
    back = sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 0.125, t["s0"])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        got = sf.linear_attention(*args, stream=stream)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(side):
        got = ops.linear_attention(*args)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs, replayed at once on two streams: their workspaces are their own
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = sf.linear_attention(*args)
            o = o + sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 0.125, t["s0"])
        graphs.append(g)
        outs.append(o)
    t["v"].mul_(2)     # exact in bf16
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    want2 = sf.linear_attention(*args) + sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], t["ds"], 0.125, t["s0"])
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want2))
    t["v"].div_(2)
    compiled = torch.compile(lambda q, k, v, s: ops.linear_attention(q, k, v, ld, 0.125, s), fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(compiled(t["q"], t["k"], t["v"], t["s0"]), want))
    del back


def test_training_step_under_compile():
    t = make(2, 4, 2, 300, 64, 64, BF, 15, True)
    ld = decays(4, "cuda")
    names = ("q", "k", "v", "s0")

    def loss(q, k, v, s0):
        y, s = ops.linear_attention(q, k, v, ld, 0.125, s0)
        return (y * t["dy"]).sum(dtype=torch.float32) + (s * t["ds"]).sum()

    grads = []
    for f in (loss, torch.compile(loss, fullgraph=True)):
        leaves = [t[n].clone().requires_grad_() for n in names]
        f(*leaves).backward()
        grads.append([x.grad for x in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_training_step_in_a_graph():
    """Forward and backward captured, with gradients in buffers of their own, and replayed on new values."""
    t = make(2, 4, 2, 300, 64, 64, BF, 16, True)
    ld = decays(4, "cuda")
    leaves = [t[n].clone().requires_grad_() for n in ("q", "k", "v")]

    def step():
        y, _ = ops.linear_attention(*leaves, ld, 0.125)
        return torch.autograd.grad(y, leaves, t["dy"])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    with torch.no_grad():
        leaves[1].mul_(2)
    g.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_threads_of_their_own():
    """Calls from threads that have made no CUDA call yet (autograd's are such), while others call too."""
    import threading
    t = make(2, 4, 4, 500, 64, 64, BF, 14)
    ld = decays(4, "cuda")
    want = sf.linear_attention(t["q"], t["k"], t["v"], ld, 0.125, t["s0"])
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = [sf.linear_attention(t["q"], t["k"], t["v"], ld, 0.125, t["s0"]) for _ in range(20)]
            torch.cuda.current_stream().synchronize()

    for n in (1, 4):      # the second time with memory at hand, so that nothing else touches CUDA first
        threads = [threading.Thread(target=work, args=(i,)) for i in range(n)]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
        assert len(got) == n
        assert all(torch.equal(a, b) for runs in got.values() for o in runs for a, b in zip(o, want))
        got.clear()
    q = t["q"].clone().requires_grad_()
    y, _ = ops.linear_attention(q, t["k"], t["v"], ld, 0.125, t["s0"])
    y.backward(t["dy"])
    assert torch.equal(q.grad, sf.linear_attention_backward(t["q"], t["k"], t["v"], ld, t["dy"], None, 0.125, t["s0"])[0])


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 values apart."""
    H, L, D = 2, 260, 64
    far = (1 << 31) + 64
    buf = torch.empty(far + 3 * H * L * D, dtype=BF, device="cuda")
    t = make(2, H, H, L, D, D, BF, 7, state=False)
    for i, n in enumerate("qkv"):
        view = torch.as_strided(buf, (2, H, L, D), (far, L * D, D, 1), i * H * L * D)
        view.copy_(t[n])
        t[n] = view
    check(t, decays(H, "cuda"), 0.125)


# ---------------------------------------------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------------------------------------------

def step_ref(q, k, v, ld, state, scale):
    H = q.shape[1]
    kk, vv = (t.double().repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    a = torch.exp(ld.double().clamp(min=-1e30))[None, :, None, None]
    s = a * state.double() + kk[..., None] * vv[..., None, :]
    smag = a * state.double().abs() + (kk[..., None] * vv[..., None, :]).abs()
    y = scale * (q.double()[..., None] * s).sum(2)
    ymag = abs(scale) * (q.double().abs()[..., None] * smag).sum(2)
    return s, smag, y, ymag


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("B,H,Hkv,D,Dv", [(1, 1, 1, 1, 1), (1, 12, 12, 64, 64), (3, 4, 2, 128, 128), (2, 3, 1, 40, 33),
                                          (5, 2, 2, 65, 100), (33, 2, 2, 256, 32), (200, 8, 8, 64, 64)])
def test_step(B, H, Hkv, D, Dv, dtype):
    g = torch.Generator(device="cuda").manual_seed(B + D)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v = r(B, H, D).to(dtype), r(B, Hkv, D).to(dtype), r(B, Hkv, Dv).to(dtype)
    pool = B + 3
    state, ld = r(pool, H, D, Dv), decays(H, "cuda", "edges" if H > 2 else "mixed")
    slots = torch.randperm(pool, generator=g, device="cuda")[:B].to(torch.int32)
    before = state.clone()
    s, smag, y, ymag = step_ref(q, k, v, ld, before[slots.long()], 0.25)
    got = ops.linear_attention_step(q, k, v, ld, state, slots, 0.25)
    # two roundings in a state, D + 2 in y, each of half a step of fp32; lambda itself is off by two
    assert ((state[slots.long()].double() - s).abs() <= 2.0 ** -22 * smag).all()
    assert ((got.double() - y).abs() <= (D + 8) * 2.0 ** -24 * ymag + ref.HALF_STEP[dtype] * y.abs()).all()
    rest = torch.ones(pool, dtype=torch.bool, device="cuda")
    rest[slots.long()] = False
    assert torch.equal(state[rest], before[rest])
    again = before.clone()
    assert torch.equal(ops.linear_attention_step(q, k, v, ld, again[:B], None, 0.25),
                       ops.linear_attention_step(q, k, v, ld, before.clone(), torch.arange(B, dtype=torch.int32, device="cuda"), 0.25))


def test_step_with_padded_rows_and_a_slot_named_twice():
    B, H, D = 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v, state = r(B, H, D), r(B, H, D), r(B, H, D), r(4, H, D, D)
    ld = decays(H, "cuda")
    slots = torch.tensor([2, -1, 0, 2, 4, 2], dtype=torch.int32, device="cuda")
    before = state.clone()
    y = ops.linear_attention_step(q, k, v, ld, state, slots)
    assert (y[[1, 3, 4, 5]] == 0).all()
    alone = before.clone()
    want = ops.linear_attention_step(q[[0, 2]], k[[0, 2]], v[[0, 2]], ld, alone, slots[[0, 2]])
    assert torch.equal(y[[0, 2]], want) and torch.equal(state, alone)
    assert torch.equal(state[[1, 3]], before[[1, 3]])


def test_step_without_a_pool():
    q = torch.ones((2, 3, 16), device="cuda")
    y = ops.linear_attention_step(q, q, q, decays(3, "cuda"), torch.empty((0, 3, 16, 16), device="cuda"),
                                  torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert (y == 0).all()


def test_step_marks_its_state_as_changed():
    q = torch.ones((1, 1, 16), device="cuda")
    s = torch.zeros((1, 1, 16, 16), device="cuda")
    x = torch.ones((1, 1, 16, 16), device="cuda", requires_grad=True)
    z = (x * s).sum()
    with torch.no_grad():
        ops.linear_attention_step(q, q, q, decays(1, "cuda"), s)
    with pytest.raises(RuntimeError):     # s was needed as it was
        z.backward()


def test_step_continues_a_prompt():
    """A prompt and then single tokens give the same as the whole row at once, within the bounds of both."""
    B, H, L, D = 2, 4, 150, 64
    t = make(B, H, H, L, D, D, BF, 21, True, state=False)
    ld = decays(H, "cuda")
    want = ref.attention(t["q"], t["k"], t["v"], ld, 0.125)
    y, s = ops.linear_attention(t["q"][:, :, :140], t["k"][:, :, :140], t["v"][:, :, :140], ld, 0.125)
    pool = torch.zeros((5, H, D, D), device="cuda")
    slots = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    pool[slots.long()] = s
    ys = [y] + [ops.linear_attention_step(t["q"][:, :, i], t["k"][:, :, i], t["v"][:, :, i], ld, pool, slots, 0.125)[:, :, None]
                for i in range(140, L)]
    for name, x in (("y", torch.cat(ys, 2)), ("state", pool[slots.long()])):
        value, mag = want[name]
        assert ((x.double() - value).abs() <= ref.attention_bound(name, value, mag, BF, L, D, D)).all(), name


def test_step_in_a_graph_and_under_compile():
    B, H, D = 3, 2, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v, state = r(B, H, D).to(BF), r(B, H, D).to(BF), r(B, H, D).to(BF), r(B, H, D, D)
    ld = decays(H, "cuda")
    start = state.clone()
    ys = [ops.linear_attention_step(q, k, v, ld, state) for _ in range(3)]
    end = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear_attention_step(q, k, v, ld, state)
    state.copy_(start)
    for want in ys:
        graph.replay()
        assert torch.equal(y, want)
    assert torch.equal(state, end)
    state.copy_(start)
    step = torch.compile(lambda s: ops.linear_attention_step(q, k, v, ld, s), fullgraph=True)
    assert torch.equal(step(state), ys[0])


def test_step_in_a_pool_beyond_32_bits():
    H, D = 16, 128
    pool = (1 << 31) // (H * D * D) + 2
    state = torch.empty((pool, H, D, D), device="cuda")
    slots = torch.tensor([pool - 1, 0], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v, small = r(2, H, D), r(2, H, D), r(2, H, D), r(2, H, D, D)
    state[pool - 1], state[0] = small[0], small[1]
    ld = decays(H, "cuda")
    y = ops.linear_attention_step(q, k, v, ld, state, slots)
    assert torch.equal(y, ops.linear_attention_step(q, k, v, ld, small))
    assert torch.equal(state[pool - 1], small[0]) and torch.equal(state[0], small[1])
