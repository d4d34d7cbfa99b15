"""The operators together, as the layers of a model use them: norm, linear attention or the convolution, norm by heads with
gate, residual stream, norm; prompts, single tokens and training."""
import ctypes

import pytest
import torch

import sffft_b200 as sf
import sffft_b200.torch_ops as ops
from tests import mixer_ref as ref

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
B, L, H, D = 2, 200, 6, 64
C = H * D


def weights(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    return dict(wn=1 + 0.1 * r(C), wp=1 + 0.1 * r(C), w2=1 + 0.1 * r(C), win=r(4 * C, C) * C ** -0.5, wout=r(C, C) * C ** -0.5,
                x=r(B, L, C), ld=torch.log1p(-torch.exp2(-torch.linspace(3, 9, H, device="cuda"))))


def layer(w, x, mix, norm):
    """h, n of one layer: x + block(norm(x)), and the next layer's norm of it.  `mix`(q, k, v) and `norm`(**) are the two
    operators, in the framework's form or in 64 bits."""
    n, dt = norm(x=x, weight=w["wn"])[1], x.dtype
    q, k, v, gate = (n @ w["win"].to(n.dtype).T).unflatten(-1, (4, H, D)).unbind(-3)
    y = mix(*(t.transpose(1, 2) for t in (q, k, v))).transpose(1, 2).flatten(2)
    a = norm(y=y, gate=gate.flatten(2), post_weight=w["wp"], groups=H, act="silu")[0]
    return norm(x=x, y=(a @ w["wout"].to(a.dtype).T).to(dt), weight=w["w2"], scale=0.5)


def exact_norm(x=None, y=None, gate=None, post_weight=None, weight=None, scale=1.0, groups=1, act="none"):
    out = ref.norm(x, y, gate, post_weight, weight, scale, 1e-6, groups, act, -1)
    return x if y is None else out["h"], out.get("n")


def test_a_layer_and_its_gradients():
    """In fp32 against 64 bits.  Four products of C terms, two norms and the attention's sums follow each other, each off by
    at most (C + 600) half steps of fp32 of its magnitude; conditions of the norms are below 2.  16 times that of the
    largest value holds the chain."""
    w = weights()
    tol = 16 * (C + 600) * 2.0 ** -24
    x = w["x"].clone().requires_grad_()
    win = w["win"].clone().requires_grad_()
    h, n = layer(dict(w, win=win), x, lambda q, k, v: ops.linear_attention(q, k, v, w["ld"], D ** -0.5)[0], ops.block_norm)
    dh, dn = torch.randn_like(h), torch.randn_like(n)
    got = (h, n) + torch.autograd.grad([h, n], [x, win], [dh, dn])
    xd, wd = w["x"].double().requires_grad_(), w["win"].double().requires_grad_()
    w64 = {k: t.double() for k, t in w.items()}

    def mix(q, k, v):
        lag = torch.arange(L, device="cuda")[:, None] - torch.arange(L, device="cuda")[None]
        a = torch.where(lag >= 0, torch.exp(w64["ld"][:, None, None] * lag.clamp(min=0)), 0.0)
        return D ** -0.5 * ((q @ k.transpose(2, 3)) * a) @ v

    h6, n6 = layer(dict(w64, win=wd), xd, mix, exact_norm)
    want = (h6, n6) + torch.autograd.grad([h6, n6], [xd, wd], [dh.double(), dn.double()])
    for a, b in zip(got, want):
        assert (a.double() - b).abs().max() <= tol * b.abs().max()


def test_prompt_and_tokens_of_a_layer_in_bf16():
    """A prompt, then single tokens, give what the whole row gives: the two differ in the roundings of y alone, which are
    carried through the layer.  y's is 2 half steps of its magnitude; the norm by heads and the output's product pass it
    on, and each value after is rounded again: 16 half steps of the largest value."""
    w = weights(1)
    x = w["x"]
    attn = lambda q, k, v: ops.linear_attention(q, k, v, w["ld"], D ** -0.5)[0]  # noqa: E731
    cast = lambda f: lambda *t: f(*(u.to(BF) for u in t)).to(F32)  # noqa: E731
    h, n = layer(w, x, cast(attn), ops.block_norm)
    cut = 190
    pool = torch.zeros((4, H, D, D), device="cuda")
    slots = torch.tensor([2, 0], dtype=torch.int32, device="cuda")

    def prompt(q, k, v):
        y, s = ops.linear_attention(q, k, v, w["ld"], D ** -0.5)
        pool[slots.long()] = s
        return y

    def token(q, k, v):
        return ops.linear_attention_step(*(t[:, :, 0] for t in (q, k, v)), w["ld"], pool, slots, D ** -0.5)[:, :, None]

    hs, ns = zip(layer(w, x[:, :cut], cast(prompt), ops.block_norm),
                 *(layer(w, x[:, i:i + 1], cast(token), ops.block_norm) for i in range(cut, L)))
    for a, b in ((torch.cat(hs, 1), h), (torch.cat(ns, 1), n)):
        assert (a - b).abs().max() <= 16 * 2.0 ** -8 * b.abs().max()


def test_the_convolution_between_its_norms():
    """norm before, convolution, gate and norm behind it, in the convolution's own [B][C][L]: its error bound of 5e-4 in
    relative L2 enters a; the norm divides by rms(y), so h's error is at most that of a, once for y and once for its rms."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    Bc, Cc, Lc = 2, 48, 256
    x, gate, w1, w2, wp = r(Bc, Cc, Lc), r(Bc, Cc, Lc), 1 + 0.1 * r(Cc), 1 + 0.1 * r(Cc), 1 + 0.1 * r(Cc)
    k = r(Cc, Lc) * torch.exp(-4 * torch.arange(Lc, device="cuda") / Lc) * Lc ** -0.5
    _, n = ops.block_norm(x, weight=w1, dim=1)
    y = ops.causal_conv(n, k)
    h, n2 = ops.block_norm(x, y, gate, wp, w2, scale=0.5, act="sigmoid", dim=1)
    n64 = ref.norm(x, None, None, None, w1, 1.0, 1e-6, 1, "none", 1)["n"]
    N = 2 * Lc
    y64 = torch.fft.irfft(torch.fft.rfft(n64, N) * torch.fft.rfft(k.double(), N), N)[..., :Lc]
    want = ref.norm(x, y64, gate, wp, w2, 0.5, 1e-6, 1, "sigmoid", 1)
    a = want["h"] - x.double()
    assert torch.linalg.norm(h.double() - want["h"]) <= 2 * 5.1e-4 * torch.linalg.norm(a) + 1e-6 * torch.linalg.norm(want["h"])
    assert torch.linalg.norm(n2.double() - want["n"]) <= 4 * 5.1e-4 * torch.linalg.norm(want["n"])


@pytest.mark.parametrize("dtype", [F32, BF])
def test_calls_without_their_workspace_are_refused(dtype):
    """In C, where the workspace is the caller's: the call does nothing, and with what was asked for it gives Python's results."""
    lib, io = sf.lib(), sf.IO["bf16" if dtype == BF else "fp32"]
    st = torch.cuda.current_stream().cuda_stream
    Hq, Hk, Lq = 2, 1, 2048
    q, k, v = (torch.randn((1, n, Lq, D), device="cuda").to(dtype) for n in (Hq, Hk, Hk))
    ld = torch.tensor([-0.01, -0.1], device="cuda")
    y, s = torch.full_like(q, 7), torch.full((1, Hq, D, D), 7.0, device="cuda")
    three = ctypes.c_longlong * 3
    sq, sk = three(Hq * Lq * D, Lq * D, D), three(Hk * Lq * D, Lq * D, D)
    desc = sf.LinearAttentionDesc(1, Hq, Hk, Lq, D, D, io, q.device.index, 0.125, sq, sk, sk, sq)
    need = ctypes.c_size_t()
    p = lambda t: t.data_ptr()  # noqa: E731

    def forward(work, n):
        return lib.sffft_linear_attention(ctypes.byref(desc), p(q), p(k), p(v), p(ld), None, None, p(y), p(s), work, n, st)

    assert forward(None, 0) == sf.ERR_WORKSPACE
    assert (y == 7).all() and (s == 7).all()
    assert lib.sffft_linear_attention_workspace_bytes(ctypes.byref(desc), 0, ctypes.byref(need)) == sf.OK and need.value > 0
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    assert forward(p(work), 256) == sf.ERR_WORKSPACE and (y == 7).all()
    assert forward(p(work), need.value) == sf.OK
    assert all(torch.equal(a, b) for a, b in zip((y, s), sf.linear_attention(q, k, v, ld, 0.125)))

    dy = torch.randn_like(q)
    dq, dk, dv = (torch.full_like(t, 7) for t in (q, k, v))
    grads = sf.LinearAttentionGrads(sq, sq, sk, sk)

    def backward(work, n):
        return lib.sffft_linear_attention_backward(ctypes.byref(desc), ctypes.byref(grads), p(q), p(k), p(v), p(ld), None, None, p(dy),
                                                   None, p(dq), p(dk), p(dv), None, work, n, st)

    assert backward(None, 0) == sf.ERR_WORKSPACE
    assert lib.sffft_linear_attention_workspace_bytes(ctypes.byref(desc), 1, ctypes.byref(need)) == sf.OK
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    assert backward(p(work), 1 << 20) == sf.ERR_WORKSPACE
    assert all((t == 7).all() for t in (dq, dk, dv))
    assert backward(p(work), need.value) == sf.OK
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), sf.linear_attention_backward(q, k, v, ld, dy, None, 0.125)))

    x, w = torch.randn((50, 64), device="cuda").to(dtype), torch.ones(64, device="cuda")
    _, _, _, r = sf.block_norm(x, weight=w, stats=True)
    dn, dx, dw = torch.randn_like(x), torch.full_like(x, 7), torch.full_like(w, 7)
    bn = sf.BlockNormDesc(50, 64, 0, 1, io, io, 0, 0, 0, 1.0, 1e-6, x.device.index, 64, 0, 0)

    def norm_backward(work, n):
        return lib.sffft_block_norm_backward(ctypes.byref(bn), p(x), None, None, None, p(w), None, p(r), None, p(dn), p(dx), None, None,
                                             None, p(dw), work, n, st)

    assert norm_backward(None, 0) == sf.ERR_WORKSPACE and (dx == 7).all() and (dw == 7).all()
    assert lib.sffft_block_norm_workspace_bytes(ctypes.byref(bn), ctypes.byref(need)) == sf.OK
    work = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    assert norm_backward(p(work), need.value) == sf.OK
    got = sf.block_norm_backward(None, dn, x, weight=w, rstd=r)
    assert torch.equal(dx, got[0]) and torch.equal(dw, got[4])
