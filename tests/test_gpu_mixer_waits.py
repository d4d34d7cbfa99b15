"""Waits of the tensor-core linear attention kernel that run out: one thread leaves out an arrival, with every wait limited to
2 ms; all roles leave, the status says so, and the next call on the same context gives what it gave before (a block that kept
its TMEM would block every later one on its SM)."""
import contextlib
import os
import subprocess
import sys

import pytest
import torch

import sffft_b200 as sf

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
X, SCALED, STAGED = 1, 2, 3


@contextlib.contextmanager
def withheld(what, limit_us=2000):
    assert sf.lib().sffft_debug_linear_attention(limit_us, what) == sf.OK
    try:
        yield
    finally:
        assert sf.lib().sffft_debug_linear_attention(0, 0) == sf.OK


# both head sizes of the kernel, few and many chunks, rows cut into segments, shared heads (their gradients are written in
# fp32 by the warps themselves), a state in and out
SHAPES = [(1, 2, 2, 100, 64, 64), (2, 3, 3, 1000, 64, 64), (1, 2, 2, 100, 128, 128), (2, 2, 2, 700, 128, 64), (1, 2, 2, 5000, 64, 64),
          (1, 2, 2, 5000, 128, 128), (2, 4, 2, 300, 64, 64), (2, 4, 1, 600, 128, 128)]


@pytest.mark.parametrize("what", [X, SCALED, STAGED])
@pytest.mark.parametrize("shape", SHAPES)
def test_all_roles_leave_when_a_wait_runs_out(shape, what):
    B, H, Hkv, L, D, Dv = shape
    g = torch.Generator(device="cuda").manual_seed(L)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v, dy = r(B, H, L, D).to(BF), r(B, Hkv, L, D).to(BF), r(B, Hkv, L, Dv).to(BF), r(B, H, L, Dv).to(BF)
    ld, s0 = torch.full((H,), -0.1, device="cuda"), r(B, H, D, Dv)
    forward = lambda: sf.linear_attention(q, k, v, ld, 0.125, s0)  # noqa: E731
    backward = lambda: sf.linear_attention_backward(q, k, v, ld, dy, s0, 0.125, s0)  # noqa: E731
    for call in (forward, backward):
        want = call()
        sf.linear_attention_check()
        with withheld(what):
            call()
        with pytest.raises(sf.SffftError) as e:
            sf.linear_attention_check()
        assert e.value.status == sf.ERR_TIMEOUT
        sf.linear_attention_check()          # the check cleared the status
        assert all(torch.equal(a, b) for a, b in zip(call(), want))
        sf.linear_attention_check()


def test_later_calls_raise_until_the_status_is_cleared():
    import sffft_b200.torch_ops as ops
    r = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    q, ld, s0 = r(1, 2, 100, 64).to(BF), torch.full((2,), -0.1, device="cuda"), r(1, 2, 64, 64)
    want, _ = sf.linear_attention(q, q, q, ld)
    leaf = q.clone().requires_grad_()
    y, _ = ops.linear_attention(leaf, q, q, ld)
    with withheld(SCALED):
        sf.linear_attention(q, q, q, ld)
    torch.cuda.synchronize()     # the kernel has reported; nothing has read it
    before = s0.clone()
    for call in (lambda: ops.linear_attention(q, q, q, ld), lambda: y.sum().backward(),
                 lambda: ops.linear_attention(q.float(), q.float(), q.float(), ld),
                 lambda: ops.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], ld, s0)):
        with pytest.raises(RuntimeError, match="timed out.*linear_attention_check"):
            call()
    for call in (lambda: sf.linear_attention(q, q, q, ld), lambda: sf.linear_attention_backward(q, q, q, ld, q),
                 lambda: sf.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], ld, s0)):
        with pytest.raises(sf.SffftError) as e:
            call()
        assert e.value.status == sf.ERR_TIMEOUT
    assert torch.equal(s0, before)
    with pytest.raises(sf.SffftError):
        sf.linear_attention_check()
    assert torch.equal(ops.linear_attention(q, q, q, ld)[0], want)
    sf.linear_attention_check()


def test_a_process_whose_first_call_is_captured():
    """The status word is allocated by the first call, which a graph may capture."""
    code = """if 1:
        import torch
        import sffft_b200 as sf
        q = torch.randn((1, 2, 300, 64), device="cuda").to(torch.bfloat16)
        ld = torch.full((2,), -0.1, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, s = sf.linear_attention(q, q, q, ld)
        g.replay()
        a, b = sf.linear_attention(q, q, q, ld)
        assert torch.equal(a, y) and torch.equal(b, s) and s.abs().max() > 0
        """
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
