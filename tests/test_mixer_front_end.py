"""Linear attention and block_norm on the CPU: what the PyTorch operators, the Python functions and the C ABI do with a call
before anything runs on a device."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import sffft_b200 as sf
import sffft_b200.torch_ops as ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def meta(*s, dtype=torch.float32):
    return torch.empty(s, device="meta", dtype=dtype)


def test_the_wait_limit_refuses_what_it_does_not_know():
    f = sf.lib().sffft_debug_linear_attention
    for bad in ((-1, 0), (1000001, 0), (2000, -1), (2000, 4), (0, 1)):
        assert f(*bad) == sf.ERR_INVALID_ARGUMENT
    assert f(2000, 3) == sf.OK and f(0, 0) == sf.OK


ATTENTION = dict(q=meta(2, 4, 10, 16), k=meta(2, 2, 10, 16), v=meta(2, 2, 10, 24), log_decay=meta(4), initial_state=meta(2, 4, 16, 24))
STEP = dict(q=meta(2, 4, 16), k=meta(2, 2, 16), v=meta(2, 2, 24), log_decay=meta(4), state=meta(5, 4, 16, 24))
NORM = dict(x=meta(3, 32), y=meta(3, 32), gate=meta(3, 32), post_weight=meta(32), weight=meta(32))


@pytest.mark.parametrize("op,args", [(ops.linear_attention, ATTENTION), (ops.linear_attention_step, STEP), (ops.block_norm, NORM)],
                         ids=["linear_attention", "linear_attention_step", "block_norm"])
def test_forward_mode_derivatives_are_refused(op, args):
    """They would come out as zero: a tensor with a tangent need not require a gradient."""
    for name, x in args.items():
        with forward_ad.dual_level():
            dual = dict(args, **{name: forward_ad.make_dual(x, torch.ones_like(x))})
            with pytest.raises(ValueError, match="forward-mode"):
                op(**dual)
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                op(**dual)
        with pytest.raises(ValueError, match="forward-mode"):
            torch.func.jvp(lambda t: op(**dict(args, **{name: t})), (x,), (x,))
        op(**args)


def strided(heads, d, L=10, B=2):
    """[B][heads][L][d] whose values are two apart and whose positions are outermost."""
    return torch.empty((B, L, heads, 2 * d), device="meta")[..., ::2].transpose(1, 2)


def test_traced_strides_where_the_last_axis_is_not_contiguous():
    """The operators copy such a tensor first, and order their outputs like the copy."""
    B, H, Hkv, L, D, Dv = 2, 4, 2, 10, 16, 24
    q, k, v, ld = strided(H, D), strided(Hkv, D), strided(Hkv, Dv), meta(H)
    y, s = ops.linear_attention(q, k, v, ld)
    assert y.stride() == (H * L * Dv, L * Dv, Dv, 1) and s.is_contiguous()
    grads = torch.ops.sffft.linear_attention_backward(q, k, v, ld, None, None, 1.0, meta(B, H, L, Dv), None)
    assert [g.stride() for g in grads] == [(H * L * D, L * D, D, 1), (Hkv * L * D, L * D, D, 1), (Hkv * L * Dv, L * Dv, Dv, 1)]
    # and where it is contiguous, like the tensor itself
    q = meta(B, L, H, D).transpose(1, 2)
    assert ops.linear_attention(q, k, v, ld)[0].stride() == (H * L * Dv, Dv, H * Dv, 1)
    grads = torch.ops.sffft.linear_attention_backward(q, k, v, ld, None, None, 1.0, meta(B, H, L, Dv), None)
    assert grads[0].stride() == (H * L * D, D, H * D, 1)


def test_a_decay_that_is_a_parameter_serves_without_gradients():
    """Where no gradient is asked for nothing is lost by it: prompts take it as single tokens do."""
    ld = meta(4).requires_grad_()
    with torch.no_grad():
        y, _ = ops.linear_attention(**dict(ATTENTION, log_decay=ld))
        assert y.shape == (2, 4, 10, 24)
        ops.linear_attention_step(**dict(STEP, log_decay=ld))
        sf.check_linear_attention(**dict(ATTENTION, log_decay=ld), scale=1.0, lengths=None)
    with torch.inference_mode():
        ops.linear_attention(**dict(ATTENTION, log_decay=ld))
    for op, args in ((ops.linear_attention, ATTENTION), (ops.linear_attention_step, STEP)):
        with pytest.raises(ValueError):
            op(**dict(args, log_decay=ld))
    with pytest.raises(ValueError):
        sf.check_linear_attention(**dict(ATTENTION, log_decay=ld), scale=1.0, lengths=None)


@pytest.mark.parametrize("what", ["missing", "not loadable"])
def test_the_convolution_does_not_need_the_mixers_library(what, tmp_path):
    """A build of lib/libsffft.so alone serves the convolution and the transforms; linear attention and block_norm say what is
    missing when they are called."""
    path = tmp_path / "libsffft_torch.so"
    if what == "not loadable":
        path.write_bytes(b"no library")
    code = f"""if 1:
        import torch, sffft_b200 as sf
        sf.TORCH_LIB_PATH = {str(path)!r}
        import sffft_b200.torch_ops as ops
        u, k = torch.empty((2, 3, 256), device="meta"), torch.empty((3, 256), device="meta")
        assert ops.causal_conv(u, k).shape == u.shape and ops.rfft(u).shape == (2, 3, 129)
        q = torch.empty((1, 2, 5, 16), device="meta")
        for call in (lambda: ops.linear_attention(q, q, q, torch.empty(2, device="meta")), lambda: ops.block_norm(q, weight=q[0, 0, 0]),
                     lambda: ops.linear_attention_step(q[:, :, 0], q[:, :, 0], q[:, :, 0], torch.empty(2, device="meta"), q)):
            try:
                call()
            except RuntimeError as e:
                assert "libsffft_torch.so" in str(e), e
            else:
                raise AssertionError("no error")
        """
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_the_build_does_without_pytorch(tmp_path):
    """A dry run with a Python that has none builds all but the PyTorch operators, and says so; with this one it builds them."""
    bare = tmp_path / "python"
    bare.write_text(f'#!/bin/sh\nexec {sys.executable} -I -S "$@"\n')
    bare.chmod(0o755)

    def dry(python):   # (whether the note was printed, what would be built)
        r = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "sffft_b200"), f"PYTHON={python}", "all"],
                           capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stderr
        return any(line.startswith("libsffft_torch.so") for line in r.stdout.splitlines()), r.stdout

    said, out = dry(bare)
    assert said and "torch_binding.cpp" not in out and "csrc/api.cu" in out and "csrc/cli.cpp" in out
    said, out = dry(sys.executable)
    assert not said and "torch_binding.cpp" in out


def test_c_abi_refuses_slots_that_overlap():
    """Rows of one call would update the same memory."""
    call = lambda d: sf.lib().sffft_linear_attention_step(ctypes.byref(d), 16, 16, 16, 16, 16, None, 16, None)  # noqa: E731
    for stride in (0, 2 * 8 * 8 - 1, -2 * 8 * 8):
        d = sf.LinearAttentionStepDesc(2, 2, 2, 8, 8, 2, 0, 0, 1.0)
        d.state_stride = stride
        assert call(d) == sf.ERR_INVALID_ARGUMENT, stride
    one = sf.LinearAttentionStepDesc(0, 2, 2, 8, 8, 1, 0, 0, 1.0)     # a pool of one slot has no stride
    assert call(one) == sf.OK
    apart = sf.LinearAttentionStepDesc(2, 2, 2, 8, 8, 2, 1, 0, 1.0)
    apart.state_stride = 2 * 8 * 8
    for i in range(7):     # and, with slots apart, an address between elements
        a = [16] * 5 + [None, 16]
        a[i] = 17
        assert sf.lib().sffft_linear_attention_step(ctypes.byref(apart), *a, None) == sf.ERR_INVALID_ARGUMENT, i
