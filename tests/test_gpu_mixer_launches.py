"""Launches of block_norm whose shared memory is near a kernel's default limit, and from several threads at once."""
import ctypes
import os
import subprocess
import sys
import threading

import pytest
import torch

import sffft_b200 as sf
from tests.test_gpu_block_norm import check, make

pytestmark = pytest.mark.gpu

F32 = torch.float32
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("C,groups", [(8192, 4096), (6144, 6144), (8184, 4092), (8148, 4074)])
def test_groups_whose_sums_take_just_48_kilobytes(C, groups):
    """In a process of its own: a kernel's limit, once raised by a larger call, stays raised."""
    code = f"""if 1:
        import torch
        from tests.test_gpu_block_norm import check, make
        t, dh, dn = make((3, {C}), -1, torch.float32, torch.float32, seed=1)
        check(t, dh, dn, {groups})
        """
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_threads_whose_calls_take_different_amounts():
    """Calls of one kernel at once, some with 53 KB of shared memory and some with 220: the limit is the kernel's, not a call's."""
    calls = []
    for C in (400, 1700):
        t, dh, dn = make((1, C, 64), 1, F32, F32, seed=C)
        want = check(t, dh, dn, dim=1)["n"]
        desc = sf.BlockNormDesc(64, C, 64, 1, 0, 0, 0, sf.GATE["full"], sf.ACT["silu"], 0.5, 1e-5, t["x"].device.index, 0, 0, 0)
        calls.append((t, desc, want))
    outs = [torch.empty_like(calls[i % 2][2]) for i in range(8)]
    hs = [torch.empty_like(o) for o in outs]
    streams = [torch.cuda.Stream() for _ in outs]
    torch.cuda.synchronize()
    status, gate = [None] * 8, threading.Barrier(8)

    def work(i):
        t, desc, _ = calls[i % 2]
        f, p = sf.lib().sffft_block_norm, ctypes.byref(desc)
        args = [t[n].data_ptr() for n in ("x", "y", "gate", "post_weight", "weight")]
        args += [hs[i].data_ptr(), outs[i].data_ptr(), None, None, streams[i].cuda_stream]
        gate.wait()
        status[i] = {f(p, *args) for _ in range(5000)}

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert status == [{sf.OK}] * 8
    assert all(torch.equal(o, calls[i % 2][2]) for i, o in enumerate(outs))
