"""Launches of block_norm whose shared memory is near a kernel's default limit."""

import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

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
