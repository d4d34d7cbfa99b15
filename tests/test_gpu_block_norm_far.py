"""block_norm on [B][C][L] tensors whose positions, or whose elements, are near or beyond 2^31."""
import pytest
import torch

import sffft_b200 as sf
from tests import mixer_ref as ref
from tests.test_gpu_block_norm import BF, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,C,L", [(1, 1, 2 ** 31 - 1), (2, 1024, 2 ** 20 + 4), (2, 512, 2 ** 21 + 33)])
def test_the_last_positions_of_large_tensors(B, C, L):
    """Zeros but for the last 45 positions, which have the values and the gradients that a call on them alone has; what comes
    before adds nothing to the weights' gradients."""
    n, groups = 45, 4 if C > 1 else 1
    small, dh, dn = make((1, C, n), 1, BF, BF, "none", C > 1, C > 1, True, seed=C, branch=C > 1)
    if C == 1:
        small["x"], dh = 2 * torch.randn((1, 1, n), device="cuda").to(BF), None

    def whole(t):
        if t is None or t.dim() == 1:
            return t
        big = torch.zeros((B, C, L), dtype=t.dtype, device="cuda")
        big[-1:, :, -n:] = t
        return big

    kw = dict(scale=0.5, eps=1e-5, groups=groups, act="none", dim=1)
    args = (small["x"], small["y"], None, small["post_weight"], small["weight"], 0.5, 1e-5, groups, "none", 1, dh, dn)
    want, mags = ref.norm(*args), ref.norm_magnitudes(*args)
    t = {name: whole(x) for name, x in small.items()}
    h, out, r1, r2 = sf.block_norm(**t, **kw, stats=True)
    got = {"n": out, "h": h if t["y"] is not None else None}
    got.update(zip(("dx", "dy", "dgate", "dpw", "dw"),
                   sf.block_norm_backward(whole(dh), whole(dn), **t, rstd_post=r1, rstd=r2, **kw)))
    for name, x in got.items():
        if x is None:
            continue
        if x.dim() == 3:
            assert x.shape == (B, C, L)
            assert not x[0, :, :64].any(), name
            x = x[-1:, :, -n:]
        off, tol = (x.double() - want[name]).abs(), ref.norm_bound(name, want[name], mags[name], x.dtype, C, n)
        assert (off <= tol).all(), (name, (off / tol).max().item())
