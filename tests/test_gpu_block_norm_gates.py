"""The activations of block_norm's gate on their own: h = act(gate), relative to the value and not only to the row."""
import pytest
import torch

import sffft_b200 as sf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [-1, 1])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
def test_gates_in_fp32_keep_their_bits(act, dim):
    """exp is off by at most 2 units in the last place, so is the approximate division; sum, product and scale add half of one
    each: 8 units hold them.  Below gate = -87 a sigmoid is smaller than the smallest normal number, which may be zero."""
    g = torch.linspace(-87, 100, 3 * 64 * 128, device="cuda").reshape(3, 64, 128)
    one = torch.ones_like(g)
    h, _ = sf.block_norm(y=one, gate=g, act=act, dim=dim)
    d = g.double()
    want = torch.sigmoid(d) * (d if act == "silu" else 1)
    assert ((h.double() - want).abs() <= 8 * 2.0 ** -23 * want.abs()).all(), ((h.double() - want).abs() / want.abs()).max().item() * 2 ** 23
    # its derivative s (1 + gate (1 - s)) or s (1 - s), where 1 - s cancels: 8 units of s, or of s (1 + |gate|)
    dg = sf.block_norm_backward(one, None, y=one, gate=g, act=act, dim=dim)[2]
    s = torch.sigmoid(d)
    want = s * (1 + d * (1 - s)) if act == "silu" else s * (1 - s)
    tol = s * (1 + d.abs()) if act == "silu" else s
    assert ((dg.double() - want).abs() <= 8 * 2.0 ** -23 * tol).all()
