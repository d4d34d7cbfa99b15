"""Linear attention under torch.compile where its tensors' last axis is not contiguous: traced strides are the real ones."""
import pytest
import torch

import sffft_b200.torch_ops as ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_values_under_compile(dtype):
    B, H, Hkv, L, D, Dv = 2, 4, 2, 50, 64, 64
    g = torch.Generator(device="cuda").manual_seed(0)

    def heads(n, d):
        return torch.randn((B, L, n, 2 * d), device="cuda", generator=g).to(dtype)[..., ::2].transpose(1, 2)

    q, k, v, ld = heads(H, D), heads(Hkv, D), heads(Hkv, Dv), torch.full((H,), -0.1, device="cuda")
    torch.library.opcheck(torch.ops.sffft.linear_attention.default, (q, k, v, ld, None, None, 0.125),
                          test_utils=("test_schema", "test_faketensor"))
    torch.library.opcheck(torch.ops.sffft.linear_attention_backward.default, (q, k, v, ld, None, None, 0.125, heads(H, Dv), None),
                          test_utils=("test_schema", "test_faketensor"))

    def loss(q, k, v):   # whose gradients are y and the state times powers of two: exact, in any order of its sums
        y, s = ops.linear_attention(q, k, v, ld, 0.125)
        return (2 * y.transpose(1, 2).float()).square().sum() + s.square().sum()

    outs, grads = [], []
    for f in (loss, torch.compile(loss, fullgraph=True)):
        leaves = [torch.empty_strided(t.shape, t.stride(), device="cuda", dtype=dtype).copy_(t).requires_grad_() for t in (q, k, v)]
        assert leaves[0].stride(-1) == 2
        outs.append(f(*leaves))
        outs[-1].backward()
        grads.append([x.grad for x in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    # sums of positive terms, each in an order of its own: half a step for each term and sum
    n = B * H * (L * Dv + D * Dv)
    assert abs(outs[0].item() - outs[1].item()) <= 2 * n * 2.0 ** -24 * outs[0].item()
