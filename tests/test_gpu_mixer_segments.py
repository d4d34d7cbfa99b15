"""Linear attention with keys and values of different sizes on rows that are cut into segments, forward and backward: the three
gradients' passes have different shapes there, and are planned and launched apart."""
import ctypes

import pytest
import torch

import sffft_b200 as sf
from tests.test_gpu_linear_attention import check, decays, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,Dv", [(64, 128), (128, 64), (96, 72), (40, 200), (192, 64)])
def test_different_sizes_in_segments(D, Dv, dtype):
    n = torch.tensor([3000, 2111], dtype=torch.int32, device="cuda")
    check(make(2, 2, 2, 3000, D, Dv, dtype, D), decays(2, "cuda"), D ** -0.5)
    check(make(2, 2, 1, 3000, D, Dv, dtype, D + 1), decays(2, "cuda"), D ** -0.5, n)


def is_cut(H, L, D, backward):
    """Whether a call in bf16 needs a workspace, which holds the segments' states where no heads are shared."""
    q = torch.zeros((1, H, L, D), dtype=torch.bfloat16, device="cuda")
    outs = [torch.empty_like(q) for _ in range(3)]
    st = (ctypes.c_longlong * 3)(*q.stride()[:3])
    desc = sf.LinearAttentionDesc(1, H, H, L, D, D, sf.IO["bf16"], q.device.index, 1.0, st, st, st, st)
    ld, s = torch.full((H,), -0.1, device="cuda"), torch.empty((1, H, D, D), device="cuda")
    p, stream = lambda t: t.data_ptr(), torch.cuda.current_stream().cuda_stream  # noqa: E731
    if backward:
        grads = sf.LinearAttentionGrads(st, st, st, st)
        rc = sf.lib().sffft_linear_attention_backward(ctypes.byref(desc), ctypes.byref(grads), p(q), p(q), p(q), p(ld), None, None, p(q),
                                                      None, *map(p, outs), None, None, 0, stream)
    else:
        rc = sf.lib().sffft_linear_attention(ctypes.byref(desc), p(q), p(q), p(q), p(ld), None, None, p(outs[0]), p(s), None, 0, stream)
    assert rc in (sf.OK, sf.ERR_WORKSPACE)
    return rc == sf.ERR_WORKSPACE


@pytest.mark.parametrize("D", [64, 128])
def test_rows_of_many_heads_stay_whole(D):
    """They were cut into up to 16 segments, which took up to three times as long (96 heads x 4096 x 128: 168 us whole, 526 as it
    was); rows of few heads are cut."""
    for H, L in ((96, 2048), (96, 4096), (128, 8192), (180, 4096)):
        assert not is_cut(H, L, D, False), (H, L)
    assert not is_cut(148, 4096, D, True)
    assert is_cut(8, 4096, D, False) and is_cut(16, 8192, D, False) and is_cut(4, 4096, D, True)
