"""Linear attention with keys and values of different sizes on rows that are cut into segments, forward and backward: the three
gradients' passes have different shapes there, and are planned and launched apart."""
import pytest
import torch

from tests.test_gpu_linear_attention import check, decays, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D,Dv", [(64, 128), (128, 64), (96, 72), (40, 200), (192, 64)])
def test_different_sizes_in_segments(D, Dv, dtype):
    n = torch.tensor([3000, 2111], dtype=torch.int32, device="cuda")
    check(make(2, 2, 2, 3000, D, Dv, dtype, D), decays(2, "cuda"), D ** -0.5)
    check(make(2, 2, 1, 3000, D, Dv, dtype, D + 1), decays(2, "cuda"), D ** -0.5, n)
