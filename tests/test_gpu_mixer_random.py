"""Linear attention at random sizes, lengths, decays, orders of axes and shared heads, forward and backward, on the kernel that
bf16 takes where sizes are multiples of 8 and on the other."""
import random

import pytest
import torch

from tests.test_gpu_linear_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(60))
def test_random_calls(seed):
    r = random.Random(seed)
    step = 1 if seed % 4 == 3 else 8
    D, Dv = (r.randrange(1, 128 // step + 1) * step for _ in range(2))
    Hkv = r.randint(1, 4)
    H, B = Hkv * r.randint(1, 3), r.randint(1, 5)
    L = round(2 ** r.uniform(0, 10.5))
    t = make(B, H, Hkv, L, D, Dv, torch.bfloat16, seed, bool(seed & 1), r.random() < 0.6)
    ld = torch.tensor([-2.0 ** r.uniform(-12, 3) for _ in range(H)], device="cuda")
    n = torch.tensor([r.randint(0, L) for _ in range(B)], dtype=torch.int32, device="cuda") if r.random() < 0.5 else None
    check(t, ld, 2.0 ** r.uniform(-5, 2), n)
