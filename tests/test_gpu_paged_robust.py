"""The paged cache's operators where they can go wrong: many requests to wide groups,
rows with nothing left, what autograd is told, memory that overlaps. The scenes and
bounds are those of test_gpu_paged.py."""
import random

import pytest
import torch

import fa_p100
import fa_p100_paged as paged
from test_gpu_paged import bits, check_attn, scene

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [1, 255, 257, 321, 1000])
@pytest.mark.parametrize("G", [65, 128, 150])
def test_attn_line_of_ten_warps(cuda, B, G):
    """Groups above 64 heads walk the line with ten warps a block, each with a sum of
    its own; more requests than threads, too. One step to several hundred a block."""
    rng = random.Random(B + G)
    lens = [rng.choice([0, 1, 128, 129, rng.randint(1, 400)]) for _ in range(B)] if B > 1 else [100003]
    s = scene(cuda, B, G, 1, 64, 16, lens, torch.bfloat16, seed=B)
    out = paged.paged_attn(*s)
    fa_p100.check_device_errors(cuda)
    check_attn(*s, *out)
    for _ in range(20):
        again = paged.paged_attn(*s)
        assert torch.equal(bits(out[0]), bits(again[0])) and torch.equal(out[1], again[1])
    fa_p100.check_device_errors(cuda)
