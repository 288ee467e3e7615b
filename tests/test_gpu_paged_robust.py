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


# ways through the kernels: a cluster a unit, the line with whole units, one cut over
# many blocks, and both kernels of wide groups
NOTHING_LEFT = [(4, 8, 2, 300), (80, 8, 8, 70), (3, 8, 1, 40000), (300, 33, 1, 200), (300, 80, 1, 200),
                (2, 40, 1, 60000)]


@pytest.mark.parametrize("case", NOTHING_LEFT, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_attn_with_nothing_left(cuda, case, D, dtype):
    """A request whose every table entry is bad is one of length 0: its weights sum to 0.
    So are those of heads whose scores are all -inf. The other requests keep their bits."""
    B, Hq, Hkv, n = case
    q, kc, vc, table, lens = scene(cuda, B, Hq, Hkv, D, 16, [n - r % 7 for r in range(B)], dtype, seed=n)
    clean = paged.paged_attn(q, kc, vc, table, lens)
    bad = list(range(1, B, 3))
    t2 = table.clone()
    for i, r in enumerate(bad):
        t2[r] = [-1, kc.size(0), 2 ** 31 - 1, -2 ** 31][i % 4]
    fa_p100.check_device_errors(cuda)
    o, lse = paged.paged_attn(q, kc, vc, t2, lens)
    with pytest.raises(RuntimeError, match="page outside"):
        fa_p100.check_device_errors(cuda)
    assert (o[bad] == 0).all() and (lse[bad] == -float("inf")).all()
    rest = [r for r in range(B) if r not in bad]
    assert torch.equal(bits(o[rest]), bits(clean[0][rest])) and torch.equal(lse[rest], clean[1][rest])
    # request 0's last head: q is 1 in one place and every key -inf there
    q2, k2 = q.clone(), kc.clone()
    q2[0, -1] = 0
    q2[0, -1, 3] = 1
    j = torch.arange(int(lens[0]), device=cuda)
    seen = k2[table[0, j // 16].long(), -1, j % 16]
    seen[:, 3], seen[:, :3], seen[:, 4:] = -float("inf"), 0, 0
    k2[table[0, j // 16].long(), -1, j % 16] = seen
    o, lse = paged.paged_attn(q2, k2, vc, table, lens)
    assert (o[0, -1] == 0).all() and (lse[0, -1] == -float("inf")).all()
    assert torch.equal(bits(o[1:]), bits(clean[0][1:])) and torch.equal(lse[1:], clean[1][1:])
