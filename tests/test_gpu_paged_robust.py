"""The paged cache's operators where they can go wrong: many requests to wide groups,
rows with nothing left, what autograd is told, memory that overlaps. The scenes and
bounds are those of test_gpu_paged.py."""
import os
import random
import subprocess
import sys

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


@pytest.mark.parametrize("D,units", [(64, 357913942), (128, 306783379)])
@pytest.mark.parametrize("heads", [(8, 2), (40, 2)], ids=["8", "40"])
def test_attn_token_strides_past_32_bits(cuda, D, units, heads):
    """Pages stored token by token over the whole pool, so that the tokens of a page lie
    4.9 GB apart (D = 128) or 5.7 GB: 14 (12) rows times the stride in units of 16 bytes
    is 2^32 and a little. Only the rows of this test's pages are ever touched."""
    Hkv, ps, P, n = 2, 16, 40, units * 8
    need = (ps - 1) * n + 2 * P * Hkv * D
    torch.cuda.empty_cache()
    assert torch.cuda.mem_get_info(cuda)[0] > 2 * need
    flat = torch.empty(need, dtype=torch.float16, device=cuda)
    kc, vc = (flat.as_strided((P, Hkv, ps, D), (2 * Hkv * D, D, n, 1), at * Hkv * D) for at in (0, 1))
    gen = torch.Generator(device=cuda).manual_seed(D)
    for t in range(ps):
        for c in (kc, vc):
            c[:, :, t] = torch.randn(P, Hkv, D, device=cuda, generator=gen).half()
    # clusters, and more units than they take
    for lens in ([500, 37], [1 + 7 * i % 300 for i in range(200)]):
        pages = torch.arange(len(lens) * 38, device=cuda).view(len(lens), 38) * 7 % P
        q = torch.randn(len(lens), heads[0], D, device=cuda, generator=gen).half()
        s = (q, kc, vc, pages.to(torch.int32), torch.tensor(lens, dtype=torch.int32, device=cuda))
        check_attn(*s, *paged.paged_attn(*s))
    rows = torch.randn(3, Hkv, D, device=cuda, generator=gen).half()
    paged.paged_append(rows, -rows, torch.tensor([15, 3 * 16 + 14, P * 16 - 1], dtype=torch.int32, device=cuda), kc, vc)
    for i, (page, t) in enumerate(((0, 15), (3, 14), (P - 1, 15))):
        assert torch.equal(kc[page, :, t], rows[i]) and torch.equal(vc[page, :, t], -rows[i])
    fa_p100.check_device_errors(cuda)
    del flat, kc, vc, s
    torch.cuda.empty_cache()


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def test_writes_are_seen_by_autograd(cuda):
    """What the operators write counts as changed in place: a backward that saved it
    raises, as after torch's own in-place operations."""
    c = paged.PagedKVCache(2, 2, 64, 9, 3, 48, 16, torch.float16, cuda)
    rows = torch.ones(3, 2, 64, device=cuda).half()
    tensors = dict(k=c.k, v=c.v, table=c.block_table, lens=c.lens, free=c.free_pages, count=c.free_count)

    def changed(call):
        before = {n: t._version for n, t in tensors.items()}
        call()
        return {n for n, t in tensors.items() if t._version != before[n]}

    w = torch.ones(64, device=cuda).half().requires_grad_(True)
    for saved in (c.k, c.k[1], c.v[1, 0]):
        c.extend(i32([1, 1, 1], cuda), 3)
        y = (saved * w).sum()      # saves the cache, or a view of it, for w's gradient
        with torch.no_grad():
            c.append(1, rows, rows)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    assert changed(lambda: c.extend(i32([1, 1, 1], cuda), 3)) == {"table", "lens", "count"}
    assert changed(lambda: c.append(0, rows, rows)) == {"k", "v"}
    assert changed(lambda: c.attn(0, rows)) == set()
    assert changed(lambda: c.release(torch.tensor([True, False, True], device=cuda))) == {"free", "lens", "count"}
    # outputs of the call's own leave the inputs as they were
    assert changed(lambda: paged.paged_extend(i32([1, 0, 0], cuda), c.lens, c.block_table, c.free_pages, c.free_count,
                                              16, 1)) == {"table"}
    # inference tensors have no version; outside inference mode they are written all the same
    with torch.inference_mode():
        c = paged.PagedKVCache(1, 2, 64, 9, 3, 48, 16, torch.float16, cuda)
        c.extend(i32([1, 1, 1], cuda), 3)
        c.append(0, rows, rows)
    c.extend(i32([1, 0, 0], cuda), 1)
    c.append(0, rows[:1], rows[:1])
    assert c.lens.tolist() == [2, 1, 1] and float(c.k.float().sum()) == 4 * 2 * 64


def test_transforms_and_fake_tensors_are_refused(cuda):
    """torch.func's wrappers, dual and fake tensors: refused, nothing written."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    import torch.autograd.forward_ad as fwAD
    half = lambda *s: torch.randn(*s, device=cuda).half()
    a = dict(k=half(5, 2, 64), v=half(5, 2, 64), slots=i32([0, 1, 2, 3, 20], cuda), k_cache=half(4, 2, 16, 64),
             v_cache=half(4, 2, 16, 64))
    b = dict(q=half(3, 4, 64), k_cache=a["k_cache"], v_cache=a["v_cache"], block_table=i32([[0, 1]] * 3, cuda),
             lens=i32([1, 20, 3], cuda))
    kept = a["k_cache"].clone(), a["v_cache"].clone()
    for op, args in ((paged.paged_append, a), (paged.paged_attn, b)):
        for name, x in args.items():
            def call(t):
                op(**{**args, name: t})
                return t
            with pytest.raises(RuntimeError):
                torch.func.vmap(call)(x[None])
            if x.is_floating_point():
                with pytest.raises(RuntimeError):
                    torch.func.jvp(call, (x,), (torch.ones_like(x),))
                with fwAD.dual_level(), pytest.raises(RuntimeError, match="carries a tangent"):
                    call(fwAD.make_dual(x, torch.ones_like(x)))
        with FakeTensorMode(allow_non_fake_inputs=True) as mode, pytest.raises(RuntimeError):
            op(**{n: mode.from_tensor(t) for n, t in args.items()})
    torch.cuda.synchronize()
    assert torch.equal(a["k_cache"], kept[0]) and torch.equal(a["v_cache"], kept[1])


def test_the_paged_kernels_are_loaded_by_their_own_first_call():
    """In a process of its own: flash_attn's first call does not wait for them."""
    code = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import fa_p100, fa_p100_paged as paged
dev = torch.device("cuda", 0)
q = torch.randn(1, 4, 256, 64, device=dev).half()
lens = torch.zeros(1, dtype=torch.int32, device=dev)
a = (lens, lens, torch.zeros(1, 2, dtype=torch.int32, device=dev), lens, lens, 16, 1)
torch.empty(1 << 20, device=dev), torch.empty(1 << 26, device=dev)     # torch's own pools
free = lambda: (torch.cuda.synchronize(), torch.cuda.mem_get_info(dev)[0])[1]
at = [free()]
fa_p100.flash_attn(q, q, q, True)
at.append(free())
paged.paged_extend(*a)
at.append(free())
paged.paged_extend(*a)
at.append(free())
print(at[0] - at[1], at[1] - at[2], at[2] - at[3])
"""
    seen = []
    for _ in range(3):      # free memory is the whole GPU's: another process may move it
        res = subprocess.run([sys.executable, "-c", code, os.path.dirname(paged.__file__)], capture_output=True,
                             text=True, timeout=300)
        assert res.returncode == 0, res.stderr[-2000:]
        first, own, again = map(int, res.stdout.split())
        if first > 0 and own > 0 and again == 0:
            return
        seen.append((first, own, again))
    assert False, f"bytes taken by the first flash_attn, the first paged call and the second: {seen}"
