"""The paged key-value cache against plain implementations: the page arithmetic
against a request-by-request allocator in Python, the copies bit for bit, the
attention against its formula in 64 bits."""
import math
import os
import random
import subprocess
import sys

import pytest
import torch

import _lib
import fa_p100
import fa_p100_paged as paged

pytestmark = pytest.mark.gpu
I32 = torch.int32


def pages_of(n, ps):
    return -(-n // ps)


def i32(values, dev):
    return torch.tensor(values, dtype=I32, device=dev)


# ---------------------------------------------------------------------------
# block tables
# ---------------------------------------------------------------------------
class Allocator:
    """Requests one after another, on Python lists."""

    def __init__(self, lens, table, stack, count, ps):
        self.lens, self.table = list(lens), [list(r) for r in table]
        self.stack, self.count, self.ps = list(stack), count, ps

    def extend(self, new, total):
        P, W, ps = len(self.stack), len(self.table[0]), self.ps
        count = min(max(self.count, 0), P)
        slots, granted, end, need, taken = [-1] * total, [], 0, 0, 0
        for r, n in enumerate(new):
            n, len0 = max(n, 0), self.lens[r]
            start, end = end, end + n
            fits = n > 0 and len0 >= 0 and len0 + n <= W * ps and end <= total
            want = pages_of(len0 + n, ps) - pages_of(len0, ps) if fits else 0
            need += want
            if not fits or (want and need > count):
                granted.append(0)
                continue
            granted.append(n)
            for j in range(want):
                self.table[r][pages_of(len0, ps) + j] = self.stack[count - 1 - taken]
                taken += 1
            for t in range(n):
                page = self.table[r][(len0 + t) // ps]
                if 0 <= page < P:
                    slots[start + t] = page * ps + (len0 + t) % ps
            self.lens[r] = len0 + n
        self.count = count - taken
        return slots, granted

    def release(self, finished):
        P, W, ps = len(self.stack), len(self.table[0]), self.ps
        at = min(max(self.count, 0), P)
        for r, done in enumerate(finished):
            if done:
                for j in range(pages_of(min(max(self.lens[r], 0), W * ps), ps)):
                    if at < P:
                        self.stack[at] = self.table[r][j]
                        at += 1
                self.lens[r] = 0
        self.count = at


def pool(B, W, ps, lens, extra, seed):
    """(table, stack, count): the requests' pages scattered over a pool."""
    used = [pages_of(min(max(n, 0), W * ps), ps) for n in lens]
    P = sum(used) + extra
    ids = list(range(max(P, 1)))
    random.Random(seed).shuffle(ids)
    table = [[-1] * W for _ in range(B)]
    for r, n in enumerate(used):
        for j in range(n):
            table[r][j] = ids.pop()
    count = len(ids)
    return table, ids + [-7] * (max(P, 1) - count), count


def run_extend(dev, lens, new, table, stack, count, ps, total, pad=0, in_place=False):
    """One call against the allocator; returns the allocator after it."""
    al = Allocator(lens, table, stack, count, ps)
    want_slots, want_granted = al.extend(new, total)
    d_lens, d_stack, d_count = i32(lens, dev), i32(stack, dev), i32([count], dev)
    wide = torch.full((len(lens), len(table[0]) + pad), -9, dtype=I32, device=dev)
    d_table = wide[:, :len(table[0])]
    d_table.copy_(i32(table, dev))
    kw = dict(lens_out=d_lens, free_count_out=d_count) if in_place else {}
    slots, granted, lens_out, count_out = paged.paged_extend(
        i32(new, dev), d_lens, d_table, d_stack, d_count, ps, total, **kw)
    assert slots.tolist() == want_slots
    assert granted.tolist() == want_granted
    assert lens_out.tolist() == al.lens and count_out.tolist() == [al.count]
    assert d_table.tolist() == al.table and (wide[:, len(table[0]):] == -9).all()
    assert d_stack.tolist() == al.stack
    if in_place:
        assert lens_out is d_lens and count_out is d_count
    else:
        assert d_lens.tolist() == list(lens) and d_count.tolist() == [count]
    return al


EXTEND = [  # B, W, ps, longest so far, most new, spare pages, total off by, seed
    (1, 1, 16, 0, 1, 1, 0, 0),
    (1, 4, 16, 0, 64, 4, 0, 1),
    (5, 8, 16, 60, 1, 3, 0, 2),
    (64, 32, 16, 500, 1, 8, 0, 3),          # the pool runs out on the way
    (64, 32, 48, 500, 700, 200, 0, 4),
    (64, 32, 16, 500, 40, 1000, -300, 5),   # the last requests have no room in the call
    (64, 32, 16, 500, 40, 1000, 77, 6),     # more room than tokens
    (1023, 12, 32, 200, 130, 2500, 0, 7),
    (1025, 12, 32, 200, 130, 6000, 0, 8),
    (2500, 9, 16, 100, 60, 9000, 5, 9),
    (3, 700, 16, 5000, 6000, 900, 0, 10),
    (2, 1, 4096, 4000, 200, 2, 0, 11),
]


@pytest.mark.parametrize("case", EXTEND, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("in_place", [False, True], ids=["new", "inplace"])
def test_extend(cuda, case, in_place):
    B, W, ps, ctx, most, extra, off, seed = case
    rng = random.Random(seed)
    lens = [rng.randint(0, min(ctx, W * ps)) for _ in range(B)]
    new = [rng.choice([most, rng.randint(0, most), 0, 1]) for _ in range(B)]
    table, stack, count = pool(B, W, ps, lens, extra, seed)
    run_extend(cuda, lens, new, table, stack, count, ps, max(0, sum(new) + off), pad=seed % 3,
               in_place=in_place)


def test_extend_many_tokens(cuda):
    """Prompts whose tokens are far more than one block of threads."""
    rng = random.Random(3)
    B, W, ps = 300, 256, 16
    lens = [rng.randint(0, 1000) for _ in range(B)]
    new = [rng.randint(0, 3000) for _ in range(B)]
    table, stack, count = pool(B, W, ps, lens, 40000, 3)
    run_extend(cuda, lens, new, table, stack, count, ps, sum(new))


def test_extend_odd_values(cuda):
    """Lengths and counts no user means: refused, never followed."""
    big = 2 ** 31 - 1
    ps, W = 16, 4
    for lens, new, count in [
            ([-1, 5, -big, 70, 64, 63], [3, 2, 1, 1, 1, 1], 9),      # negative, past the row, full
            ([0, 0, 0], [big, big, 2], 9),                          # sums past 32 bits
            ([0, 3], [-4, 5], 9),                                    # negative new tokens
            ([0, 0], [20, 20], -3), ([0, 0], [20, 20], 500),         # counts outside the stack
            ([0, 0], [0, 0], 0)]:
        table, stack, _ = pool(len(lens), W, ps, lens, 9, 1)
        run_extend(cuda, lens, new, table, stack, count, ps, 12)
        run_extend(cuda, lens, new, table, stack, count, ps, 0)
    # a page so far that does not exist: its tokens get no slot
    run_extend(cuda, [5, 5, 5], [20, 20, 1], [[99, -1, -1, -1], [-1] * 4, [2, -1, -1, -1]],
               [0, 1, 3, 4, 5, 6, 7, 8], 8, ps, 41)


def test_extend_most_tokens(cuda):
    """A call of 2^31 - 1 tokens: a request too long for its row, and one that fits
    behind which the slots end."""
    table = i32([[-1] * 4, [-1] * 4], cuda)
    stack, count, total = i32([5, 4, 3, 2, 1, 0], cuda), i32([6], cuda), 2 ** 31 - 1
    slots, granted, lens, left = paged.paged_extend(i32([2 ** 31 - 41, 40], cuda), i32([0, 0], cuda), table, stack,
                                                    count, 16, total)
    assert granted.tolist() == [0, 40] and lens.tolist() == [0, 40] and left.tolist() == [3]
    assert slots[-40:].tolist() == list(range(40)) and int(slots[:-40].max()) == -1
    slots, granted, _, left = paged.paged_extend(i32([total, 0], cuda), i32([0, 40], cuda), table, stack, left, 16, total)
    assert granted.tolist() == [0, 0] and left.tolist() == [3] and int(slots.max()) == -1


RELEASE = [(1, 1, 16, 16, 1, 0), (7, 9, 16, 140, 2, 1), (64, 40, 48, 1500, 3, 2),
           (1024, 10, 32, 300, 1, 3), (2100, 7, 16, 100, 2, 4), (4, 3000, 16, 48000, 1, 5),
           (128, 255, 16, 4080, 1, 6), (129, 256, 16, 4096, 1, 7), (100, 20, 16, 320, 5, 8)]


@pytest.mark.parametrize("case", RELEASE, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("in_place", [False, True], ids=["new", "inplace"])
def test_release(cuda, case, in_place):
    B, W, ps, ctx, every, seed = case
    rng = random.Random(seed)
    lens = [rng.randint(0, ctx) for _ in range(B)]
    fin = [rng.randrange(every) == 0 for _ in range(B)]
    table, stack, count = pool(B, W, ps, lens, 3, seed)
    check_release(cuda, lens, fin, table, stack, count, ps, in_place)


def check_release(dev, lens, fin, table, stack, count, ps, in_place=False):
    al = Allocator(lens, table, stack, count, ps)
    al.release(fin)
    d_lens, d_table, d_stack, d_count = i32(lens, dev), i32(table, dev), i32(stack, dev), i32([count], dev)
    kw = dict(lens_out=d_lens, free_count_out=d_count) if in_place else {}
    lens_out, count_out = paged.paged_release(torch.tensor(fin, device=dev), d_lens, d_table, d_stack,
                                              d_count, ps, **kw)
    assert lens_out.tolist() == al.lens and count_out.tolist() == [al.count]
    assert d_stack.tolist() == al.stack and d_table.tolist() == table


def test_release_odd_values(cuda):
    table, stack, count = pool(3, 4, 16, [64, 64, 20], 2, 0)
    check_release(cuda, [-5, 1000, 20], [True, True, True], table, stack, count, 16)
    check_release(cuda, [64, 64, 20], [True, True, True], table, stack, 8, 16)     # more than fit
    check_release(cuda, [64, 64, 20], [False] * 3, table, stack, -1, 16)
    check_release(cuda, [64, 64, 20], [True] * 3, table, stack, 99, 16)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------
def bits(t):
    return t.contiguous().view(torch.int16)


def make_cache(dev, P, Hkv, ps, D, dtype, layout, gen):
    """Two caches in one of three layouts; "pair" interleaves k and v page by page."""
    mk = lambda *s: torch.randn(*s, device=dev, generator=gen).to(dtype)
    if layout == "head":
        return mk(P, Hkv, ps, D), mk(P, Hkv, ps, D)
    if layout == "row":
        return mk(P, ps, Hkv, D).transpose(1, 2), mk(P, ps, Hkv, D).transpose(1, 2)
    kv = mk(P, 2, Hkv, ps, D + 8)[..., :D]
    return kv[:, 0], kv[:, 1]


@pytest.mark.parametrize("layout", ["head", "row", "pair"])
@pytest.mark.parametrize("case", [(0, 2, 64, 16), (1, 1, 64, 16), (1, 8, 128, 48), (37, 5, 128, 32),
                                  (300, 3, 64, 64), (2049, 8, 128, 16)],
                         ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_append(cuda, case, layout, dtype):
    T, Hkv, D, ps = case
    gen = torch.Generator(device=cuda).manual_seed(T)
    host = torch.Generator().manual_seed(T)
    P = pages_of(T, ps) + 3
    kc, vc = make_cache(cuda, P, Hkv, ps, D, dtype, layout, gen)
    rows = torch.randn(T, 4 + 2 * Hkv, D, device=cuda, generator=gen).to(dtype)
    if T:
        rows[0, :, 0], rows[0, :, 1], rows[0, :, 2] = math.nan, math.inf, -0.0
    slots = torch.randperm(P * ps, generator=host)[:T].to(I32)
    slots[::7] = torch.tensor([-1, P * ps, 2 ** 31 - 1, -2 ** 31], dtype=torch.int64).to(I32).repeat(
        T)[:slots[::7].numel()]
    for k, v in ((rows[:, 4:4 + Hkv], rows[:, 4 + Hkv:]),
                 (rows[:, 4:4 + Hkv].clone(), rows[:, :Hkv].clone())):
        want_k, want_v = kc.clone(), vc.clone()
        for t, s in enumerate(slots.tolist()):
            if 0 <= s < P * ps:
                want_k[s // ps, :, s % ps] = k[t]
                want_v[s // ps, :, s % ps] = v[t]
        paged.paged_append(k, v, slots.to(cuda), kc, vc)
        assert torch.equal(bits(kc), bits(want_k)) and torch.equal(bits(vc), bits(want_v))


def test_append_unaligned_input_is_copied(cuda):
    kc = torch.zeros(3, 2, 16, 64, device=cuda, dtype=torch.float16)
    vc = torch.zeros_like(kc)
    flat = torch.randn(5 * 2 * 65 + 1, device=cuda).half()
    k = flat[1:].view(5, 2, 65)[..., :64]
    paged.paged_append(k, k, i32([0, 17, 47, 5, 30], cuda), kc, vc)
    for t, s in enumerate([0, 17, 47, 5, 30]):
        assert torch.equal(kc[s // 16, :, s % 16], k[t]) and torch.equal(vc[s // 16, :, s % 16], k[t])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def scene(dev, B, Hq, Hkv, D, ps, lens, dtype, layout="head", seed=0, width=None, q_scale=1.0):
    """q, caches, table and lengths; everything a request must not read is NaN."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    n = [pages_of(x, ps) for x in lens]
    P = sum(n) + 2
    kc, vc = make_cache(dev, P, Hkv, ps, D, dtype, layout, gen)
    ids = torch.randperm(P, generator=host).tolist()
    W = width or max(1, max(n))
    table = [[-1] * W for _ in range(B)]
    owned = torch.zeros(P, ps, dtype=torch.bool)
    for r in range(B):
        for j in range(n[r]):
            p = table[r][j] = ids.pop()
            owned[p, :min(ps, lens[r] - j * ps)] = True
    hole = (~owned).to(dev)[:, None, :, None]
    kc.masked_fill_(hole, math.nan)
    vc.masked_fill_(hole, math.nan)
    q = (torch.randn(B, Hq, D, device=dev, generator=gen) * q_scale).to(dtype)
    return q, kc, vc, i32(table, dev), i32(lens, dev)


def check_attn(q, kc, vc, table, lens, o, lse, skip=()):
    """Against the formula in 64 bits. What may differ, with eps the spacing of the
    output's type, u = 2^-24 and A = sum_j p_j |v_j| (p normalised):
      * the output's rounding: eps/2 |o|
      * the weights as two 16-bit terms in their product with v: eps^2/4 A
      * scores in fp32: D + 4 roundings of at most u sum_d |q_d k_d| / sqrt(D) each, and
        3 of the exponent's argument, u |s|; with the exponential's own 4 u they are a
        relative error of every weight, and act on numerator and sum: 2 (..) A
      * fp32 sums over n keys: n u A twice."""
    B, Hq, D = q.shape
    Hkv, ps = kc.shape[1], kc.shape[2]
    G, eps, u = Hq // Hkv, torch.finfo(q.dtype).eps, 2.0 ** -24
    for r in range(B):
        n = int(lens[r])
        if n == 0:
            assert (o[r] == 0).all() and (lse[r] == -math.inf).all()
            continue
        j = torch.tensor([x for x in range(n) if (r, x // ps) not in skip], device=q.device)
        if j.numel() == 0:
            continue
        page = table[r, j // ps].long()
        k = kc[page, :, j % ps].double().repeat_interleave(G, 1)      # (n, Hq, D)
        v = vc[page, :, j % ps].double().repeat_interleave(G, 1)
        x = q[r].double()
        s = torch.einsum("hd,nhd->hn", x, k) / math.sqrt(D)
        mag = torch.einsum("hd,nhd->hn", x.abs(), k.abs()).amax(1) / math.sqrt(D)
        want_lse = torch.logsumexp(s, 1)
        p = torch.exp(s - want_lse[:, None])
        want = torch.einsum("hn,nhd->hd", p, v)
        A = torch.einsum("hn,nhd->hd", p, v.abs())
        score = u * ((D + 4) * mag + 3 * s.abs().amax(1) + 4)
        rel = 2 * score + 2 * n * u
        tol = eps / 2 * want.abs() + (rel[:, None] + eps * eps / 4) * A
        tol = tol * (1 + eps) + torch.finfo(q.dtype).smallest_normal * eps
        err = (o[r].double() - want).abs()
        assert (err <= tol).all(), f"row {r}: o off by {(err / tol).max().item():.3f} of its bound"
        tol = score + n * u + 4 * u * want_lse.abs()
        err = (lse[r].double() - want_lse).abs()
        assert (err <= tol).all(), f"row {r}: lse off by {(err / tol).max().item():.3f} of its bound"


HEADS = [(1, 1), (4, 4), (16, 8), (32, 8), (10, 2), (16, 2), (9, 1), (16, 1), (17, 1), (32, 1),
         (33, 1), (71, 1), (48, 2)]
LENS = [0, 1, 2, 15, 16, 17, 31, 33, 47, 48, 49, 63, 64, 65, 127, 128, 129, 255, 257, 500]


@pytest.mark.parametrize("heads", HEADS, ids=lambda h: f"{h[0]}-{h[1]}")
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_attn_heads(cuda, heads, D, dtype):
    lens = LENS[::-1]
    s = scene(cuda, len(lens), *heads, D, 16, lens, dtype, seed=sum(heads) + D)
    check_attn(*s, *paged.paged_attn(*s))


@pytest.mark.parametrize("ps", [16, 32, 48, 64, 112, 128, 4096])
@pytest.mark.parametrize("layout", ["head", "row", "pair"])
@pytest.mark.parametrize("D", [64, 128])
def test_attn_pages(cuda, ps, layout, D):
    s = scene(cuda, len(LENS), 8, 2, D, ps, LENS, torch.float16, layout, seed=ps)
    check_attn(*s, *paged.paged_attn(*s))


@pytest.mark.parametrize("G", [17, 32, 33, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_attn_wide_groups(cuda, G, D, dtype):
    """More units than clusters can take, groups above 16 heads: the kernel on
    tensor memory, with lengths around its steps of 128 keys."""
    rng = random.Random(G)
    lens = [rng.choice([0, 1, 15, 16, 17, 127, 128, 129, 255, 256, 257, rng.randint(1, 700)]) for _ in range(300)]
    s = scene(cuda, 300, G, 1, D, 16, lens, dtype, seed=G + D)
    out = paged.paged_attn(*s)
    fa_p100.check_device_errors(cuda)
    check_attn(*s, *out)
    again = paged.paged_attn(*s)
    assert torch.equal(bits(out[0]), bits(again[0])) and torch.equal(out[1], again[1])
    fa_p100.check_device_errors(cuda)


@pytest.mark.parametrize("ps", [16, 48, 64, 80, 128, 4096])
@pytest.mark.parametrize("layout", ["head", "row", "pair"])
def test_attn_wide_pages(cuda, ps, layout):
    """Page sizes and layouts in the same kernel, and table entries without a page."""
    rng = random.Random(ps)
    lens = [rng.randint(0, 600) for _ in range(160)]
    s = scene(cuda, 160, 80, 2, 128, ps, lens, torch.bfloat16, layout, seed=ps)
    check_attn(*s, *paged.paged_attn(*s))
    fa_p100.check_device_errors(cuda)
    table, skip = s[3], set()
    for r in range(0, 160, 7):
        j = rng.randrange(table.size(1))
        table[r, j] = rng.choice([-1, s[1].size(0), 2 ** 31 - 1, -2 ** 31])
        skip.add((r, j))
    check_attn(*s, *paged.paged_attn(*s), skip=skip)
    _lib.device_error(0)


def test_attn_wide_checked_build(cuda):
    """The wide groups' kernel in the checked library, whose TMA copies test their
    coordinates and alignment first."""
    import _build
    _build.build(checked=True)
    paths = [os.path.dirname(os.path.abspath(x)) for x in (__file__, paged.__file__)]
    code = f"""
import sys
sys.path[:0] = {paths!r}
import test_gpu_paged as t
dev = t.torch.device("cuda", 0)
t._lib.tma_check_word(0, reset=True)
for D, heads in ((64, 40), (128, 40), (64, 100), (128, 100)):
    s = t.scene(dev, 160, heads, 1, D, 48, [(7 * i) % 500 for i in range(160)], t.torch.bfloat16)
    t.check_attn(*s, *t.paged.paged_attn(*s))
print(t.os.path.basename(t._lib.loaded_path()), t._lib.tma_check_word(0), t._lib.device_error(0))
"""
    res = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, FA_B200_DEBUG="1"),
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout[-2000:] + res.stderr[-4000:]
    assert res.stdout.split()[-3:] == ["libfa_b200_debug.so", "0", "0"]


def test_attn_outputs(cuda):
    """o and lse share an allocation, but neither's values nor its graph the other's;
    the table calls' outputs likewise."""
    s = scene(cuda, 3, 8, 2, 64, 16, [5, 0, 40], torch.float16)
    o, lse = paged.paged_attn(*s)
    o0, lse0 = o.clone(), lse.clone()
    assert o.is_contiguous() and lse.is_contiguous() and not o.requires_grad and not lse.requires_grad
    w = torch.ones(64, device=cuda, requires_grad=True)
    (o.float() * w).sum().backward()
    torch.testing.assert_close(w.grad, o0.float().sum((0, 1)))
    lse.fill_(7.0)
    assert torch.equal(o, o0)
    o.zero_()
    assert (lse == 7.0).all()
    with torch.inference_mode():
        o, lse = paged.paged_attn(*s)
        assert o.is_inference() and torch.equal(o, o0) and torch.equal(lse, lse0)
    lens, free = i32([5, 0, 40], cuda), i32(list(range(9)), cuda)
    out = paged.paged_extend(i32([1, 2, 0], cuda), lens, s[3].clone(), free, i32([9], cuda), 16, 3)
    kept = [x.clone() for x in out]
    for i, x in enumerate(out):
        x.fill_(99)
        for y, k in zip(out[i + 1:], kept[i + 1:]):
            assert torch.equal(y, k)


@pytest.mark.parametrize("G", [4, 16, 32, 40])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dim", [0, 1])
def test_attn_expanded(cuda, G, D, dim):
    """Caches that repeat one head, or one page, by a stride of 0 are only read."""
    q, kc, vc, table, lens = scene(cuda, 160, 2 * G, 1, D, 32, [1 + 3 * i for i in range(160)],
                                   torch.bfloat16, seed=G + D)
    if dim == 0:   # page 0 for every page, all of it tokens
        kc, vc = (torch.randn(1, 2, 32, D, device=cuda).to(x).expand(x.size(0), -1, -1, -1) for x in (kc, vc))
    else:
        kc, vc = kc.expand(-1, 2, -1, -1), vc.expand(-1, 2, -1, -1)
    check_attn(q, kc, vc, table, lens, *paged.paged_attn(q, kc, vc, table, lens))
    fa_p100.check_device_errors(cuda)


@pytest.mark.parametrize("lens", [[1], [0], [16], [300], [1537], [5000], [40000], [1, 30000], [0, 0, 9000],
                                  [30000, 0, 1, 7], [2048] * 16, [777] * 100, [1] * 300,
                                  list(range(0, 2000, 13))], ids=lambda l: f"{len(l)}x{max(l)}")
@pytest.mark.parametrize("heads", [(8, 8), (16, 2), (32, 1)], ids=lambda h: f"{h[0]}-{h[1]}")
def test_attn_lengths(cuda, lens, heads):
    """One key to tens of thousands, few rows and many, ragged: the split and its join."""
    s = scene(cuda, len(lens), *heads, 128, 16, lens, torch.bfloat16, seed=len(lens),
              width=pages_of(max(max(lens), 1), 16) + 3)
    out = paged.paged_attn(*s)
    check_attn(*s, *out)
    again = paged.paged_attn(*s)
    assert torch.equal(bits(out[0]), bits(again[0])) and torch.equal(out[1], again[1])


def test_attn_sharp_and_flat(cuda):
    """Scores far apart (one key takes all), equal ones, and a running maximum
    that grows to the last key."""
    q, kc, vc, table, lens = scene(cuda, 3, 8, 2, 64, 16, [700, 1000, 333], torch.float16, q_scale=30.0)
    check_attn(q, kc, vc, table, lens, *paged.paged_attn(q, kc, vc, table, lens))
    zero = torch.zeros_like(q)
    check_attn(zero, kc, vc, table, lens, *paged.paged_attn(zero, kc, vc, table, lens))
    for r, n in enumerate([700, 1000, 333]):
        j = torch.arange(n, device=cuda)
        kc[table[r, j // 16].long(), :, j % 16] = (j.float() / 64).half()[:, None, None].expand(n, 2, 64)
    one = torch.ones_like(q)
    check_attn(one, kc, vc, table, lens, *paged.paged_attn(one, kc, vc, table, lens))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("heads", [(8, 2), (20, 2), (50, 2), (100, 2)], ids=lambda h: f"{h[0]}-{h[1]}")
@pytest.mark.parametrize("B", [4, 40, 400])
def test_attn_non_finite_values(cuda, heads, dtype, B):
    """Infinities and NaN in keys and values that are seen act as in the formula;
    in another request's pages they do not act at all."""
    Hq, G = heads[0], heads[0] // 2
    s = scene(cuda, B, Hq, 2, 128, 16, [200] * B, dtype, seed=4)
    q, kc, vc, table, lens = s
    clean = paged.paged_attn(*s)
    place = lambda r, j: (int(table[r, j // 16]), j % 16)
    p, off = place(1, 77)
    vc[p, 0, off, 5], vc[p, 0, off, 6] = math.inf, -math.inf
    p, off = place(2, 199)
    kc[p, 1, off, 0] = math.nan
    p, off = place(3, 0)
    kc[p, :, off, :] = torch.where(q[3, 0] >= 0, math.inf, -math.inf).to(dtype)   # head 0: score +inf
    o, lse = paged.paged_attn(*s)
    assert torch.equal(o[0], clean[0][0]) and torch.equal(lse[0], clean[1][0])
    assert (o[1, :G, 5] == math.inf).all() and (o[1, :G, 6] == -math.inf).all()
    keep = torch.ones(Hq, 128, dtype=torch.bool, device=cuda)
    keep[:G, 5:7] = False
    assert torch.equal(o[1][keep], clean[0][1][keep])
    assert torch.isnan(o[2, G:]).all() and torch.isnan(lse[2, G:]).all()
    assert torch.equal(o[2, :G], clean[0][2, :G])
    assert torch.isnan(o[3, 0]).all()


def test_attn_strided_query_and_views(cuda):
    """q as a slice of a fused projection, a wider table, and an unaligned q."""
    q, kc, vc, table, lens = scene(cuda, 6, 8, 4, 64, 32, [5, 900, 0, 64, 100, 33], torch.bfloat16)
    o, lse = paged.paged_attn(q, kc, vc, table, lens)
    fused = torch.randn(6, 16, 64, device=cuda).bfloat16()
    fused[:, :8] = q
    wide = torch.full((6, table.size(1) + 5), 10 ** 9, dtype=I32, device=cuda)
    wide[:, :table.size(1)] = table
    flat = torch.empty(6 * 8 * 64 + 1, device=cuda, dtype=torch.bfloat16)
    flat[1:] = q.reshape(-1)
    for q2, t2 in ((fused[:, :8], wide[:, :table.size(1)]), (flat[1:].view(6, 8, 64), wide)):
        o2, lse2 = paged.paged_attn(q2, kc, vc, t2, lens)
        check_attn(q, kc, vc, table, lens, o2, lse2)


def test_attn_lengths_out_of_range(cuda):
    """A negative length is an empty row, one past the table is the whole table."""
    q, kc, vc, table, lens = scene(cuda, 3, 4, 4, 64, 16, [64, 64, 64], torch.float16)
    want = paged.paged_attn(q, kc, vc, table, lens)
    o, lse = paged.paged_attn(q, kc, vc, table, i32([-2 ** 31, 2 ** 31 - 1, 65], cuda))
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all()
    assert torch.equal(o[1:], want[0][1:]) and torch.equal(lse[1:], want[1][1:])


def test_attn_offsets_past_32_bits(cuda):
    """Pages whose elements lie behind 2^31 elements (and 2^33 bytes) of the pool."""
    P, ps, D = (1 << 31) // (2 * 16 * 128) + 600, 16, 128
    kv = torch.empty(P, 2, 1, ps, D, dtype=torch.float16, device=cuda)
    kc, vc = kv[:, 0], kv[:, 1]
    gen = torch.Generator(device=cuda).manual_seed(1)
    kv[-600:] = torch.randn(600, 2, 1, ps, D, device=cuda, generator=gen).half()
    kv[:600] = math.nan
    lens = [3000, 17, 5000]
    ids = iter(torch.randperm(600, generator=torch.Generator().manual_seed(2)).tolist())
    table = [[P - 600 + next(ids) if j < pages_of(n, ps) else -1 for j in range(320)] for n in lens]
    q = torch.randn(3, 4, D, device=cuda, generator=gen).half()
    s = (q, kc, vc, i32(table, cuda), i32(lens, cuda))
    check_attn(*s, *paged.paged_attn(*s))
    rows = torch.randn(2, 1, D, device=cuda, generator=gen).half()
    paged.paged_append(rows, rows, i32([(P - 1) * ps + 3, 5], cuda), kc, vc)
    assert torch.equal(kc[P - 1, 0, 3], rows[0, 0]) and torch.equal(vc[0, 0, 5], rows[1, 0])


def test_attn_bad_pages(cuda):
    """Table entries that name no page: reported, and their tokens left out."""
    fa_p100.check_device_errors(cuda)
    q, kc, vc, table, lens = scene(cuda, 3, 8, 2, 64, 16, [100, 500, 40], torch.float16)
    P = kc.size(0)
    table[0, 2], table[1, 0], table[1, 31] = -1, P, 2 ** 31 - 1
    table[2, :3] = -2 ** 31
    o, lse = paged.paged_attn(q, kc, vc, table, lens)
    with pytest.raises(RuntimeError, match="page outside"):
        fa_p100.check_device_errors(cuda)
    check_attn(q, kc, vc, table, lens, o, lse, skip={(0, 2), (1, 0), (1, 31), (2, 0), (2, 1), (2, 2)})
    assert _lib.device_error(0) == 0


# ---------------------------------------------------------------------------
# streams, graphs, and the operators together
# ---------------------------------------------------------------------------
def test_attn_two_streams(cuda):
    """Calls of different inputs at once on two streams keep apart."""
    scenes = [scene(cuda, 24, 16, 2, 128, 16, [1500 + 31 * i for i in range(24)], torch.float16, seed=i)
              for i in range(2)]
    want = [paged.paged_attn(*s) for s in scenes]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(paged.paged_attn(*scenes[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for o, lse in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])


def decode_setup(dev, seed, batch=5, layers=2, Hkv=2, D=64, dtype=torch.float16, page_size=16, pages=60):
    c = paged.PagedKVCache(layers, Hkv, D, pages, batch, 160, page_size, dtype, dev)
    gen = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s: torch.randn(*s, device=dev, generator=gen).to(dtype)
    return c, mk


def test_decode_steps_match_full_attention(cuda):
    """Prompts, then tokens one by one, requests that end and others that take their
    pages: every step's attention is the last row of causal flash_attn over the
    request's whole history."""
    B, layers, Hq, Hkv, D = 5, 2, 4, 2, 64
    c, mk = decode_setup(cuda, 0)
    history = [[[] for _ in range(B)] for _ in range(layers)]   # [layer][request]: (k, v) rows
    rng = random.Random(5)
    lens = [0] * B
    for step in range(30):
        if step % 10 == 0:      # new prompts where there is no request
            new = [rng.randint(1, 50) if lens[r] == 0 else 0 for r in range(B)]
        else:
            new = [1 if lens[r] else 0 for r in range(B)]
        total = sum(new)
        granted = c.extend(i32(new, cuda), total)
        assert granted.tolist() == new
        lens = [a + b for a, b in zip(lens, new)]
        for layer in range(layers):
            k, v, q = mk(total, Hkv, D), mk(total, Hkv, D), mk(B, Hq, D)
            c.append(layer, k, v)
            o = c.attn(layer, q)
            at = 0
            for r in range(B):
                history[layer][r].append((k[at:at + new[r]], v[at:at + new[r]]))
                at += new[r]
                if lens[r] == 0:
                    assert (o[r] == 0).all()
                    continue
                K = torch.cat([x for x, _ in history[layer][r]]).transpose(0, 1)[None]
                V = torch.cat([x for _, x in history[layer][r]]).transpose(0, 1)[None]
                Q = torch.zeros(1, Hq, lens[r], D, device=cuda, dtype=q.dtype)
                Q[0, :, -1] = q[r]
                full = fa_p100.flash_attn(Q, K, V, True)[0, :, -1]
                # flash_attn rounds the weights, both the output, to fp16: together below 4 eps max |v|
                bound = 4 * torch.finfo(q.dtype).eps * V.float().abs().amax(2).repeat_interleave(2, 1)[0]
                assert ((o[r].float() - full.float()).abs() <= bound).all()
        if step % 10 == 9:
            fin = [rng.random() < 0.6 for _ in range(B)]
            c.release(torch.tensor(fin, device=cuda))
            for r in range(B):
                if fin[r]:
                    lens[r] = 0
                    for layer in range(layers):
                        history[layer][r] = []
        assert c.lens.tolist() == lens
        used = [p for r in range(B) for p in c.block_table[r, :pages_of(lens[r], 16)].tolist()]
        free = c.free_pages[:int(c.free_count)].tolist()
        assert sorted(used + free) == list(range(60))     # no page lost or given twice


def test_decode_step_in_a_graph(cuda):
    """A decoding step captured once and replayed gives the bits of eager steps, and
    two captured steps over different caches may run side by side."""
    B, Hq, Hkv, D = 5, 4, 2, 64
    runs = []
    for seed in (0, 1):
        pair = []
        for _ in range(2):
            c, mk = decode_setup(cuda, seed)
            c.extend(i32([7, 30, 1, 16, 0], cuda), 54)
            for layer in range(2):
                c.append(layer, mk(54, Hkv, D), mk(54, Hkv, D))
            pair.append((c, mk))
        runs.append(pair)
    one = i32([1, 1, 1, 1, 0], cuda)

    def step(c, rows, q, out):
        c.extend(one, 4)
        for layer in range(2):
            c.append(layer, rows[layer, 0], rows[layer, 1])
            out[layer].copy_(c.attn(layer, q))

    state = []
    for (eager, mk), (graphed, _) in runs:
        rows = mk(2, 2, 4, Hkv, D)
        q = mk(B, Hq, D)
        out_e, out_g = torch.empty(2, B, Hq, D, device=cuda).half(), torch.empty(2, B, Hq, D, device=cuda).half()
        # warm up on a cache of its own: a captured region must not be the first call
        warm, _ = decode_setup(cuda, 9)
        step(warm, rows, q, out_g)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(graphed, rows, q, out_g)
        state.append((eager, graphed, rows, q, out_e, out_g, g, mk))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(40):
        for eager, graphed, rows, q, out_e, out_g, g, mk in state:
            rows.copy_(mk(2, 2, 4, Hkv, D))
            q.copy_(mk(B, Hq, D))
            step(eager, rows, q, out_e)
        torch.cuda.synchronize()
        for s, st in zip(streams, state):
            with torch.cuda.stream(s):
                st[6].replay()
        torch.cuda.synchronize()
        for eager, graphed, rows, q, out_e, out_g, g, mk in state:
            assert torch.equal(out_e, out_g)
            assert torch.equal(eager.lens, graphed.lens)
            assert torch.equal(eager.block_table, graphed.block_table)
            assert torch.equal(eager.k, graphed.k) and torch.equal(eager.v, graphed.v)
    assert state[0][0].lens.tolist() == [47, 70, 41, 56, 0]


def test_first_calls_may_be_captured(cuda):
    """In a process of its own, the operators' very first calls inside a captured graph."""
    code = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import fa_p100_paged as paged
dev = torch.device("cuda", 0)
c = paged.PagedKVCache(1, 1, 64, 4000, 3, 20000, 16, torch.float16, dev)
new = torch.tensor([9000, 40, 1], dtype=torch.int32, device=dev)
fin = torch.tensor([True, False, True], device=dev)
k, q = torch.ones(9041, 1, 64, device=dev).half(), torch.ones(3, 1, 64, device=dev).half()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c.extend(new, 9041)
    c.append(0, k, k)
    o = c.attn(0, q)
    c.release(fin)
g.replay()
torch.cuda.synchronize()
assert c.lens.tolist() == [0, 40, 0] and int(c.free_count) == 4000 - 3
assert torch.equal(o, torch.ones_like(o))
"""
    import os
    import subprocess
    import sys
    res = subprocess.run([sys.executable, "-c", code, os.path.dirname(paged.__file__)],
                         capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stderr[-2000:]
