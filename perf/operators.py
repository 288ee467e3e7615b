"""Cases and plain forms of the paged key-value cache and its attention.

Four operators that share one cache: `extend` hands pages to requests and maps
their new tokens to slots, `append` writes new keys and values into those slots,
`attn` is the attention of one new token per request over its pages, `release`
gives a finished request's pages back. A cache is (P, Hkv, ps, D): P pages of ps
tokens; a block table (B, W) int32 lists each request's pages; a token's slot is
page * ps + offset; the free pages are the first free_count entries of a stack.

`run` with own = False computes them with elementary torch operations; with
own = True it calls the package.
"""
import math
import os
import random
import sys

import torch

own = False

_GOLDEN = 0.6180339887498949
_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
# no drawn case moves more bytes than the largest listed one (about 1.1 GB)
_MAX_BYTES = 1.0e9


def _paged():
    """The package's module (only imported when its kernels are called)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "flash-attention-p100_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import fa_p100_paged
    return fa_p100_paged


def _spread(n, lo, hi):
    """n whole numbers spread evenly over [lo, hi] in a fixed scattered order."""
    if n == 1:
        return [hi]
    return [lo + int((hi - lo + 1) * (((i + 0.5) * _GOLDEN) % 1.0)) for i in range(n)]


def _pages(tokens, ps):
    return -(-tokens // ps)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of a serving batch: every request gains a token
        dict(name="extend_decode", op="extend", B=64, ps=16, width=512, ctx_lo=1, ctx_hi=8000,
             new_lo=1, new_hi=1, idle=0, free=2.0),
        # a thousand prompts of up to 2048 tokens admitted at once, some onto earlier turns
        dict(name="extend_prompts", op="extend", B=1024, ps=16, width=512, ctx_lo=0, ctx_hi=4096,
             new_lo=1, new_hi=2048, idle=16, free=1.1),
        # a few requests of a decoding batch end
        dict(name="release_few", op="release", B=64, ps=16, width=512, ctx_lo=1, ctx_hi=8192,
             every=8),
        # half of a very large offline batch ends
        dict(name="release_many", op="release", B=2048, ps=16, width=512, ctx_lo=1, ctx_hi=8192,
             every=2),
        # one token per request of a decoding batch, one layer of a 16/8-head model
        dict(name="append_decode", op="append", T=64, Hkv=8, D=128, ps=16, pages=8192,
             dtype="bf16", fused=4, drop=0, layout="head"),
        # one ragged prompt of a multi-query model, k and v sliced out of a fused projection
        dict(name="append_ragged", op="append", T=1537, Hkv=1, D=64, ps=64, pages=500,
             dtype="fp16", fused=18, drop=7, layout="row"),
        # a long prompt batch written by one layer
        dict(name="append_prompts", op="append", T=65536, Hkv=8, D=128, ps=16, pages=4608,
             dtype="fp16", fused=0, drop=0, layout="head"),
        # one chat request: latency
        dict(name="attn_one", op="attn", B=1, Hq=16, Hkv=8, D=128, ps=16, len_lo=1000, len_hi=1000,
             width=512, empty=0, dtype="fp16", layout="head"),
        # one request over a very long context
        dict(name="attn_long", op="attn", B=1, Hq=32, Hkv=8, D=128, ps=64, len_lo=131001,
             len_hi=131001, width=2048, empty=0, dtype="fp16", layout="head"),
        # a ragged serving batch with grouped heads, some of its rows without a request
        dict(name="attn_ragged", op="attn", B=64, Hq=32, Hkv=8, D=128, ps=16, len_lo=1,
             len_hi=8192, width=512, empty=3, dtype="bf16", layout="head"),
        # multi-query attention, ragged lengths
        dict(name="attn_mqa", op="attn", B=32, Hq=16, Hkv=1, D=64, ps=64, len_lo=1, len_hi=1537,
             width=32, empty=0, dtype="fp16", layout="head"),
        # multi-head attention, pages stored token by token
        dict(name="attn_mha", op="attn", B=16, Hq=16, Hkv=16, D=64, ps=32, len_lo=512,
             len_hi=2048, width=64, empty=0, dtype="bf16", layout="row"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["extend", "release", "append", "append", "attn", "attn", "attn"])
    ps = rng.choice([16, 32, 48, 64, 128])
    if op in ("extend", "release"):
        B = _log(rng, 1, 2048)
        ctx_hi = _log(rng, 1, 8192)
        case = dict(op=op, B=B, ps=ps, ctx_lo=rng.choice([0, 1, ctx_hi]), ctx_hi=ctx_hi)
        if op == "release":
            case.update(every=rng.choice([1, 2, 3, 8]), width=_pages(ctx_hi, ps) + rng.randrange(9))
        else:
            new_hi = rng.choice([1, _log(rng, 1, max(1, min(4096, (1 << 20) // B)))])
            case.update(new_lo=rng.choice([1, new_hi]), new_hi=new_hi, idle=rng.randrange(B),
                        free=rng.choice([0.0, 0.5, 1.0, 1.5]),
                        width=max(1, _pages(ctx_hi + new_hi, ps) - rng.choice([0, 0, 1])
                                  + rng.choice([0, 5])))
        return case
    dtype = rng.choice(["fp16", "bf16"])
    layout = rng.choice(["head", "row"])
    D = rng.choice([64, 128])
    if op == "append":
        Hkv = rng.choice([1, 2, 5, 8, 16])
        T = _log(rng, 1, 65536)
        T = max(1, min(T, int(_MAX_BYTES / (8 * Hkv * D))))
        return dict(op=op, T=T, Hkv=Hkv, D=D, ps=ps, pages=_pages(T, ps) + _log(rng, 1, 500),
                    dtype=dtype, fused=rng.choice([0, Hkv * 2, Hkv * 4]),
                    drop=rng.choice([0, 0, T // 3]), layout=layout)
    Hq, Hkv = rng.choice([(16, 8), (32, 8), (16, 1), (16, 16), (8, 8), (40, 8), (6, 2), (32, 1),
                          (64, 8), (12, 12)])
    B = _log(rng, 1, 256)
    room = int(_MAX_BYTES / (4 * Hkv * D * B))
    len_hi = _log(rng, 1, max(1, min(262144, room)))
    return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, D=D, ps=ps, len_lo=rng.choice([1, len_hi // 2 + 1, len_hi]),
                len_hi=len_hi, width=_pages(len_hi, ps) + rng.choice([0, 3, 40]),
                empty=rng.choice([0, 0, (B - 1) // 4]), dtype=dtype, layout=layout)


def _attn_lens(case):
    lens = _spread(case["B"], case["len_lo"], case["len_hi"])
    for i in range(case["empty"]):
        lens[(i * 7) % case["B"]] = 0
    return lens


def _extend_lens(case):
    """(length so far, new tokens) of every request."""
    B = case["B"]
    ctx = _spread(B, case["ctx_lo"], case["ctx_hi"])
    new = _spread(B, case["new_lo"], case["new_hi"])
    for i in range(case["idle"]):
        new[(i * 5) % B] = 0
    cap = case["width"] * case["ps"]
    return [(min(c, cap), n) for c, n in zip(ctx, new[::-1])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _cache(case, pages, gen):
    """A (pages, Hkv, ps, D) cache; layout "row" stores it (pages, ps, Hkv, D)."""
    Hkv, ps, D = case["Hkv"], case["ps"], case["D"]
    shape = (pages, Hkv, ps, D) if case["layout"] == "head" else (pages, ps, Hkv, D)
    t = torch.randn(shape, device="cuda", generator=gen, dtype=_DT[case["dtype"]])
    return t if case["layout"] == "head" else t.transpose(1, 2)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _tables(lens, width, ps, perm):
    """A block table whose rows hold their pages in turn from `perm` (-1 behind
    them), made on the host, and the number of pages in use."""
    need = torch.tensor([_pages(n, ps) for n in lens])
    start = torch.cumsum(need, 0) - need
    j = torch.arange(width)
    at = (start[:, None] + j).clamp(max=perm.numel() - 1)
    table = torch.where(j < need[:, None], perm[at], torch.full_like(at, -1))
    return table.to(torch.int32).cuda(), int(need.sum())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed + 1)
    rng = random.Random(seed + 2)
    op, ps = case["op"], case["ps"]
    s = dict(op=op, ps=ps)
    if op == "append":
        T, Hkv, D = case["T"], case["Hkv"], case["D"]
        dt = _DT[case["dtype"]]
        s["k_cache"] = _cache(case, case["pages"], gen)
        s["v_cache"] = _cache(case, case["pages"], gen)
        if case["fused"]:
            # rows of a fused projection: `fused` heads wide, k and v the last 2 Hkv of them
            rows = torch.randn(T, case["fused"] + 2 * Hkv, D, device="cuda", generator=gen, dtype=dt)
            s["k"], s["v"] = rows[:, -2 * Hkv:-Hkv], rows[:, -Hkv:]
        else:
            s["k"] = torch.randn(T, Hkv, D, device="cuda", generator=gen, dtype=dt)
            s["v"] = torch.randn(T, Hkv, D, device="cuda", generator=gen, dtype=dt)
        if T >= 1024:     # prompts: runs of tokens, whole pages after another in scattered order
            page = torch.randperm(case["pages"], generator=host)[:_pages(T, ps)]
            t = torch.arange(T)
            slots = page[t // ps] * ps + t % ps
        else:             # decoding: a token per request, each in a page of its own where they suffice
            slots = torch.randperm(case["pages"] * ps, generator=host)[:T]
        slots = slots.to(torch.int32)
        if case["drop"]:  # tokens whose request got no pages
            slots[torch.randperm(T, generator=host)[:case["drop"]]] = -1
        s["slots"] = slots.cuda()
        return s
    if op == "attn":
        lens = _attn_lens(case)
        rng.shuffle(lens)
        pages = sum(_pages(n, ps) for n in lens) + 8
        perm = torch.randperm(pages, generator=host)
        s["table"], _ = _tables(lens, case["width"], ps, perm)
        s["lens"] = _i32(lens)
        s["k_cache"] = _cache(case, pages, gen)
        s["v_cache"] = _cache(case, pages, gen)
        s["q"] = torch.randn(case["B"], case["Hq"], case["D"], device="cuda", generator=gen,
                             dtype=_DT[case["dtype"]])
        return s
    if op == "extend":
        pairs = _extend_lens(case)
        rng.shuffle(pairs)
        lens = [c for c, _ in pairs]
        need = sum(_pages(c + n, ps) - _pages(c, ps) for c, n in pairs)
        used = sum(_pages(c, ps) for c in lens)
        free = int(need * case["free"])
        pages = used + free + 3
        s["new_lens"] = _i32([n for _, n in pairs])
        s["total"] = sum(n for _, n in pairs)
    else:
        lens = _spread(case["B"], case["ctx_lo"], case["ctx_hi"])
        rng.shuffle(lens)
        used = sum(_pages(c, ps) for c in lens)
        free = 5
        pages = used + free
        fin = [(i + seed) % case["every"] == 0 for i in range(case["B"])]
        rng.shuffle(fin)
        s["finished"] = torch.tensor(fin).cuda()
    perm = torch.randperm(pages, generator=host)
    s["table"], _ = _tables(lens, case["width"], ps, perm)
    s["lens"] = _i32(lens)
    stack = torch.full((pages,), -1, dtype=torch.int32)
    stack[:free] = perm[used:used + free].to(torch.int32)
    s["free_pages"] = stack.cuda()
    s["free_count"] = _i32([free])
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_extend(s):
    ps, T = s["ps"], s["total"]
    table, stack = s["table"], s["free_pages"].long()
    B, W = table.shape
    P = stack.numel()
    length, new = s["lens"].long(), s["new_lens"].long().clamp(min=0)
    count = s["free_count"].long().clamp(0, P)
    end = torch.cumsum(new, 0)
    fits = (new > 0) & (length >= 0) & (length + new <= W * ps) & (end <= T)
    p0 = (length + ps - 1) // ps
    p1 = (length + new + ps - 1) // ps
    want = torch.where(fits, p1 - p0, 0)
    csum = torch.cumsum(want, 0)
    ok = fits & ((want == 0) | (csum <= count))
    granted = torch.where(ok, new, 0)
    taken = torch.where(ok & (want > 0), csum, 0).max()
    j = torch.arange(W, device=table.device)
    fresh = ok[:, None] & (j >= p0[:, None]) & (j < p1[:, None])
    at = count - 1 - (csum - want)[:, None] - (j - p0[:, None])
    table.copy_(torch.where(fresh, stack[at.clamp(0, P - 1)], table.long()))
    t = torch.arange(T, device=table.device)
    r = torch.searchsorted(end, t, right=True)
    inside = r < B
    r = r.clamp(max=B - 1)
    pos = (length + new - end)[r] + t
    page = table[r, (pos // ps).clamp(0, W - 1)].long()
    good = inside & ok[r] & (page >= 0) & (page < P)
    slots = torch.where(good, page * ps + pos % ps, -1)
    i32 = torch.int32
    return (slots.to(i32), granted.to(i32), (length + granted).to(i32), (count - taken).to(i32), table)


def _plain_release(s):
    ps, table = s["ps"], s["table"]
    B, W = table.shape
    P = s["free_pages"].numel()
    length, fin = s["lens"].long(), s["finished"]
    n = torch.where(fin, (length.clamp(0, W * ps) + ps - 1) // ps, 0)
    back = torch.arange(W, device=table.device) < n[:, None]
    count = s["free_count"].long().clamp(0, P)
    at = count + torch.cumsum(back.reshape(-1).long(), 0) - 1
    at = torch.where(back.reshape(-1) & (at < P), at, P)
    stack = torch.cat([s["free_pages"], s["free_pages"][:1]])
    stack[at] = table.reshape(-1)
    stack = stack[:P]
    s["free_pages"].copy_(stack)
    i32 = torch.int32
    return (torch.where(fin, 0, length).to(i32), (count + n.sum()).clamp(max=P).to(i32),
            s["free_pages"])


def _plain_append(s):
    ps, slots = s["ps"], s["slots"].long()
    P = s["k_cache"].size(0)
    good = (slots >= 0) & (slots < P * ps)
    # rows without a slot repeat the first row that has one (the same values to the same place);
    # where no row has one, what is in slot 0 is put back
    first = good.to(torch.int8).argmax()
    some = good[first]
    row = torch.where(good, torch.arange(slots.numel(), device=slots.device), first)
    at = torch.where(some, slots[row], 0)
    page, off = at // ps, at % ps
    for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
        cache[page, :, off] = torch.where(some, new[row], cache[page, :, off])
    return s["k_cache"], s["v_cache"]


def _plain_attn(s):
    q, lens = s["q"], s["lens"]
    B, Hq, D = q.shape
    P, Hkv, ps, _ = s["k_cache"].shape
    W = s["table"].size(1)
    out, lses = [], []
    j = torch.arange(W * ps, device=q.device)
    for b in range(B):
        page = s["table"][b].long().clamp(0, P - 1)
        k = s["k_cache"][page].transpose(0, 1).reshape(Hkv, W * ps, D).float()
        v = s["v_cache"][page].transpose(0, 1).reshape(Hkv, W * ps, D).float()
        seen = j < lens[b]
        x = q[b].float().reshape(Hkv, Hq // Hkv, D) @ k.transpose(1, 2) / math.sqrt(D)
        x = x.masked_fill(~seen, -math.inf)
        m = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
        l = p.sum(-1, keepdim=True)
        v = torch.where(seen[:, None], v, 0.0)
        out.append((p @ v / torch.where(l == 0, 1.0, l)).reshape(Hq, D))
        lses.append((m + torch.log(l)).reshape(Hq))
    return torch.stack(out).to(q.dtype), torch.stack(lses)


def run(state):
    s = state
    op = s["op"]
    if not own:
        return {"extend": _plain_extend, "release": _plain_release, "append": _plain_append,
                "attn": _plain_attn}[op](s)
    paged = _paged()
    if op == "extend":
        slots, granted, lens, count = paged.paged_extend(
            s["new_lens"], s["lens"], s["table"], s["free_pages"], s["free_count"], s["ps"], s["total"])
        return slots, granted, lens, count, s["table"]
    if op == "release":
        lens, count = paged.paged_release(s["finished"], s["lens"], s["table"], s["free_pages"],
                                          s["free_count"], s["ps"])
        return lens, count, s["free_pages"]
    if op == "append":
        paged.paged_append(s["k"], s["v"], s["slots"], s["k_cache"], s["v_cache"])
        return s["k_cache"], s["v_cache"]
    o, lse = paged.paged_attn(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"])
    return o, lse


def exact(case, seed):
    """The attention in 64 bits, key by key from the definition, and the caches
    after a copy of the rows that have a slot; the other operators give whole
    numbers."""
    if case["op"] in ("extend", "release"):
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        kept = s["slots"] >= 0
        page, off = s["slots"][kept].long() // s["ps"], s["slots"][kept].long() % s["ps"]
        caches = []
        for cache, new in ((s["k_cache"], s["k"]), (s["v_cache"], s["v"])):
            by_token = cache.double().transpose(1, 2).contiguous()
            by_token[page, off] = new[kept].double()
            caches.append(by_token.transpose(1, 2))
        return tuple(caches)
    q = s["q"].double()
    B, Hq, D = q.shape
    _, Hkv, ps, _ = s["k_cache"].shape
    group = Hq // Hkv
    o = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64, device=q.device)
    lens = s["lens"].tolist()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        slot = torch.arange(n, device=q.device)
        page = s["table"][b, slot // ps].long()
        for g in range(Hkv):
            keys = s["k_cache"][page, g, slot % ps].double()
            values = s["v_cache"][page, g, slot % ps].double()
            heads = slice(g * group, (g + 1) * group)
            w = torch.einsum("hd,nd->hn", q[b, heads], keys) * D ** -0.5
            top = w.max(dim=1).values
            e = torch.exp(w - top[:, None])
            z = e.sum(dim=1)
            o[b, heads] = torch.einsum("hn,nd->hd", e, values) / z[:, None]
            lse[b, heads] = top + torch.log(z)
    return o, lse


def work(case):
    ps = case["ps"]
    if case["op"] == "append":
        done = case["T"] - case["drop"]
        return {"bytes": 8 * done * case["Hkv"] * case["D"] + 4 * case["T"], "flops": 0}
    if case["op"] == "attn":
        lens = _attn_lens(case)
        total = sum(lens)
        B, Hq, Hkv, D = case["B"], case["Hq"], case["Hkv"], case["D"]
        return {"bytes": (4 * total * Hkv * D + 4 * B * Hq * D + 4 * B * Hq
                          + 4 * sum(_pages(n, ps) for n in lens) + 4 * B),
                "flops": 4 * total * Hq * D}
    B = case["B"]
    if case["op"] == "extend":
        pairs = _extend_lens(case)
        tokens = sum(n for _, n in pairs)
        fresh = sum(_pages(c + n, ps) - _pages(c, ps) for c, n in pairs)
        return {"bytes": 16 * B + 8 + 4 * tokens + 8 * int(fresh * min(1.0, case["free"])), "flops": 0}
    lens = _spread(B, case["ctx_lo"], case["ctx_hi"])
    back = sum(_pages(n, ps) for n in lens) // case["every"]
    return {"bytes": 9 * B + 8 + 8 * back, "flops": 0}
