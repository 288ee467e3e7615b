"""Generation with a paged key-value cache: what a model needs after `flash_attn`
has read its prompt. The reference has no cache (its HuggingFace backend refuses
one, fa_p100_hf.py:103-105); these operators have no counterpart there.

    cache = PagedKVCache(layers, Hkv, D, pages, batch, max_len)
    cache.extend(new_lens, total_tokens)        # pages and slots for the new tokens
    cache.append(layer, k, v)                   # their keys and values, every layer
    o = cache.attn(layer, q)                    # one new token per request
    cache.release(finished)                     # pages of the requests that ended

`PagedKVCache` holds the tensors and calls the four operators below, which take
them one by one:

  * a cache is k_cache, v_cache (P, Hkv, page_size, D), fp16 or bf16: P pages of
    page_size tokens (a multiple of 16, at most 4096). Any strides whose D axis is
    contiguous and which are multiples of 16 bytes, so a (P, page_size, Hkv, D)
    cache is passed as its transpose(1, 2);
  * block_table int32 (B, W): row r lists request r's pages in order;
  * lens int32 (B): the tokens each request has;
  * free_pages int32 (P): a stack whose first free_count[0] entries are the free
    pages, taken from its top;
  * a token's slot is page * page_size + its offset in the page.

Everything stays on the GPU: the operators run on torch's current stream, never
wait for the GPU, and may be captured in a CUDA graph. Lengths, pages and slots
are data the host does not see, so the kernels check them: a request that cannot
be served is refused (granted 0, slots -1), and a table entry that names no page
of the cache leaves its tokens out of the attention and sets the device error
word, which `fa_p100.check_device_errors()` reports. Arguments the host can check raise
RuntimeError before anything is launched. There is no backward: tensors that
require a gradient are refused while gradients are recorded.
"""
import functools

import torch

import _lib

_I32 = torch.int32
_KINDS = {torch.float16: _lib.DTYPE_FP16, torch.bfloat16: _lib.DTYPE_BF16}
_DENSE = torch.contiguous_format
# a structure of three numbers costs ctypes as much as a small allocation
_Strides = functools.lru_cache(maxsize=4096)(_lib.Strides)


def _ints(t, name, shape, dtype=_I32):
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape:
        raise RuntimeError(f"{name} must be a {dtype} tensor of shape {tuple(shape)}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _table(block_table, B):
    """(W, row stride) of a block table of B rows."""
    if (not isinstance(block_table, torch.Tensor) or block_table.dtype is not _I32
            or block_table.dim() != 2 or block_table.size(0) != B or block_table.size(1) < 1):
        raise RuntimeError(f"block_table must be an int32 tensor of shape ({B}, W), W >= 1")
    W = block_table.size(1)
    row, col = block_table.stride()
    if (W > 1 and col != 1) or (B > 1 and row < W):
        raise RuntimeError("block_table: the columns must be contiguous and the rows apart")
    return W, row if B > 1 else W


def _check_page_size(page_size, P, W):
    if not 16 <= page_size <= 4096 or page_size % 16:
        raise RuntimeError(f"page_size must be a multiple of 16 up to 4096, got {page_size}")
    if P < 1:
        raise RuntimeError("the cache needs at least one page")
    if max(P, W) * page_size > 1 << 30:
        raise RuntimeError("a cache, or a row of the block table, may hold up to 2**30 tokens")


def _caches(k_cache, v_cache):
    """(P, Hkv, page_size, D) and the two layouts."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise RuntimeError(f"{name} must be (P, Hkv, page_size, D)")
    dtype, shape = k_cache.dtype, k_cache.shape
    if dtype not in _KINDS:
        raise RuntimeError("k_cache must be fp16 or bf16")
    if shape != v_cache.shape or v_cache.dtype is not dtype:
        raise RuntimeError("k_cache and v_cache must have one shape and one dtype")
    P, Hkv, page_size, D = shape
    if D != 64 and D != 128:
        raise RuntimeError(f"head dim must be 64 or 128, got {D}")
    if Hkv < 1:
        raise RuntimeError("the cache needs at least one head")
    _check_page_size(page_size, P, 1)
    sk, sv = _strides(k_cache, *k_cache.stride()), _strides(v_cache, *v_cache.stride())
    if sk is None or sv is None:
        raise RuntimeError("the caches' D axis must be contiguous, and their bases and strides "
                           "multiples of 16 bytes")
    return P, Hkv, page_size, D, sk, sv


def _strides(t, batch, head, row, d):
    """fa_b200_strides of a 16-bit tensor with these strides, None where 16-byte
    accesses cannot address it. The common case of _lib.strides_of without its
    look at every size; that one decides where a stride of this does not fit."""
    if d == 1 and not (batch | head | row) & 7 and batch and head and row and not t.data_ptr() & 15:
        return _Strides(batch, head, row)
    return _lib.strides_of(t) if t.dim() == 4 else None


def _on_device(names, *tensors):
    """Index of the one GPU that holds all tensors."""
    dev = tensors[0].get_device()
    for t, name in zip(tensors, names):
        if t.get_device() < 0:
            raise RuntimeError(f"{name} must be a CUDA tensor")
        if t.get_device() != dev:
            raise RuntimeError(f"{name} must be on cuda:{dev}, got {t.device}")
    return dev


def _no_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError("the paged cache has no backward: call it under torch.no_grad() or "
                                   "detach its inputs")


def _call(dev, name, *args):
    """Entry point `name` on GPU `dev`'s current stream."""
    fn = getattr(_lib.lib(), name)
    if torch.cuda.current_device() == dev:
        st = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _lib.check(st, name)


def _requests(lens, block_table, free_pages, free_count, page_size):
    """Checks what extend and release share; (B, W, row stride, P)."""
    if not isinstance(lens, torch.Tensor) or lens.dim() != 1 or lens.numel() < 1:
        raise RuntimeError("lens must be an int32 tensor of shape (B,), B >= 1")
    B = lens.numel()
    _ints(lens, "lens", (B,))
    W, stride = _table(block_table, B)
    P = free_pages.numel() if isinstance(free_pages, torch.Tensor) else 0
    _ints(free_pages, "free_pages", (P,))
    _ints(free_count, "free_count", (1,))
    _check_page_size(page_size, P, W)
    return B, W, stride, P


def _outputs(lens, lens_out, free_count_out, *sizes):
    """A workspace of 16 B + 16 bytes, int32 tensors of `sizes`, and the two
    counts where the caller gave none: views of one allocation, one call of the
    allocator instead of five (each costs as much host time as a kernel launch)."""
    B = lens.numel()
    sizes = (4 * B + 4, *sizes, *(() if lens_out is not None else (B,)),
             *(() if free_count_out is not None else (1,)))
    ws, *out = lens.new_empty(sum(sizes)).unsafe_split_with_sizes(sizes)
    if free_count_out is None:
        free_count_out = out.pop()
    else:
        _ints(free_count_out, "free_count_out", (1,))
    if lens_out is None:
        lens_out = out.pop()
    else:
        _ints(lens_out, "lens_out", (B,))
    if lens_out.get_device() != lens.get_device() or free_count_out.get_device() != lens.get_device():
        raise RuntimeError("lens_out and free_count_out must be on the device of lens")
    return ws, out, lens_out, free_count_out


def paged_extend(new_lens, lens, block_table, free_pages, free_count, page_size, total_tokens,
                 lens_out=None, free_count_out=None):
    """Room for new_lens[r] more tokens in every request r (negative counts as 0):
    takes the pages from the stack, writes them into `block_table` behind the
    request's pages so far (in place) and maps the tokens.

    Returns (slots, granted, lens_out, free_count_out). slots (total_tokens,)
    holds the slots of the new tokens packed request by request, -1 behind the
    last; granted (B,) is new_lens[r], or 0 for a refused request, whose tokens
    keep their places in `slots` with -1. Requests are served in order; one is
    refused if its row of the table or total_tokens has no room for it, or if the
    free pages do not cover what it and the requests before it need. lens_out and
    free_count_out are new tensors, or the caller's: pass lens and free_count
    themselves to update them in place."""
    B, W, stride, P = _requests(lens, block_table, free_pages, free_count, page_size)
    _ints(new_lens, "new_lens", (B,))
    total = int(total_tokens)
    if not 0 <= total <= 0x7fffffff:
        raise RuntimeError(f"total_tokens must be in [0, 2**31), got {total}")
    dev = _on_device(("lens", "new_lens", "block_table", "free_pages", "free_count"),
                     lens, new_lens, block_table, free_pages, free_count)
    ws, (slots, granted), lens_out, free_count_out = _outputs(lens, lens_out, free_count_out, total, B)
    _call(dev, "fa_b200_paged_extend", new_lens.data_ptr(), lens.data_ptr(), block_table.data_ptr(),
          stride, free_pages.data_ptr(), free_count.data_ptr(), slots.data_ptr(), granted.data_ptr(),
          lens_out.data_ptr(), free_count_out.data_ptr(), ws.data_ptr(), 16 * B + 16, B, W, P,
          page_size, total)
    return slots, granted, lens_out, free_count_out


def paged_release(finished, lens, block_table, free_pages, free_count, page_size, lens_out=None,
                  free_count_out=None):
    """Gives the pages of every request with finished[r] (bool) back: they go onto
    the stack `free_pages` (in place; requests in order, each one's pages in order)
    and the request's length becomes 0. The table's rows are left as they are. A
    page must belong to one request only. Returns (lens_out, free_count_out), new
    tensors or the caller's, as in paged_extend."""
    B, W, stride, P = _requests(lens, block_table, free_pages, free_count, page_size)
    _ints(finished, "finished", (B,), torch.bool)
    dev = _on_device(("lens", "finished", "block_table", "free_pages", "free_count"),
                     lens, finished, block_table, free_pages, free_count)
    ws, _, lens_out, free_count_out = _outputs(lens, lens_out, free_count_out)
    _call(dev, "fa_b200_paged_release", finished.data_ptr(), lens.data_ptr(), block_table.data_ptr(),
          stride, free_pages.data_ptr(), free_count.data_ptr(), lens_out.data_ptr(),
          free_count_out.data_ptr(), ws.data_ptr(), 16 * B + 16, B, W, P, page_size)
    return lens_out, free_count_out


def paged_append(k, v, slots, k_cache, v_cache):
    """Writes the keys and values (T, Hkv, D) of T tokens into their slots of the
    caches, in place. slots is int32 (T,); a token whose slot is outside the cache
    (-1) is skipped, the others' slots must differ from each other. k and v may be
    strided views (slices of a fused projection); they have the caches' dtype."""
    P, Hkv, page_size, D, skc, svc = _caches(k_cache, v_cache)
    for t, name in ((k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.size(1) != Hkv or t.size(2) != D:
            raise RuntimeError(f"{name} must be (T, {Hkv}, {D})")
        if t.dtype is not k_cache.dtype:
            raise RuntimeError(f"{name} must have the caches' dtype {k_cache.dtype}, got {t.dtype}")
    T = k.size(0)
    if T != v.size(0):
        raise RuntimeError("k and v must match")
    _ints(slots, "slots", (T,))
    for name, st in (("k_cache", skc), ("v_cache", svc)):
        if st.batch == 0 or st.head == 0 or st.row == 0:
            raise RuntimeError(f"{name} is written and must not be an expanded view")
    if k_cache.data_ptr() == v_cache.data_ptr():
        raise RuntimeError("k_cache and v_cache must be different memory")
    _no_grad(k, v, k_cache, v_cache)
    dev = _on_device(("k_cache", "v_cache", "k", "v", "slots"), k_cache, v_cache, k, v, slots)
    if T == 0:
        return
    (k, sk), (v, sv) = _token_rows(k), _token_rows(v)
    _call(dev, "fa_b200_paged_append", k.data_ptr(), sk, v.data_ptr(), sv, slots.data_ptr(),
          k_cache.data_ptr(), skc, v_cache.data_ptr(), svc, T, Hkv, D, P, page_size,
          _KINDS[k_cache.dtype])


def _token_rows(t):
    """(t, its strides) of a (T, H, D) tensor, a copy where the kernel's 16-byte
    accesses cannot address it."""
    row, head, d = t.stride()
    st = _strides(t, 0x40000000, head, row, d)   # no batch axis: any stride serves
    if st is None:
        t4 = t.permute(1, 0, 2).unsqueeze(0)
        st = _lib.strides_of(t4)
        if st is None:
            t = t.clone(memory_format=_DENSE)    # a new base: aligned
            st = _lib.strides_of(t.permute(1, 0, 2).unsqueeze(0))
    return t, st


@functools.lru_cache(maxsize=1024)
def _attn_workspace_bytes(dev, B, Hq, Hkv, W, D, page_size):
    with torch.cuda.device(dev):
        return _lib.lib().fa_b200_paged_attn_workspace_bytes(B, Hq, Hkv, W, D, page_size)


def paged_attn(q, k_cache, v_cache, block_table, lens):
    """Attention of one new token per request, q (B, Hq, D), over the request's
    cached tokens 0 .. lens[r] - 1 (the new token among them once it is appended).
    Returns (o, lse): o (B, Hq, D) in q's dtype, lse (B, Hq) fp32, natural log, as
    `fa_p100_ext.forward` gives them; a request of length 0 gets o = 0 and lse =
    -inf. Hq is a multiple of Hkv; what lies behind a request's last token in its
    last page is never used, whatever it holds. The same inputs give the same bits."""
    P, Hkv, page_size, D, skc, svc = _caches(k_cache, v_cache)
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.size(2) != D or q.size(0) < 1:
        raise RuntimeError(f"q must be (B, Hq, {D}), B >= 1")
    if q.dtype is not k_cache.dtype:
        raise RuntimeError(f"q must have the caches' dtype {k_cache.dtype}, got {q.dtype}")
    B, Hq, _ = shape = q.shape
    if Hq < 1 or Hq % Hkv:
        raise RuntimeError(f"query heads ({Hq}) must be a multiple of key/value heads ({Hkv})")
    _ints(lens, "lens", (B,))
    W, stride = _table(block_table, B)
    _check_page_size(page_size, P, W)
    _no_grad(q, k_cache, v_cache)
    dev = _on_device(("q", "k_cache", "v_cache", "block_table", "lens"),
                     q, k_cache, v_cache, block_table, lens)
    batch, head, d = q.stride()
    sq = _strides(q, batch, head, 8, d)          # no row axis
    if sq is None:
        sq = _lib.strides_of(q.unsqueeze(2))
        if sq is None:
            q = q.clone(memory_format=_DENSE)    # a new base: aligned
            sq = _lib.strides_of(q.unsqueeze(2))
    o = q.new_empty(shape)
    lse = q.new_empty((B, Hq), dtype=torch.float32)
    ws_bytes = _attn_workspace_bytes(dev, B, Hq, Hkv, W, D, page_size)
    ws = lens.new_empty(ws_bytes // 4) if ws_bytes else None
    _call(dev, "fa_b200_paged_attn", q.data_ptr(), sq, k_cache.data_ptr(), skc, v_cache.data_ptr(), svc,
          block_table.data_ptr(), stride, lens.data_ptr(), o.data_ptr(), _Strides(Hq * D, D, D),
          lse.data_ptr(), ws.data_ptr() if ws_bytes else None, ws_bytes, B, Hq, Hkv, D, P, W, page_size,
          _KINDS[q.dtype])
    return o, lse


class PagedKVCache:
    """The keys and values of up to `batch` requests of up to `max_len` tokens, for
    `layers` layers that share one block table, in `pages` pages of `page_size`
    tokens. `k` and `v` are (layers, pages, Hkv, page_size, D). Every method works
    in place and on the GPU alone, so a decoding step can be captured in a CUDA
    graph and replayed."""

    def __init__(self, layers, kv_heads, head_dim, pages, batch, max_len, page_size=64,
                 dtype=torch.float16, device=None):
        if dtype not in _KINDS:
            raise RuntimeError(f"the cache must be fp16 or bf16, got {dtype}")
        if head_dim not in (64, 128):
            raise RuntimeError(f"head dim must be 64 or 128, got {head_dim}")
        if min(layers, kv_heads, pages, batch, max_len) < 1:
            raise RuntimeError("layers, kv_heads, pages, batch and max_len must be positive")
        width = -(-max_len // page_size) if page_size > 0 else 0
        _check_page_size(page_size, pages, width)
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_size, self.max_len = page_size, width * page_size
        # zeroed once: memory never written holds no NaN that a dump of the cache would show
        self.k = torch.zeros((layers, pages, kv_heads, page_size, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.block_table = torch.full((batch, width), -1, dtype=_I32, device=device)
        self.lens = torch.zeros(batch, dtype=_I32, device=device)
        # the top of the stack is page 0
        self.free_pages = torch.arange(pages - 1, -1, -1, dtype=_I32, device=device)
        self.free_count = torch.full((1,), pages, dtype=_I32, device=device)
        self.slots = torch.empty(0, dtype=_I32, device=device)

    def extend(self, new_lens, total_tokens):
        """Room for the requests' new tokens; `append` and `attn` then work on them.
        Returns granted (B,): new_lens, 0 where a request was refused."""
        self.slots, granted, _, _ = paged_extend(
            new_lens, self.lens, self.block_table, self.free_pages, self.free_count, self.page_size,
            total_tokens, lens_out=self.lens, free_count_out=self.free_count)
        return granted

    def append(self, layer, k, v):
        """Keys and values (total_tokens, Hkv, D) of the tokens of the last `extend`."""
        paged_append(k, v, self.slots, self.k[layer], self.v[layer])

    def attn(self, layer, q):
        """Attention (B, Hq, D) of every request's newest token over its tokens."""
        return paged_attn(q, self.k[layer], self.v[layer], self.block_table, self.lens)[0]

    def release(self, finished):
        """Takes the pages of the requests with finished[r] back."""
        paged_release(finished, self.lens, self.block_table, self.free_pages, self.free_count,
                      self.page_size, lens_out=self.lens, free_count_out=self.free_count)
