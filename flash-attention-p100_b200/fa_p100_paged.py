"""Generation with a paged key-value cache: what a model needs after `flash_attn`
has read its prompt. The reference has no cache (its HuggingFace backend refuses
one, fa_p100_hf.py:64-105); these operators have no counterpart there.

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
require a gradient are refused while gradients are recorded, and ones that carry a
forward-mode tangent always. What an operator writes in place counts as changed for
a backward that saved it.
"""
import ctypes

import torch

import _build
import _lib


def _load():
    """The operators' native half (csrc/fa_paged_py.cpp), built when it is missing
    or stale, over the library _lib loads."""
    _build.build_binding()
    import _fa_paged

    lib = _lib.lib()
    names = ("fa_b200_paged_extend", "fa_b200_paged_release", "fa_b200_paged_append", "fa_b200_paged_attn",
             "fa_b200_paged_attn_workspace_bytes", "fa_b200_paged_table_workspace_bytes",
             "fa_b200_status_string", "fa_b200_last_error")
    _fa_paged.bind({n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in names})
    return _fa_paged


_native = _load()
_I32 = torch.int32


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
    return _native.extend(new_lens, lens, block_table, free_pages, free_count, page_size, total_tokens,
                          lens_out, free_count_out)


def paged_release(finished, lens, block_table, free_pages, free_count, page_size, lens_out=None,
                  free_count_out=None):
    """Gives the pages of every request with finished[r] (bool) back: they go onto
    the stack `free_pages` (in place; requests in order, each one's pages in order)
    and the request's length becomes 0. The table's rows are left as they are. A
    page must belong to one request only. Returns (lens_out, free_count_out), new
    tensors or the caller's, as in paged_extend."""
    return _native.release(finished, lens, block_table, free_pages, free_count, page_size, lens_out,
                           free_count_out)


def paged_append(k, v, slots, k_cache, v_cache):
    """Writes the keys and values (T, Hkv, D) of T tokens into their slots of the
    caches, in place. slots is int32 (T,); a token whose slot is outside the cache
    (-1) is skipped, the others' slots must differ from each other. k and v may be
    strided views (slices of a fused projection); they have the caches' dtype. Caches
    that share memory with each other, k, v or slots are refused; slices of one
    buffer that interleave without an element in common are not."""
    _native.append(k, v, slots, k_cache, v_cache)


def paged_attn(q, k_cache, v_cache, block_table, lens):
    """Attention of one new token per request, q (B, Hq, D), over the request's
    cached tokens 0 .. lens[r] - 1 (the new token among them once it is appended).
    Returns (o, lse): o (B, Hq, D) in q's dtype, lse (B, Hq) fp32, natural log, as
    `fa_p100_ext.forward` gives them, in one allocation; a request of length 0 gets
    o = 0 and lse = -inf, and so does a head with nothing to add up: every token's
    page outside the cache, or every score -inf. Hq is a multiple of Hkv; what lies behind
    a request's last token in its last page is never used, whatever it holds. The same
    inputs give the same bits."""
    return _native.attn(q, k_cache, v_cache, block_table, lens)


class PagedKVCache:
    """The keys and values of up to `batch` requests of up to `max_len` tokens, for
    `layers` layers that share one block table, in `pages` pages of `page_size`
    tokens. `k` and `v` are (layers, pages, Hkv, page_size, D). Every method works
    in place and on the GPU alone, so a decoding step can be captured in a CUDA
    graph and replayed."""

    def __init__(self, layers, kv_heads, head_dim, pages, batch, max_len, page_size=64,
                 dtype=torch.float16, device=None):
        if dtype not in (torch.float16, torch.bfloat16):
            raise RuntimeError(f"the cache must be fp16 or bf16, got {dtype}")
        if head_dim not in (64, 128):
            raise RuntimeError(f"head dim must be 64 or 128, got {head_dim}")
        if min(layers, kv_heads, pages, batch, max_len) < 1:
            raise RuntimeError("layers, kv_heads, pages, batch and max_len must be positive")
        width = -(-max_len // page_size) if page_size > 0 else 0
        _native.check_page_size(page_size, pages, width)
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
