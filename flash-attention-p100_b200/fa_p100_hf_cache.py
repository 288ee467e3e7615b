"""The paged key-value cache as a transformers cache, for generation through the
"fa_p100" backend:

    from fa_p100_hf import enable_fa_p100, make_cache
    enable_fa_p100(model)
    cache = make_cache(model, batch=4, max_len=4096)
    model.generate(ids, past_key_values=cache, use_cache=True, max_new_tokens=100)

No counterpart in the reference, whose backend refuses every cache
(fa_p100_hf.py:64-105). A prompt runs through flash_attn as without a cache and
leaves its keys and values in the pages; every token after it runs through
fa_p100_paged.paged_attn over them. All sequences of a batch have one length, as
the backend takes no padding. What it cannot do raises: a second prompt on a
cache that already holds tokens (NotImplementedError), beam search and other
calls that reorder or cut a cache (NotImplementedError), more than max_len tokens
(RuntimeError), a model whose attention is not "fa_p100" (RuntimeError: it would
see the newest tokens alone), and, as the cache has no backward, keys that need a
gradient (RuntimeError).
"""
import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from fa_p100_paged import PagedKVCache


class _PagedLayer(CacheLayerMixin):
    """One layer's view of the pages. `update` stores the new keys and values and
    hands them on with a mark from which the attention call finds this layer."""

    is_compileable = False
    is_sliding = False

    def __init__(self, cache, index):
        super().__init__()
        self._cache, self._index, self._tokens = cache, index, 0

    def lazy_initialization(self, key_states, value_states):
        self.is_initialized = True

    def update(self, key_states, value_states, *args, **kwargs):
        c = self._cache
        if c.handed is not None:
            raise RuntimeError(
                f"the keys that layer {c.handed} got from this cache did not reach the fa_p100 attention, and any other "
                "would see the newest tokens alone: call enable_fa_p100 on the model (or, if that call failed, "
                "reset the cache)")
        B, heads, N, D = key_states.shape
        if self._tokens and N > 1:              # before anything is stored
            raise NotImplementedError(
                f"fa_p100 adds one token at a time to a cache that holds tokens ({self._tokens} here, "
                f"{N} new); reset the cache, or run the prompt in one call")
        if B != c.batch:
            raise RuntimeError(f"this cache was made for a batch of {c.batch}, got {B}")
        if self._tokens == c.tokens:            # the first layer of a step
            c.extend(N)
        elif self._tokens + N != c.tokens:
            raise RuntimeError(f"layer {self._index} got {N} tokens where an earlier one got "
                               f"{c.tokens - self._tokens}")
        dtype = c.paged.k.dtype
        rows = [t.to(dtype).transpose(1, 2).reshape(B * N, heads, D) for t in (key_states, value_states)]
        c.paged.append(self._index, *rows)
        past, self._tokens = self._tokens, self._tokens + N
        # a tensor of its own to carry the mark: the caller's may serve elsewhere
        key_states = key_states.view_as(key_states)
        key_states._fa_p100_paged = (self, past)
        c.handed = self._index
        return key_states, value_states

    def reached(self):
        """The attention call has this layer's keys."""
        self._cache.handed = None

    def attention(self, query):
        """(B, 1, Hq, D) of the queries (B, Hq, 1, D) of the newest tokens."""
        paged = self._cache.paged
        return paged.attn(self._index, query.squeeze(2).to(paged.k.dtype)).unsqueeze(1)

    def get_mask_sizes(self, query_length):
        # transformers 5 passes the query length, earlier ones the tokens' positions
        n = query_length if isinstance(query_length, int) else query_length.shape[0]
        return self._tokens + n, 0

    def get_seq_length(self, *args):
        return self._tokens

    def get_max_cache_shape(self):
        return self._cache.paged.max_len

    def reset(self):
        self._tokens = 0

    def _refuse(self, *args, **kwargs):
        raise NotImplementedError("the fa_p100 cache keeps its sequences in place: no beam search, "
                                  "no cutting or repeating of a cache")

    reorder_cache = crop = batch_repeat_interleave = batch_select_indices = offload = prefetch = _refuse


class FaP100Cache(Cache):
    """A transformers cache whose layers share one PagedKVCache."""

    _fa_p100_paged = True

    def __init__(self, layers, kv_heads, head_dim, batch, max_len, page_size=64, dtype=torch.float16,
                 device=None):
        if max_len < 1 or page_size < 1:
            raise RuntimeError("max_len and page_size must be positive")
        self.batch, self.tokens = batch, 0
        self.handed = None      # the layer whose keys are on their way to its attention call
        # a full row of pages for every sequence: no request is ever refused
        pages = batch * -(-max_len // page_size)
        self.paged = PagedKVCache(layers, kv_heads, head_dim, pages, batch, max_len, page_size, dtype, device)
        super().__init__(layers=[_PagedLayer(self, i) for i in range(layers)])

    def extend(self, tokens):
        if self.tokens + tokens > self.paged.max_len:
            raise RuntimeError(f"the cache holds {self.paged.max_len} tokens a sequence, {self.tokens} are "
                               f"in it and {tokens} more do not fit")
        new = torch.full((self.batch,), tokens, dtype=torch.int32, device=self.paged.lens.device)
        self.paged.extend(new, self.batch * tokens)
        self.tokens += tokens

    def reset(self):
        """Empties the cache for another batch of prompts."""
        if self.tokens:
            self.paged.release(torch.ones(self.batch, dtype=torch.bool, device=self.paged.lens.device))
        self.tokens, self.handed = 0, None
        for layer in self.layers:
            layer.reset()
