"""The paged cache without a GPU: every refusal of the Python operators and of the
C entry points comes before a kernel is reached."""
import pytest
import torch

import _lib
import fa_p100_paged as paged

P = 4096          # a 16-byte aligned fake device address, never dereferenced


def ints(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype)


def cache(pages=4, Hkv=2, ps=16, D=64, dtype=torch.float16):
    return torch.zeros(pages, Hkv, ps, D, dtype=dtype)


def extend(**kw):
    a = dict(new_lens=ints(3), lens=ints(3), block_table=ints(3, 5), free_pages=ints(4),
             free_count=ints(1), page_size=16, total_tokens=7)
    a.update(kw)
    return paged.paged_extend(**a)


@pytest.mark.parametrize("kw,match", [
    (dict(lens=ints(3, 1)), "lens"),
    (dict(lens=ints(0)), "lens"),
    (dict(lens=ints(3, dtype=torch.int64)), "lens"),
    (dict(new_lens=ints(2)), "new_lens"),
    (dict(new_lens=ints(6)[::2]), "contiguous"),
    (dict(block_table=ints(2, 5)), "block_table"),
    (dict(block_table=ints(3, 0)), "block_table"),
    (dict(block_table=ints(5, 3).t()), "columns"),
    (dict(block_table=ints(1, 5).expand(3, 5)), "rows"),
    (dict(free_pages=ints(0)), "page"),
    (dict(free_pages=ints(2, 2)), "free_pages"),
    (dict(free_count=ints(2)), "free_count"),
    (dict(page_size=8), "page_size"),
    (dict(page_size=24), "page_size"),
    (dict(page_size=8192), "page_size"),
    (dict(page_size=4096, free_pages=ints((1 << 18) + 1)), "2\\*\\*30"),
    (dict(total_tokens=-1), "total_tokens"),
    (dict(lens_out=ints(4)), "CUDA"),
    (dict(), "CUDA"),
])
def test_extend_refusals(kw, match):
    with pytest.raises(RuntimeError, match=match):
        extend(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(finished=ints(3)), "finished"),
    (dict(finished=ints(4, dtype=torch.bool)), "finished"),
    (dict(lens=None), "lens"),
    (dict(page_size=0), "page_size"),
    (dict(), "CUDA"),
])
def test_release_refusals(kw, match):
    a = dict(finished=ints(3, dtype=torch.bool), lens=ints(3), block_table=ints(3, 5),
             free_pages=ints(4), free_count=ints(1), page_size=16)
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        paged.paged_release(**a)


def rows(T=5, H=2, D=64, dtype=torch.float16):
    return torch.zeros(T, H, D, dtype=dtype)


@pytest.mark.parametrize("kw,match", [
    (dict(k=rows(H=3)), "k must be"),
    (dict(v=rows(D=128)), "v must be"),
    (dict(v=rows(T=6)), "match"),
    (dict(k=rows(dtype=torch.bfloat16)), "dtype"),
    (dict(k=rows().requires_grad_(True)), "backward"),
    (dict(slots=ints(4)), "slots"),
    (dict(slots=ints(5, dtype=torch.int64)), "slots"),
    (dict(k_cache=cache(D=96), v_cache=cache(D=96)), "head dim"),
    (dict(k_cache=cache(ps=20), v_cache=cache(ps=20)), "page_size"),
    (dict(k_cache=cache(pages=0), v_cache=cache(pages=0)), "page"),
    (dict(v_cache=cache(pages=5)), "one shape"),
    (dict(v_cache=cache(dtype=torch.bfloat16)), "one shape"),
    (dict(k_cache=cache(dtype=torch.float32)), "fp16 or bf16"),
    (dict(k_cache=torch.zeros(4, 2, 16, 68, dtype=torch.float16)[..., :64]), "16 bytes"),
    (dict(k_cache=cache(Hkv=1).expand(4, 2, 16, 64)), "expanded"),
    (dict(), "CUDA"),
])
def test_append_refusals(kw, match):
    a = dict(k=rows(), v=rows(), slots=ints(5), k_cache=cache(), v_cache=cache())
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        paged.paged_append(**a)


def test_append_refuses_one_cache_for_both():
    c = cache()
    with pytest.raises(RuntimeError, match="different memory"):
        paged.paged_append(rows(), rows(), ints(5), c, c)


@pytest.mark.parametrize("kw,match", [
    (dict(q=rows(3, 4, 128)), "q must be"),
    (dict(q=rows(0, 4)), "q must be"),
    (dict(q=rows(3, 3)), "multiple"),
    (dict(q=rows(3, 4, dtype=torch.bfloat16)), "dtype"),
    (dict(q=rows(3, 4).requires_grad_(True)), "backward"),
    (dict(lens=ints(2)), "lens"),
    (dict(block_table=ints(2, 5)), "block_table"),
    (dict(), "CUDA"),
])
def test_attn_refusals(kw, match):
    a = dict(q=rows(3, 4), k_cache=cache(), v_cache=cache(), block_table=ints(3, 5), lens=ints(3))
    a.update(kw)
    with pytest.raises(RuntimeError, match=match):
        paged.paged_attn(**a)


def test_cache_refusals():
    ok = dict(layers=1, kv_heads=1, head_dim=64, pages=1, batch=1, max_len=1, device="cpu")
    for kw in (dict(head_dim=80), dict(dtype=torch.float32), dict(pages=0), dict(max_len=0),
               dict(page_size=0), dict(page_size=40)):
        with pytest.raises(RuntimeError):
            paged.PagedKVCache(**{**ok, **kw})
    c = paged.PagedKVCache(**{**ok, "max_len": 130, "batch": 2, "pages": 7})
    assert c.max_len == 192 and tuple(c.block_table.shape) == (2, 3)
    assert c.free_pages.tolist() == [6, 5, 4, 3, 2, 1, 0] and c.free_count.tolist() == [7]


# ---- the C entry points ----
S = _lib.Strides(2 * 16 * 64, 16 * 64, 64)


def c_extend(new_lens=P, table=P, stride=5, slots=P, ws=P, ws_bytes=1 << 20, B=3, W=5, pages=4,
             ps=16, T=7):
    return _lib.lib().fa_b200_paged_extend(new_lens, P, table, stride, P, P, slots, P, P, P, ws,
                                           ws_bytes, B, W, pages, ps, T, None)


def test_extend_argument_errors():
    assert c_extend(new_lens=None) == 1
    assert c_extend(slots=None) == 1
    assert c_extend(B=0) == 3
    assert c_extend(T=-1) == 3
    assert c_extend(stride=4) == 3
    assert c_extend(ps=17) == 13
    assert c_extend(ps=0) == 13
    assert c_extend(pages=0) == 13
    assert c_extend(W=(1 << 26) + 1, stride=1 << 27) == 13
    assert c_extend(ws=None) == 7
    need = _lib.lib().fa_b200_paged_table_workspace_bytes(3)
    assert need == 16 * 3 + 16
    assert c_extend(ws_bytes=need - 1) == 7
    assert c_extend(ws=P + 8) == 4


def c_release(finished=P, stride=5, ws_bytes=1 << 20, B=3, ps=16):
    return _lib.lib().fa_b200_paged_release(finished, P, P, stride, P, P, P, P, P, ws_bytes, B, 5, 4,
                                            ps, None)


def test_release_argument_errors():
    assert c_release(finished=None) == 1
    assert c_release(B=-1) == 3
    assert c_release(stride=1) == 3
    assert c_release(ps=32768) == 13
    assert c_release(ws_bytes=0) == 7


def c_append(k=P, sk=S, skc=S, T=5, Hkv=2, D=64, ps=16, dtype=0):
    return _lib.lib().fa_b200_paged_append(k, sk, P, S, P, P, skc, P, S, T, Hkv, D, 4, ps, dtype, None)


def test_append_argument_errors():
    assert c_append(k=None) == 1
    assert c_append(k=None, T=0) == 0          # nothing to write
    assert c_append(T=-1) == 3
    assert c_append(Hkv=0) == 3
    assert c_append(D=80) == 2
    assert c_append(ps=15) == 13
    assert c_append(dtype=2) == 11
    assert c_append(k=P + 2) == 4
    assert c_append(sk=_lib.Strides(0, 68, 64)) == 4
    assert c_append(skc=_lib.Strides(2 * 16 * 64, -64, 64)) == 4


def c_attn(q=P, sq=S, stride=5, B=3, Hq=4, Hkv=2, D=64, pages=4, W=5, ps=16, dtype=0):
    return _lib.lib().fa_b200_paged_attn(q, sq, P, S, P, S, P, stride, P, P, S, P, P, 1 << 30, B, Hq, Hkv,
                                         D, pages, W, ps, dtype, None)


def test_attn_argument_errors():
    assert c_attn(q=None) == 1
    assert c_attn(D=96) == 2
    assert c_attn(Hq=3) == 3
    assert c_attn(B=0) == 3
    assert c_attn(stride=4) == 3
    assert c_attn(ps=100) == 13
    assert c_attn(pages=1 << 27) == 13
    assert c_attn(dtype=5) == 11
    assert c_attn(q=P + 1) == 4
    assert c_attn(sq=_lib.Strides(4 * 64 + 4, 64, 64)) == 4
    assert "page" in _lib.status_string(13)


# ---- the HuggingFace cache ----
def _model():
    import fa_p100_hf
    from transformers import Qwen3Config, Qwen3ForCausalLM
    cfg = Qwen3Config(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=2,
                      num_attention_heads=2, num_key_value_heads=1, head_dim=64,
                      max_position_embeddings=64, tie_word_embeddings=True)
    return fa_p100_hf.enable_fa_p100(Qwen3ForCausalLM(cfg))


def test_hf_cache_shape_and_guards():
    import fa_p100_hf
    model = _model()
    cache = fa_p100_hf.make_cache(model, batch=3, max_len=100, page_size=32)
    assert cache.paged.k.shape == (2, 12, 1, 32, 64) and cache.paged.k.dtype == torch.float16
    assert len(cache.layers) == 2 and cache.get_seq_length() == 0 and cache.get_max_cache_shape() == 128
    assert fa_p100_hf.make_cache(model.bfloat16(), 1, 10).paged.k.dtype == torch.bfloat16
    ids = torch.zeros(3, 8, dtype=torch.long)
    # the guard lets this cache through (the operators then refuse CPU tensors) and no other
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        model(ids, past_key_values=cache, use_cache=True)
    with pytest.raises(NotImplementedError, match="KV cache"):
        model(ids, use_cache=True)
    with pytest.raises(NotImplementedError, match="padding mask"):
        model(ids, past_key_values=cache, use_cache=True, attention_mask=torch.tensor([[0] + [1] * 7] * 3))
    with pytest.raises(NotImplementedError, match="in place"):
        cache.reorder_cache(torch.tensor([0, 0, 1]))
    with pytest.raises(RuntimeError, match="batch of 3"):
        cache.update(torch.zeros(2, 1, 4, 64), torch.zeros(2, 1, 4, 64), 0)
    with pytest.raises(RuntimeError, match="do not fit"):
        cache.update(torch.zeros(3, 1, 129, 64), torch.zeros(3, 1, 129, 64), 0)


def test_hf_attention_refuses_a_second_prompt():
    import fa_p100_hf

    class Layer:
        is_causal = True

    k = torch.zeros(1, 2, 8, 64, dtype=torch.float16)
    k._fa_p100_paged = (None, 5)
    with pytest.raises(NotImplementedError, match="one token at a time"):
        fa_p100_hf.fa_p100_attention_forward(Layer(), torch.zeros(1, 4, 8, 64).half(), k, k, None)
