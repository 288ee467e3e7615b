"""Generation through the HuggingFace backend with the paged cache: each cached
step's logits against the same model run over the whole sequence, and
model.generate end to end."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(impl, dev, dtype=torch.float32):
    from transformers import Qwen3Config, Qwen3ForCausalLM
    cfg = Qwen3Config(vocab_size=2048, hidden_size=256, intermediate_size=768,
                      num_hidden_layers=4, num_attention_heads=4, num_key_value_heads=2,
                      head_dim=64, max_position_embeddings=4096, initializer_range=0.02,
                      rope_parameters={"rope_theta": 1e6, "rope_type": "default"},
                      tie_word_embeddings=True, attn_implementation="sdpa" if impl == "fa_p100" else impl)
    torch.manual_seed(0)
    with torch.device(dev):
        m = Qwen3ForCausalLM(cfg).to(dtype)
    if impl == "fa_p100":
        import fa_p100_hf
        fa_p100_hf.enable_fa_p100(m)
    return m.eval()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
def test_cached_steps_match_the_whole_sequence(cuda, dtype):
    """The envelope of the uncached backend's logits test: the deviation of the
    cached steps from sdpa stays within 2x (mean) and 4x (p99.99) of eager's."""
    import fa_p100_hf
    B, N, steps = 3, 201, 12
    ids = torch.randint(0, 2048, (B, N + steps), generator=torch.Generator().manual_seed(1)).to(cuda)
    whole = {}
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        for impl in ("sdpa", "eager"):
            whole[impl] = _model(impl, cuda)(input_ids=ids, use_cache=False).logits.float()[:, N - 1:]
        m = _model("fa_p100", cuda)
        cache = fa_p100_hf.make_cache(m, B, N + steps, page_size=16, dtype=dtype)
        got = [m(input_ids=ids[:, :N], past_key_values=cache, use_cache=True).logits[:, -1:]]
        for t in range(N, N + steps):
            got.append(m(input_ids=ids[:, t:t + 1], past_key_values=cache, use_cache=True).logits)
    got = torch.cat(got, 1).float()
    assert cache.get_seq_length() == N + steps and cache.paged.lens.tolist() == [N + steps] * B
    dev_eager = (whole["eager"] - whole["sdpa"]).abs().flatten()
    dev_fa = (got - whole["sdpa"]).abs().flatten()
    assert dev_fa.mean() <= 2 * dev_eager.mean() + 1e-6
    assert torch.quantile(dev_fa, 0.9999) <= 4 * torch.quantile(dev_eager, 0.9999) + 1e-5


def test_generate_with_the_cache(cuda):
    """generate() with the cache gives the tokens of greedy steps over the whole
    sequence wherever the best token leads by more than rounding, and the cache
    serves another batch after reset()."""
    import fa_p100_hf
    m = _model("fa_p100", cuda, torch.bfloat16)
    cache = fa_p100_hf.make_cache(m, 2, 300)
    for seed in (0, 1):
        ids = torch.randint(0, 2048, (2, 60 + 7 * seed), generator=torch.Generator().manual_seed(seed)).to(cuda)
        with torch.no_grad():
            out = m.generate(ids, past_key_values=cache, use_cache=True, max_new_tokens=20, min_new_tokens=20,
                             do_sample=False, pad_token_id=0)
            assert out.shape == (2, ids.size(1) + 20) and torch.equal(out[:, :ids.size(1)], ids)
            logits = m(input_ids=out, use_cache=False).logits.float()[:, ids.size(1) - 1:-1]
        best = logits.max(-1).values
        taken = logits.gather(-1, out[:, ids.size(1):, None])[..., 0]
        # bf16 logits of about 1: a few roundings of 2^-8 either way
        assert (best - taken <= 0.1 * best.abs().clamp(min=1)).all()
        assert cache.get_seq_length() == ids.size(1) + 19
        cache.reset()
        assert cache.get_seq_length() == 0 and cache.paged.lens.tolist() == [0, 0]
        assert int(cache.paged.free_count) == cache.paged.free_pages.numel()


def test_cache_refuses_what_it_cannot_do(cuda):
    import fa_p100_hf
    m = _model("fa_p100", cuda, torch.bfloat16)
    cache = fa_p100_hf.make_cache(m, 1, 64)
    ids = torch.zeros(1, 10, dtype=torch.long, device=cuda)
    with torch.no_grad():
        m(ids, past_key_values=cache, use_cache=True)
        with pytest.raises(NotImplementedError, match="one token at a time"):
            m(ids, past_key_values=cache, use_cache=True)
    cache.reset()
    with pytest.raises(RuntimeError, match="backward"):
        m(ids, past_key_values=cache, use_cache=True)
    cache.reset()
    with torch.no_grad(), pytest.raises(RuntimeError, match="do not fit"):
        m(torch.zeros(1, 65, dtype=torch.long, device=cuda), past_key_values=cache, use_cache=True)
