"""The paged cache's sizes and refusals that need no GPU, beside test_paged_cpu.py."""
import os
import random
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import _build
import fa_p100_paged as paged


def compiles(tmp_path, code):
    """Whether a translation unit over the kernels' headers compiles."""
    src = tmp_path / "unit.cu"
    src.write_text(code)
    res = subprocess.run([_build._nvcc(), *_build.NVCC_FLAGS[:2], "-std=c++17", "-O0", f"-I{_build.CSRC}", "-c",
                          str(src), "-o", os.devnull], capture_output=True, text=True)
    return res.returncode == 0, res.stderr


@pytest.mark.parametrize("warps", [4, 4 + 2, 8 + 2])
def test_the_line_has_a_sum_per_warp(tmp_path, warps):
    """The blocks that walk the line: paged_attn_kernel's and the two of
    paged_wide_kernel, whose softmax warps have two more beside them."""
    ok, err = compiles(tmp_path, f"""
#include <cuda.h>
#include "fa_paged_wide.cuh"
static_assert(sizeof(fab::LineShared::sums) / sizeof(long long) >= {warps}, "fewer sums than warps");
""")
    assert ok, err


def test_the_join_follows_no_record_that_was_not_written(tmp_path):
    """A block that gave up a wait has written no record: whatever the workspace holds
    there must name a unit of the call and blocks of its launch, or be passed over."""
    int_max, int_min = 2 ** 31 - 1, -2 ** 31
    units, blocks = 12, 7
    good = [(0, 0, 0), (11, 0, 6), (5, 6, 6)]
    bad = [(-1, 0, 0), (12, 0, 0), (int_max, 0, 0), (int_min, 0, 0), (3, -1, 2), (3, int_min, 2), (3, 5, 4),
           (3, 0, 7), (3, 0, int_max), (3, int_max, int_min)]
    checks = [f"static_assert({'' if r in good else '!'}fab::record_in_range({r[0]}ll, {r[1]}ll, {r[2]}ll, "
              f"{units}, {blocks}));" for r in good + bad]
    ok, err = compiles(tmp_path, "#include <cuda.h>\n#include \"fa_paged.cuh\"\n" + "\n".join(checks))
    assert ok, err
    # the kernel asks before it uses one
    body = open(os.path.join(_build.CSRC, "fa_paged.cuh")).read().split("paged_join_kernel(const", 1)[1]
    assert body.index("record_in_range(record.x, record.y, record.z") < body.index("record.x %")


def half(*shape):
    return torch.randn(*shape).half()


def append_args():
    return dict(k=half(5, 2, 64), v=half(5, 2, 64), slots=torch.zeros(5, dtype=torch.int32), k_cache=half(4, 2, 16, 64),
                v_cache=half(4, 2, 16, 64))


def attn_args():
    return dict(q=half(3, 4, 64), k_cache=half(4, 2, 16, 64), v_cache=half(4, 2, 16, 64),
                block_table=torch.zeros(3, 5, dtype=torch.int32), lens=torch.zeros(3, dtype=torch.int32))


@pytest.mark.parametrize("op,args,name", [
    (paged.paged_append, append_args, n) for n in ("k", "v", "k_cache", "v_cache")] + [
    (paged.paged_attn, attn_args, n) for n in ("q", "k_cache", "v_cache")])
@pytest.mark.parametrize("no_grad", [False, True])
def test_a_forward_mode_tangent_is_refused(op, args, name, no_grad):
    a = args()
    with fwAD.dual_level(), torch.set_grad_enabled(not no_grad):
        a[name] = fwAD.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(RuntimeError, match=f"{name} carries a tangent"):
            op(**a)
        a[name] = fwAD.unpack_dual(a[name]).primal     # as any other CPU tensor then
        with pytest.raises(RuntimeError, match="CUDA"):
            op(**a)


@pytest.mark.parametrize("op,args,name", [(paged.paged_append, append_args, "k"), (paged.paged_attn, attn_args, "q")])
def test_transformed_and_fake_tensors_are_refused(op, args, name):
    """torch.func's wrappers and fake tensors hold no memory to pass to a kernel."""
    a = args()

    def call(x):
        op(**{**a, name: x})
        return x

    x = a[name]
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(x[None])
    with FakeTensorMode() as mode:
        b = {n: mode.from_tensor(t) for n, t in a.items()}
        with pytest.raises(RuntimeError):
            op(**b)


def slices(name):
    """Two caches of (4, 2, 16, 64) out of one buffer, and whether they share memory."""
    shape = (4, 2, 16, 64)
    b = torch.zeros(1 << 16, dtype=torch.float16)
    page = 2 * 16 * 64
    view = lambda at, *stride: b.as_strided(shape, stride, at)
    head = (page, 1024, 64, 1)
    return {
        "next to each other": ((view(0, *head), view(4 * page, *head)), False),
        "last page and first": ((view(0, *head), view(3 * page, *head)), True),
        "heads 0-1 and 1-2 of 5": ((view(0, 5120, 1024, 64, 1), view(1024, 5120, 1024, 64, 1)), True),
        "heads 0-1 and 2-3 of 4": ((view(0, 4096, 1024, 64, 1), view(2048, 4096, 1024, 64, 1)), False),
        "pages in turn": ((view(0, 2 * page, 1024, 64, 1), view(page, 2 * page, 1024, 64, 1)), False),
        "pages in turn, a row over": ((view(0, 2 * page, 1024, 64, 1), view(page - 64, 2 * page, 1024, 64, 1)), True),
        "by token, k and v in turn": ((view(0, 16 * 256, 64, 256, 1), view(128, 16 * 256, 64, 256, 1)), False),
        "by token, one head over": ((view(0, 16 * 192, 64, 192, 1), view(64, 16 * 192, 64, 192, 1)), True),
        "rows in turn": ((view(0, 2 * page, 2048, 128, 1), view(64, 2 * page, 2048, 128, 1)), False),
        "half a row": ((view(0, 2 * page, 2048, 128, 1), view(32, 2 * page, 2048, 128, 1)), True),
        "page's first 8 bytes": ((view(0, *head), view(4 * page - 8, *head)), True),
        "two layouts apart": ((view(0, *head), view(4 * page, page, 64, 128, 1)), False),
        "two layouts over": ((view(0, *head), view(3 * page + 1024, page, 64, 128, 1)), True),
        "two layouts in turn": ((view(0, 2 * page, 1024, 64, 1), view(page, 2 * page, 64, 128, 1)), False),
    }[name]


@pytest.mark.parametrize("name", [
    "next to each other", "last page and first", "heads 0-1 and 1-2 of 5", "heads 0-1 and 2-3 of 4", "pages in turn",
    "pages in turn, a row over", "by token, k and v in turn", "by token, one head over", "rows in turn", "half a row",
    "page's first 8 bytes", "two layouts apart", "two layouts over", "two layouts in turn"])
def test_append_refuses_caches_that_share_memory(name):
    (k, v), shared = slices(name)
    # what the views really touch
    marks = torch.zeros(1 << 16, dtype=torch.int32)
    for x in (k, v):
        marks.as_strided(x.shape, x.stride(), x.storage_offset()).add_(1)
    assert bool((marks > 1).any()) == shared
    for a, b in ((k, v), (v, k)):
        with pytest.raises(RuntimeError, match="different memory" if shared else "CUDA"):
            paged.paged_append(**{**append_args(), "k_cache": a, "v_cache": b})


@pytest.mark.parametrize("name", ["k", "v", "slots"])
@pytest.mark.parametrize("cache", [0, 1])
def test_append_refuses_rows_inside_the_caches(name, cache):
    """k, v and slots in a cache's memory, in the gap between its pages, and behind it."""
    page = 2 * 16 * 64
    b = torch.zeros(10 * page, dtype=torch.float16)
    gaps = b.as_strided((4, 2, 16, 64), (2 * page, 1024, 64, 1))      # every other page
    for at, shared in ((0, True), (7 * page, False), (6 * page + 1024, True), (page, False), (page - 8, True),
                       (page + 1024, False), (2 * page - 8, True), (8 * page, False)):
        if name == "slots":
            x = b.view(torch.int32)[at // 2:][:5]
        else:
            x = b[at:][:5 * 128].view(5, 2, 64)
        a = append_args()
        a[name], a[("k_cache", "v_cache")[cache]] = x, gaps
        with pytest.raises(RuntimeError, match=f"{name} must not overlap" if shared else "CUDA"):
            paged.paged_append(**a)


def test_append_overlap_against_every_element():
    """Random layouts of one buffer: refused exactly where an element is in both."""
    rng = random.Random(0)
    n = 0
    for _ in range(300):
        def layout():
            axes = [(4, None), (2, None), (16, None)]
            order = rng.sample(range(3), 3)
            stride, at = [0, 0, 0], 64 + 8 * rng.randrange(3)
            for i in order:
                stride[i] = at * rng.choice([1, 1, 2])
                at = stride[i] * axes[i][0] + 8 * rng.randrange(2)
            return (*stride, 1)
        sk = layout()
        sv = sk if rng.random() < 0.7 else layout()
        off = rng.choice([64, 72, 1024, 2048, sk[0], sk[1], sk[2], sk[1] // 2 // 8 * 8, 4 * sk[0], 8 * rng.randrange(900)])
        b = torch.zeros(off + 4 * max(sk[0], sk[1], sk[2], sv[0], sv[1], sv[2]) * 16, dtype=torch.float16)
        k, v = (b.as_strided((4, 2, 16, 64), s, o) for s, o in ((sk, 0), (sv, off)))
        marks = torch.zeros(b.numel(), dtype=torch.bool)
        marks.as_strided(k.shape, k.stride(), 0).fill_(True)
        shared = bool(marks.as_strided(v.shape, v.stride(), off).any())
        with pytest.raises(RuntimeError) as e:
            paged.paged_append(**{**append_args(), "k_cache": k, "v_cache": v})
        assert ("different memory" in str(e.value)) == shared, (sk, sv, off)
        n += shared
    assert 0 < n < 300     # both kinds were among them


def test_the_native_module_is_kept_for_its_torch_alone(monkeypatch, tmp_path):
    """_fa_paged.so uses torch's class layouts: another torch, interpreter or flags mean
    another module."""
    import sysconfig
    import _fa_paged
    _build.build_binding()
    assert _build.binding_up_to_date() and _fa_paged.build_key == _build.binding_key()
    for target, name, value in ((torch, "__version__", "2.12.0"), (torch.version, "git_version", "0" * 40),
                                (sysconfig, "get_config_var", lambda n: ".cpython-313-x86_64-linux-gnu.so"),
                                (torch, "compiled_with_cxx11_abi", lambda: not ABI)):
        with monkeypatch.context() as m:
            m.setattr(target, name, value)
            assert not _build.binding_up_to_date(), name
    with monkeypatch.context() as m:     # asking needs no compiler
        m.setattr(_build, "_nvcc", lambda: 1 / 0)
        m.setenv("CXX", "/nowhere/c++")
        assert _build.build_binding() == _build.BINDING_PATH
    # a file cut short, newer than every source
    cut = tmp_path / "_fa_paged.so"
    cut.write_bytes(b"\x7fELF")
    with monkeypatch.context() as m:
        m.setattr(_build, "BINDING_PATH", str(cut))
        assert not _build.binding_up_to_date()
    assert _build.binding_up_to_date()


ABI = torch.compiled_with_cxx11_abi()


# ---- the HuggingFace cache, its operators recorded and not run ----
def hf_model(layers=2, impl="fa_p100"):
    import fa_p100_hf
    from transformers import Qwen3Config, Qwen3ForCausalLM
    cfg = Qwen3Config(vocab_size=64, hidden_size=128, intermediate_size=256, num_hidden_layers=layers,
                      num_attention_heads=2, num_key_value_heads=1, head_dim=64, max_position_embeddings=64,
                      tie_word_embeddings=True, attn_implementation="sdpa")
    torch.manual_seed(0)
    m = Qwen3ForCausalLM(cfg).eval()
    return fa_p100_hf.enable_fa_p100(m) if impl == "fa_p100" else m


def hf_cache(model, monkeypatch, batch=1, max_len=48):
    """A cache whose calls of the GPU operators are listed, with attention in torch's own."""
    import fa_p100_hf
    cache, calls = fa_p100_hf.make_cache(model, batch, max_len), []
    for name in ("extend", "append", "release", "attn"):
        monkeypatch.setattr(cache.paged, name, lambda *a, name=name: (calls.append(name), a[-1])[1])
    monkeypatch.setattr(fa_p100_hf, "_warned_cast", True)     # other tests look for the one warning
    monkeypatch.setattr(fa_p100_hf, "flash_attn_bnhd", lambda q, k, v, causal, full_precision:
                        torch.nn.functional.scaled_dot_product_attention(
                            q, k, v, is_causal=causal, enable_gqa=True).transpose(1, 2))
    return cache, calls


def ids(n):
    return torch.arange(n)[None]


def test_hf_cache_refuses_a_second_prompt_unchanged(monkeypatch):
    """The refusal comes before the prompt's keys are stored: the cache goes on as it was."""
    model = hf_model()
    cache, calls = hf_cache(model, monkeypatch)
    with torch.no_grad():
        model(ids(5), past_key_values=cache, use_cache=True)
        assert calls == ["extend", "append", "append"] and cache.get_seq_length() == 5
        with pytest.raises(NotImplementedError, match="one token at a time"):
            model(ids(3), past_key_values=cache, use_cache=True)
        assert calls == ["extend", "append", "append"] and cache.tokens == 5 and cache.get_seq_length() == 5
        model(ids(1), past_key_values=cache, use_cache=True)
    assert calls[3:] == ["extend", "append", "attn", "append", "attn"] and cache.get_seq_length() == 6


def test_hf_cache_refuses_another_attention(monkeypatch):
    """The cache hands on the new keys alone, which only the fa_p100 attention can
    complete: under sdpa a decoding step would see one token, without a word."""
    model = hf_model(impl="sdpa")
    cache, calls = hf_cache(model, monkeypatch)
    with torch.no_grad(), pytest.raises(RuntimeError, match="enable_fa_p100"):
        model(ids(5), past_key_values=cache, use_cache=True)
    assert calls == ["extend", "append"]
    cache.reset()
    model = hf_model(layers=1, impl="sdpa")     # one layer: the second call shows it
    cache, calls = hf_cache(model, monkeypatch)
    with torch.no_grad():
        model(ids(5), past_key_values=cache, use_cache=True)
        with pytest.raises(RuntimeError, match="enable_fa_p100"):
            model(ids(1), past_key_values=cache, use_cache=True)
    # reset, and a model that has it
    cache.reset()
    model = hf_model(layers=1)
    with torch.no_grad():
        for n in (5, 1, 1):
            model(ids(n), past_key_values=cache, use_cache=True)
    assert cache.get_seq_length() == 7
    # a call that the attention refuses does not count as lost
    with torch.no_grad(), pytest.raises(NotImplementedError, match="head_mask"):
        model(ids(1), past_key_values=cache, use_cache=True, head_mask=torch.ones(2))
    assert cache.handed is None


def test_no_cluster_is_larger_than_the_device_can_place(tmp_path):
    """One kv head or eight, short tables to long, on a whole B200 and on a context of
    fewer SMs, with and without room for clusters of 16."""
    checks = []
    for units in (1, 2, 8, 9, 18, 37, 74, 148, 296, 297):
        for most in (1, 2, 5, 16, 64, 128, 129, 1 << 20):
            for sms in (148, 74, 18, 8):
                for top in (16, 8):
                    checks.append(f"static_assert(sane(fab::paged_cluster({units}, {most}, {sms}, {top}), {units}, {most}, "
                                  f"{sms}, {top}));")
    ok, err = compiles(tmp_path, """
#include <cuda.h>
#include "fa_paged.cuh"
// none, or a power of two up to the top whose blocks are on the GPU at once
constexpr bool sane(int c, long long units, long long most, int sms, int top) {
  return c == 0 || (c > 0 && c <= top && (c & (c - 1)) == 0 && units * c <= (c == 16 ? sms : 2 * sms) && most <= 16ll * c);
}
static_assert(fab::paged_cluster(8, 64, 148, 16) == 16 && fab::paged_cluster(8, 64, 148, 8) == 0);
static_assert(fab::paged_cluster(8, 32, 148, 16) == 16 && fab::paged_cluster(8, 32, 148, 8) == 8);
""" + "\n".join(checks))
    assert ok, err


def test_the_library_is_not_unpacked_by_every_process():
    """Compressed device code is a third of the size and costs each first call."""
    assert "--no-compress" in _build.NVCC_FLAGS
