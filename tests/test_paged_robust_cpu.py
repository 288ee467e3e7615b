"""The paged cache's sizes and refusals that need no GPU, beside test_paged_cpu.py."""
import os
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
