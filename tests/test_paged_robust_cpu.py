"""The paged cache's sizes and refusals that need no GPU, beside test_paged_cpu.py."""
import os
import subprocess

import pytest

import _build


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
