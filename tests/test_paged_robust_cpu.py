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
