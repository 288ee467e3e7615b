"""Builds the sm_100a shared library libfa_b200.so in this directory.

The reference JIT-compiles its extension with torch.utils.cpp_extension.load
on first import (fa_p100.py:21-28, -arch=sm_60). Here the library is a plain
C-ABI shared object compiled by nvcc for sm_100a only, built in-tree so it
travels with the source tree; `build()` is idempotent and skips the compile
when the library is newer than every source file.
"""
import hashlib
import os
import shutil
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
INCLUDE = os.path.join(ROOT, "include")
LIB_PATH = os.path.join(HERE, "libfa_b200.so")
# The checked build: every TMA copy tests its coordinates and shared-memory
# alignment first (-DFAB_CHECK_TMA, fa_b200_debug_tma_check). Selected at load
# time by FA_B200_DEBUG=1; the release library is the default.
DEBUG_LIB_PATH = os.path.join(HERE, "libfa_b200_debug.so")

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    # nvcc compresses device code of this size (12 MB to 4), and the first call of every
    # process unpacks it: 17 ms against 12
    "--no-compress",
    "-Xcompiler", "-fPIC", "-shared",
]


def _sources():
    out = []
    for d in (CSRC, INCLUDE):
        for name in sorted(os.listdir(d)):
            if name.endswith((".cu", ".cuh", ".h")):
                out.append(os.path.join(d, name))
    return out


def _nvcc():
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and os.path.exists(cand):
            return cand
    raise RuntimeError("nvcc not found: cannot build libfa_b200.so")


def checked_requested():
    """Whether FA_B200_DEBUG=1 asks for the checked library."""
    return os.environ.get("FA_B200_DEBUG", "0") == "1"


def lib_path(checked=None):
    if checked is None:
        checked = checked_requested()
    return DEBUG_LIB_PATH if checked else LIB_PATH


def up_to_date(checked=None):
    path = lib_path(checked)
    if not os.path.exists(path):
        return False
    lib_mtime = os.path.getmtime(path)
    return all(os.path.getmtime(s) <= lib_mtime for s in _sources())


def build(force=False, verbose=False, checked=None):
    """Compile csrc/fa_b200.cu into libfa_b200.so, or with checked (default:
    FA_B200_DEBUG=1) into libfa_b200_debug.so with -DFAB_CHECK_TMA (sm_100a
    either way). Returns the library's path."""
    if checked is None:
        checked = checked_requested()
    path = lib_path(checked)
    if not force and up_to_date(checked):
        return path
    tmp = path + ".tmp"
    cmd = [_nvcc(), *NVCC_FLAGS, *(["-DFAB_CHECK_TMA"] if checked else []), "-o", tmp,
           os.path.join(CSRC, "fa_b200.cu")]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"nvcc failed building {os.path.basename(path)}:\n" + res.stdout + res.stderr)
    if verbose:
        print(res.stdout + res.stderr)
    os.replace(tmp, path)
    return path


# The paged operators' torch module (csrc/fa_paged_py.cpp), built against the
# installed torch by the host compiler.
BINDING_SOURCE = os.path.join(CSRC, "fa_paged_py.cpp")
BINDING_PATH = os.path.join(HERE, "_fa_paged.so")


def _binding_flags():
    import torch
    return ["-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}"]


def binding_key():
    """What the module is compiled against: it uses torch's and Python's class layouts,
    so it serves the torch, the interpreter and the flags it was built with alone."""
    import sysconfig

    import torch
    parts = [torch.__version__, str(torch.version.git_version), str(sysconfig.get_config_var("EXT_SUFFIX")),
             *_binding_flags()]
    return "fa_paged-" + hashlib.sha256("\0".join(parts).encode()).hexdigest()


def binding_up_to_date():
    """Newer than its sources, and of this binding_key(), which the module holds: read
    from the file, as a module of another torch must not be loaded to ask it."""
    if not os.path.exists(BINDING_PATH):
        return False
    built = os.path.getmtime(BINDING_PATH)
    if any(os.path.getmtime(s) > built for s in (BINDING_SOURCE, os.path.join(INCLUDE, "fa_b200.h"))):
        return False
    with open(BINDING_PATH, "rb") as f:
        return binding_key().encode() in f.read()


def build_binding(force=False):
    """Compile csrc/fa_paged_py.cpp into _fa_paged.so, a CPython module over the
    installed torch. Returns its path."""
    if not force and binding_up_to_date():
        return BINDING_PATH
    import sysconfig

    import torch
    home = os.path.dirname(torch.__file__)
    cuda = os.path.dirname(os.path.dirname(_nvcc()))
    tmp = f"{BINDING_PATH}.{os.getpid()}.tmp"
    cmd = [os.environ.get("CXX") or shutil.which("g++") or "g++", *_binding_flags(),
           f'-DFA_PAGED_KEY="{binding_key()}"',
           f"-I{home}/include", f"-I{home}/include/torch/csrc/api/include",
           f"-I{sysconfig.get_path('include')}", f"-I{cuda}/include", BINDING_SOURCE, "-o", tmp,
           f"-L{home}/lib", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-ltorch_python"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError("g++ failed building _fa_paged.so:\n" + res.stdout + res.stderr)
    os.replace(tmp, BINDING_PATH)
    return BINDING_PATH


if __name__ == "__main__":
    print(build(force=True, verbose=True))
    print(build_binding(force=True))
