"""In-tree build of libmegamoe.so for sm_100a (nvcc cross-compiles without a GPU), and
of _dense.so, the dense operators' calls on torch tensors (host code over the C ABI).

Each translation unit compiles to its own object (in parallel), then one link:
mm_gate_dsv41.cu takes the DeepSeek-V4.1 gate's floating-point flags
(flush-to-zero, approximate square root and division, the reference's NVRTC
options for that gate), every other file the default IEEE ones.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.dirname(HERE)
REPO = os.path.dirname(PKG)
CSRC = os.path.join(PKG, "csrc")
SOURCES = ["mm_api.cu", "mm_route.cu", "mm_gate_dsv41.cu", "mm_experts.cu", "mm_finalize.cu", "mm_comm.cu", "mm_norm.cu",
           "mm_int8.cu"]
HEADERS = ["mm_dense.cuh", "mm_gate.cuh", "mm_kernels.cuh", "mm_layout.cuh", "mm_numerics.cuh", "mm_ptx.cuh"]
TORCH_SOURCE = "mm_dense_torch.cpp"
OUTPUT = os.path.join(HERE, "libmegamoe.so")
TORCH_OUTPUT = os.path.join(HERE, "_dense.so")
OBJDIR = os.path.join(HERE, "_build")
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
CXX = os.environ.get("CXX", "g++")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
COMPILE = [*ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC"]
# per-file floating-point flags (the DeepSeek-V4.1 gate's, routed_expert_gemm.py:213-220)
FILE_FLAGS = {"mm_gate_dsv41.cu": ["-ftz=true", "-prec-sqrt=false", "-prec-div=false"]}


def compile_flags(source: str) -> list:
    """nvcc flags of one translation unit (without -c / -o)."""
    return [*COMPILE, *FILE_FLAGS.get(source, []), "-I", os.path.join(REPO, "include"), "-I", CSRC]


def _torch_headers() -> dict:
    """The include folders of _dense.so: a header that each has to hold, and where."""
    import sysconfig

    import torch

    include = os.path.join(os.path.dirname(torch.__file__), "include")
    return {"Python.h": sysconfig.get_paths()["include"], "torch/csrc/Dtype.h": include,
            "torch/torch.h": os.path.join(include, "torch", "csrc", "api", "include"),
            "cuda_runtime_api.h": os.path.join(os.path.dirname(os.path.dirname(NVCC)), "include")}


def torch_command() -> list:
    """g++ command that builds _dense.so against the running Python and torch."""
    import torch

    root = os.path.dirname(torch.__file__)
    lib = os.path.join(root, "lib")
    abi = int(torch.compiled_with_cxx11_abi())
    includes = [os.path.join(REPO, "include"), *_torch_headers().values()]
    return [CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={abi}", *(f"-I{i}" for i in includes),
            os.path.join(CSRC, TORCH_SOURCE), "-o", TORCH_OUTPUT, f"-L{HERE}", "-l:libmegamoe.so", "-Wl,-rpath,$ORIGIN",
            f"-L{lib}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda",
            f"-Wl,-rpath,{lib}",
            # the C++ runtime that torch runs on: a toolchain with a static one alone would put
            # a second copy, and a second set of stream locales, beside it
            "-nostdlib++", "-l:libstdc++.so.6"]


def _older(output: str, deps) -> bool:
    return not os.path.exists(output) or any(os.path.getmtime(p) > os.path.getmtime(output) for p in deps)


def _own() -> list:
    return [os.path.join(REPO, "include", "megamoe.h"), os.path.abspath(__file__)]


def _stale() -> bool:
    return _older(OUTPUT, [os.path.join(CSRC, f) for f in SOURCES + HEADERS] + _own())


def _torch_abi() -> str:
    """What _dense.so is compiled against: it loads beside no other."""
    import sysconfig

    import torch

    return f"{sysconfig.get_config_var('SOABI')} torch {torch.__version__} {torch.__file__} cxx11 {int(torch.compiled_with_cxx11_abi())}"


def _torch_stamp() -> str:
    return os.path.join(OBJDIR, "_dense.abi")


def _torch_stale() -> bool:
    if _older(TORCH_OUTPUT, [os.path.join(CSRC, TORCH_SOURCE)] + _own()):
        return True
    try:
        with open(_torch_stamp()) as f:
            return f.read() != _torch_abi()
    except OSError:
        return True


def _run(cmd, verbose):
    res = subprocess.run(cmd, capture_output=True, text=True)
    if verbose:
        sys.stderr.write(res.stderr)
    return res


def build(force: bool = False, verbose: bool = False) -> str:
    """Compile the library, and the binding of the dense operators, where a source is newer
    than they are (the binding: or where torch or Python is another); returns the library's path."""
    if force or _stale():
        _build_library(verbose)
    if force or _torch_stale():
        _build_binding(verbose)
    return OUTPUT


def _build_library(verbose: bool) -> None:
    os.makedirs(OBJDIR, exist_ok=True)
    objs = [os.path.join(OBJDIR, s.replace(".cu", ".o")) for s in SOURCES]
    cmds = [[NVCC, *compile_flags(s), *(["-Xptxas", "-v"] if verbose else []), "-c", os.path.join(CSRC, s), "-o", o]
            for s, o in zip(SOURCES, objs)]
    with ThreadPoolExecutor(max_workers=len(cmds)) as pool:
        results = list(pool.map(lambda c: _run(c, verbose), cmds))
    for cmd, res in zip(cmds, results):
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError(f"nvcc failed ({res.returncode}): {' '.join(cmd)}")
    link = [NVCC, *ARCH, "-shared", "-cudart", "static", "-o", OUTPUT, *objs]
    res = _run(link, verbose)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"nvcc link failed ({res.returncode}) building {OUTPUT}")


def _build_binding(verbose: bool) -> None:
    missing = [h for h, folder in _torch_headers().items() if not os.path.exists(os.path.join(folder, h))]
    missing += [] if shutil.which(CXX) else [CXX]
    if missing:
        # the library and its MoE chain need none of them; the dense operators' calls will say
        # that _dense.so is not there, so one built for something else must not be
        if os.path.exists(TORCH_OUTPUT):
            os.remove(TORCH_OUTPUT)
        sys.stderr.write(f"megamoe: _dense.so is left out, the dense operators cannot be called: no {', '.join(missing)} here\n")
        return
    cmd = torch_command()
    res = _run(cmd, verbose)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError(f"g++ failed ({res.returncode}): {' '.join(cmd)}")
    os.makedirs(OBJDIR, exist_ok=True)
    with open(_torch_stamp(), "w") as f:
        f.write(_torch_abi())


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
