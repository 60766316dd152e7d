"""Build ``libr4q.so`` (all of csrc/*.cu) in-tree with nvcc for sm_100a, and the
Python module ``_r4q_torch`` (csrc/torch_ops.cpp) against the installed torch.

    python -m r4q.build        (from the rdna4-quant_b200 folder)

Objects go to ``_build/``; the shared library lands next to the Python
modules so that it travels with the source tree.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent.parent
CSRC = PKG / "csrc"
OUT = PKG / "libr4q.so"
TORCH_SRC = CSRC / "torch_ops.cpp"
TORCH_OUT = PKG / "_r4q_torch.so"
BUILD = PKG / "_build"
INCLUDE = PKG.parent / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
         f"-I{INCLUDE}", f"-I{CSRC}"]


def _nvcc() -> str:
    for c in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", "nvcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "nvcc"


def sources():
    return sorted(CSRC.glob("*.cu"))


def _stale(obj: Path, src: Path, headers) -> bool:
    if not obj.exists():
        return True
    t = obj.stat().st_mtime
    return src.stat().st_mtime > t or any(h.stat().st_mtime > t for h in headers)


def _torch_command(out: Path) -> list:
    """nvcc passes a .cpp file on to its host compiler, the one of the .cu files: one C++ runtime, the shared one
    that torch uses (a compiler that links its own copy statically breaks streams and exceptions across the two)."""
    import torch
    root = Path(torch.__file__).resolve().parent
    return [_nvcc(), "-O2", "-std=c++17", "-shared", "--cudart=none", "-Xcompiler", "-fPIC",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{root / 'include'}",
            f"-I{root / 'include/torch/csrc/api/include'}", f"-I{sysconfig.get_paths()['include']}", str(TORCH_SRC),
            "-o", str(out), f"-L{root / 'lib'}", "-ltorch_python", "-ltorch", "-ltorch_cpu", "-lc10", "-lc10_cuda",
            "-Xlinker", f"-rpath,{root / 'lib'}"]


def _torch_identity(command) -> str:
    """What the module is bound to besides its source: the torch and Python builds, and the command."""
    import torch
    return "\n".join([torch.__version__, str(torch.version.git_version), sys.version, *command])


def build(verbose: bool = False, force: bool = False) -> Path:
    BUILD.mkdir(exist_ok=True)
    headers = list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))
    nvcc = _nvcc()
    jobs = []
    objs = []
    for s in sources():
        o = BUILD / (s.stem + ".o")
        objs.append(o)
        if force or _stale(o, s, headers):
            jobs.append([nvcc, *ARCH, *FLAGS, "-c", str(s), "-o", str(o)])

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed: {' '.join(cmd)}\n{r.stdout}\n{r.stderr}")
        return r

    module = TORCH_OUT.with_suffix(".so.tmp")
    command, made_by = _torch_command(module), BUILD / "torch_ops.made_by"
    about = _torch_identity(command)
    stale_module = (force or _stale(TORCH_OUT, TORCH_SRC, [INCLUDE / "r4q.h"]) or not made_by.exists()
                    or made_by.read_text() != about)
    if stale_module:
        jobs.insert(0, command)                     # the longest first
    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 4)) as ex:
        list(ex.map(run, jobs))
    if stale_module:
        os.replace(module, TORCH_OUT)
        made_by.write_text(about)
        jobs.pop(0)
    if jobs or force or not OUT.exists() or any(o.stat().st_mtime > OUT.stat().st_mtime for o in objs):
        tmp = OUT.with_suffix(".so.tmp")
        run([nvcc, *ARCH, "-shared", "-o", str(tmp), *map(str, objs), "-lcudart"])
        os.replace(tmp, OUT)
    return OUT


if __name__ == "__main__":
    print(build(verbose="-v" in sys.argv, force="-f" in sys.argv))
