"""Build libzimage_b200.so (sm_100a) in-tree with nvcc, and _ops.so, torch functions over its C ABI.

    python comfyui-zimage-triton_b200/csrc/build.py [--force] [--verbose]

Objects go to csrc/_build/, the shared libraries to zimage_b200/.  Rebuilds only when a source or
header is newer than a library.
"""

from __future__ import annotations

import argparse
import os
import shutil
import subprocess
import sys
from pathlib import Path

CSRC = Path(__file__).resolve().parent
PKG = CSRC.parent / "zimage_b200"
INCLUDE = CSRC.parent.parent / "include"
OUT = PKG / "libzimage_b200.so"
OPS = PKG / "_ops.so"
SOURCES = ["zib_api.cu", "rowops.cu", "gemm_w8a8.cu", "rotary.cu", "group_norm.cu", "fp8_block.cu",
           "fp8_gemm.cu", "fp8_linear.cu"]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-fvisibility=hidden",
         "--expt-relaxed-constexpr", "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found")


def _older(out: Path, deps: list[Path]) -> bool:
    return not out.exists() or any(p.stat().st_mtime > out.stat().st_mtime for p in deps)


def _stale() -> bool:
    return _older(OUT, [CSRC / s for s in SOURCES] + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h")))


def build_ops(force: bool = False, verbose: bool = False) -> Path:
    """The torch functions (for the running interpreter and its torch), linked against the library."""
    src = CSRC / "torch_ops.cpp"
    if not force and not _older(OPS, [src, *INCLUDE.glob("*.h")]):
        return OPS
    import sysconfig

    import torch  # its C++ runtime is the system's shared one: the system compiler links against that
    from torch.utils import cpp_extension

    inc = cpp_extension.include_paths("cuda") + [sysconfig.get_paths()["include"]]
    lib = cpp_extension.library_paths("cuda")
    gxx = next(c for c in ("/usr/bin/g++", shutil.which("g++") or "g++") if Path(c).exists() or c == "g++")
    tmp = OPS.with_suffix(".so.tmp")
    cmd = [gxx, "-O2", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", *(f"-I{p}" for p in inc), str(src),
           "-o", str(tmp), *(f"-L{p}" for p in lib), "-lc10", "-ltorch_cpu", "-ltorch", "-ltorch_python", "-lc10_cuda",
           f"-L{PKG}", "-l:libzimage_b200.so", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, OPS)
    return OPS


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or _stale():
        _build_library(verbose)
    build_ops(force, verbose)
    return OUT


def _build_library(verbose: bool) -> None:
    bdir = CSRC / "_build"
    bdir.mkdir(exist_ok=True)
    objs = []
    running = []
    for s in SOURCES:  # at once: each takes one core for seconds to a minute
        o = bdir / (Path(s).stem + ".o")
        cmd = [nvcc(), *ARCH, *FLAGS, "-I", str(INCLUDE), "-c", str(CSRC / s), "-o", str(o)]
        if verbose:
            cmd += ["-Xptxas", "-v"]
            print(" ".join(cmd), flush=True)
        running.append((cmd, subprocess.Popen(cmd)))
        objs.append(str(o))
    codes = [p.wait() for _, p in running]
    for (cmd, _), rc in zip(running, codes):
        if rc:
            raise subprocess.CalledProcessError(rc, cmd)
    tmp = OUT.with_suffix(".so.tmp")
    cmd = [nvcc(), *ARCH, "-shared", "-o", str(tmp), *objs, "-lcudart_static",
           "-Xcompiler", "-fPIC"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, OUT)


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(a.force, a.verbose))
    sys.exit(0)
