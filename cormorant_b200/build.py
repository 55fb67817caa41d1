"""Build libcormorant_cuda.so (and its CPython binding _bind.*.so) in-tree for sm_100a (nvcc cross-compiles; no GPU needed).

    python -m cormorant_b200.build [--force] [--ptxas-info]
"""
from __future__ import annotations

import argparse
import os
import shlex
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
BUILD = PKG / "_build"
LIB = PKG / "libcormorant_cuda.so"
# The CPython side of the 8-bit floating-point entries (csrc/bind.c).  Its name carries the interpreter's
# ABI tag: another Python neither finds it nor takes it for its own.
BIND = PKG / ("_bind" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
INCLUDE = ROOT / "include"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ARCH + ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC,-O2",
                     "-I", str(INCLUDE), "-I", str(CSRC)]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or "/usr/local/cuda/bin/nvcc"
    return cand if Path(cand).exists() else "nvcc"


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build_binding(force: bool = False, quiet: bool = True) -> Path | None:
    """The CPython binding, or None (and a line on stderr) where Python's headers or a C compiler ($CC,
    else gcc) are missing: the library and its C users need neither, the 8-bit Python entries then
    raise ImportError."""
    src, include, cc = CSRC / "bind.c", Path(sysconfig.get_paths()["include"]), shlex.split(os.environ.get("CC") or "gcc")
    old = BIND.with_name("_bind.so")         # without a tag, which every Python would load
    if old != BIND:
        old.unlink(missing_ok=True)
    for what, there in ((include / "Python.h", (include / "Python.h").exists()), (cc[0], shutil.which(cc[0]))):
        if not there:
            print(f"{BIND.name} is not built: no {what}", file=sys.stderr)
            return None
    if force or _stale(BIND, [src, INCLUDE / "cormorant_cuda.h", Path(__file__)]):
        cmd = [*cc, "-O2", "-Wall", "-Wextra", "-Werror", "-std=gnu11", "-shared", "-fPIC", "-fvisibility=hidden",
               "-I", str(include), "-I", str(INCLUDE), "-o", str(BIND), str(src)]
        if not quiet:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
    return BIND


def build(force: bool = False, ptxas_info: bool = False, quiet: bool = True) -> Path:
    BUILD.mkdir(exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    objs = []
    for src in sorted(CSRC.glob("*.cu")):
        obj = BUILD / (src.stem + ".o")
        objs.append(obj)
        if force or ptxas_info or _stale(obj, [src, *headers, Path(__file__)]):
            cmd = [_nvcc(), *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if ptxas_info:
                cmd += ["-Xptxas", "-v"]
            if not quiet:
                print(" ".join(cmd), file=sys.stderr)
            subprocess.run(cmd, check=True)
    if force or _stale(LIB, objs):
        cmd = [_nvcc(), *ARCH, "-shared", "--cudart", "static", "-o", str(LIB), *map(str, objs), "-lrt", "-ldl", "-lpthread"]
        subprocess.run(cmd, check=True)
    build_binding(force, quiet)
    return LIB


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--ptxas-info", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, ptxas_info=a.ptxas_info, quiet=False))
