"""In-tree build of the C-ABI library ``libflash_muon_b200.so`` for sm_100a and of ``_host``, the
Python extension that turns lists of tensors into the library's arrays.

``python flash_muon_b200/build.py`` compiles every ``csrc/*.cu`` with nvcc and links one shared
object next to this file, then ``csrc/host.cpp`` with g++ against the installed torch.  No GPU is
needed to build (nvcc cross-compiles).
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libflash_muon_b200.so"
HOST_PATH = PKG_DIR / ("_host" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
BUILD_DIR = PKG_DIR / "build"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-std=c++17", "-lineinfo",
    "-Xcompiler", "-fPIC",
    "-Xptxas", "-v",
]


def _nvcc() -> str:
    cand = os.environ.get("NVCC") or shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(cand).exists():
        raise RuntimeError("nvcc not found; set NVCC or put it on PATH")
    return cand


def _stale(target: Path, sources: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(s.stat().st_mtime > t for s in sources)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile what is out of date and return the path of the shared library."""
    nvcc = _nvcc()
    BUILD_DIR.mkdir(exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted((PKG_DIR.parent / "include").glob("*.h"))
    objs = []
    for src in sorted(CSRC.glob("*.cu")):
        obj = BUILD_DIR / (src.stem + ".o")
        objs.append(obj)
        if force or _stale(obj, [src] + headers):
            cmd = [nvcc, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            res = subprocess.run(cmd, capture_output=True, text=True)
            (BUILD_DIR / (src.stem + ".ptxas.log")).write_text(res.stderr)
            if verbose or res.returncode != 0:
                sys.stderr.write(res.stdout + res.stderr)
            if res.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}")
    if force or _stale(LIB_PATH, objs):
        cmd = [nvcc, "-shared", "-gencode", "arch=compute_100a,code=sm_100a", "-o", str(LIB_PATH),
               *map(str, objs), "-cudart", "static"]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            sys.stderr.write(res.stdout + res.stderr)
            raise RuntimeError("link failed")
    _build_host(headers, force)
    return LIB_PATH


def _build_host(headers: list[Path], force: bool) -> None:
    import torch
    root = Path(torch.__file__).resolve().parent
    src, libs = CSRC / "host.cpp", root / "lib"
    # a torch installed after the last build makes it stale too
    if not (force or _stale(HOST_PATH, [src, libs / "libtorch_python.so", *[h for h in headers if h.suffix == ".h"]])):
        return
    cuda = Path(_nvcc()).resolve().parent.parent / "include"
    cmd = [os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-isystem", str(root / "include"), "-isystem", str(root / "include" / "torch" / "csrc" / "api" / "include"),
           "-isystem", str(cuda), "-isystem", sysconfig.get_path("include"), str(src), "-o", str(HOST_PATH),
           f"-L{libs}", "-ltorch_python", "-ltorch_cpu", "-lc10", "-lc10_cuda", f"-Wl,-rpath,{libs}"]
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        sys.stderr.write(res.stdout + res.stderr)
        raise RuntimeError("g++ failed on host.cpp")


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
