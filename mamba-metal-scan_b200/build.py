"""Build libmms_scan.so (the sm_100a selective-scan library) in-tree.

    python mamba-metal-scan_b200/build.py [--force] [--verbose]

nvcc compiles csrc/*.cu for sm_100a only, file by file in parallel, and links
them into mamba_metal/lib/libmms_scan.so, next to the Python package that
loads it. Without --force, objects newer than their source and every header
are kept.
The library is plain C ABI (include/mms_scan.h); it links the CUDA runtime
statically so it loads without a matching libcudart on the library path.
"""
from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_ROOT = Path(__file__).resolve().parent
REPO_ROOT = PKG_ROOT.parent
CSRC = PKG_ROOT / "csrc"
INCLUDE = REPO_ROOT / "include"
LIB_DIR = PKG_ROOT / "mamba_metal" / "lib"
LIB = LIB_DIR / "libmms_scan.so"
OBJ_DIR = PKG_ROOT / "_build"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found (set NVCC or put /usr/local/cuda/bin on PATH)")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale() -> bool:
    if not LIB.exists():
        return True
    newest = max(p.stat().st_mtime for p in
                 list(CSRC.glob("*")) + list(INCLUDE.glob("*.h")) + [Path(__file__)])
    return LIB.stat().st_mtime < newest


def build(force: bool = False, verbose: bool = False) -> Path:
    if not force and not _stale():
        return LIB
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    flags = [nvcc_path(), *ARCH, "-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC",
             "-I", str(INCLUDE), "-I", str(CSRC)]
    if verbose:
        flags += ["-Xptxas", "-v"]
    headers = [p.stat().st_mtime for p in [*CSRC.glob("*.h"), *CSRC.glob("*.cuh"),
                                           *INCLUDE.glob("*.h"), Path(__file__)]]

    def compile_one(src: Path) -> Path:
        obj = OBJ_DIR / f"{src.stem}.o"
        if force or not obj.exists() or obj.stat().st_mtime < max([src.stat().st_mtime, *headers]):
            tmp = OBJ_DIR / f".{src.stem}.{os.getpid()}.o"
            cmd = [*flags, "-c", str(src), "-o", str(tmp)]
            if verbose:
                print(" ".join(cmd), flush=True)
            subprocess.run(cmd, check=True)
            os.replace(tmp, obj)
        return obj

    with ThreadPoolExecutor(max_workers=os.cpu_count() or 1) as pool:
        objects = list(pool.map(compile_one, sources()))
    tmp = LIB_DIR / f".libmms_scan.{os.getpid()}.so"
    subprocess.run([nvcc_path(), *ARCH, "-shared", "-cudart", "static",
                    *(str(o) for o in objects), "-o", str(tmp)], check=True)
    os.replace(tmp, LIB)
    return LIB


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="--verbose" in sys.argv))
