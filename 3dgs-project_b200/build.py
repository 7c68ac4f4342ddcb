"""Builds libsplat_b200.so (all csrc/*.cu for sm_100a, nvcc) and _tensors.so (csrc/tensor_list.cpp, g++) in place.
The first needs the CUDA toolkit only; the second is passed over where torch or Python's headers are absent.

    python 3dgs-project_b200/build.py [--force] [--verbose]

Objects go to csrc/_build/ (git-ignored); the shared libraries land next to this file so they travel
with the source tree. A rebuild happens only when a source, header or flag changed.
"""
from __future__ import annotations

import argparse
import concurrent.futures as cf
import hashlib
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = CSRC / "_build"
LIB = PKG / "libsplat_b200.so"
TENSORS = PKG / "_tensors.so"

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "-Xcompiler", "-fPIC", "-Xcompiler", "-O3",
              "-Xptxas", "-warn-spills", f"-I{INCLUDE}", f"-I{CSRC}"]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(path).exists():
        raise RuntimeError("nvcc not found: libsplat_b200.so cannot be built")
    return path


def _digest(sources: list[Path]) -> str:
    h = hashlib.sha256()
    for p in sorted(sources + list(CSRC.glob("*.cuh")) + list(INCLUDE.glob("*.h"))):
        h.update(p.name.encode())
        h.update(p.read_bytes())
    h.update(" ".join(ARCH + NVCC_FLAGS).encode())
    return h.hexdigest()


def python_header() -> Path:
    return Path(sysconfig.get_paths()["include"]) / "Python.h"


def build_tensors(force: bool = False, verbose: bool = False) -> Path | None:
    """The host-only module that reads lists of torch tensors: g++ against this interpreter's and torch's headers. None
    where these are absent: the Python package cannot be used there (its calls on lists say so), the C ABI can."""
    torch = importlib.util.find_spec("torch")
    absent = "torch" if torch is None else "Python.h" if not python_header().exists() else None
    if absent:
        print(f"{TENSORS.name} is not built: {absent} is absent", file=sys.stderr)
        return None
    torch_dir = Path(torch.submodule_search_locations[0])
    src = CSRC / "tensor_list.cpp"
    cmd = ["g++", "-O3", "-std=c++17", "-fPIC", "-shared", str(src), f"-I{torch_dir / 'include'}",
           f"-I{torch_dir / 'include/torch/csrc/api/include'}", f"-I{python_header().parent}",
           f"-I{Path(nvcc()).resolve().parent.parent / 'include'}", f"-L{torch_dir / 'lib'}", "-lc10", "-lc10_cuda",
           "-ltorch_cpu", "-ltorch_python"]
    version = (torch_dir / "version.py").read_bytes()
    header = (INCLUDE / "splat_b200.h").read_bytes()
    digest = hashlib.sha256(src.read_bytes() + header + version + " ".join([sys.version, *cmd]).encode()).hexdigest()
    stamp = BUILD / "stamp_tensors"
    if not force and TENSORS.exists() and stamp.exists() and stamp.read_text() == digest:
        return TENSORS
    BUILD.mkdir(parents=True, exist_ok=True)
    tmp = TENSORS.with_suffix(".so.tmp")
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run([*cmd, "-o", str(tmp)], capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {src.name}:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, TENSORS)
    stamp.write_text(digest)
    return TENSORS


def build(force: bool = False, verbose: bool = False) -> Path:
    lib = build_library(force, verbose)
    build_tensors(force, verbose)
    return lib


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """The C ABI library."""
    sources = sorted(CSRC.glob("*.cu"))
    stamp = BUILD / "stamp"
    digest = _digest(sources)
    if not force and LIB.exists() and stamp.exists() and stamp.read_text() == digest:
        return LIB
    BUILD.mkdir(parents=True, exist_ok=True)
    cc = nvcc()

    def compile_one(src: Path) -> Path:
        obj = BUILD / (src.stem + ".o")
        cmd = [cc, *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr, flush=True)
        return obj

    with cf.ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 2)) as ex:
        objs = list(ex.map(compile_one, sources))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [cc, *ARCH, "-shared", "-o", str(tmp), *map(str, objs)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    stamp.write_text(digest)
    return LIB


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--verbose", action="store_true")
    a = ap.parse_args()
    print(build(force=a.force, verbose=a.verbose))
    return 0


if __name__ == "__main__":
    sys.exit(main())
