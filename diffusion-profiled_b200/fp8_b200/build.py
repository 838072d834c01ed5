"""Ahead-of-time build of the CUDA library ``libfp8ops.so`` (sm_100a only) and of the torch
operators over it, ``libfp8torch.so`` (csrc/torch_ops.cpp, host code).

The libraries are built in-tree next to this file so that they travel with the
source tree; nothing is JIT-compiled at import time.  ``python -m fp8_b200.build``
(with ``diffusion-profiled_b200`` on ``sys.path``) or ``build_library()`` runs nvcc.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
SRC_DIR = PKG_DIR.parent / "csrc"
INCLUDE_DIR = PKG_DIR.parent.parent / "include"
LIB_NAME = "libfp8ops.so"
LIB_PATH = PKG_DIR / LIB_NAME
TORCH_LIB_PATH = PKG_DIR / "libfp8torch.so"
TORCH_SRC = SRC_DIR / "torch_ops.cpp"
TORCH_MARK = "fp8_b200 operators for torch "
OBJ_DIR = PKG_DIR / "_build"

NVCC_FLAGS = [
    "-gencode",
    "arch=compute_100a,code=sm_100a",
    "-lineinfo",
    "-O3",
    "-std=c++17",
    "-Xcompiler",
    "-fPIC",
]


def _nvcc() -> str:
    cand = shutil.which("nvcc")
    if cand:
        return cand
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = os.path.join(cuda_home, "bin", "nvcc")
    if os.path.exists(path):
        return path
    raise RuntimeError("nvcc not found: set CUDA_HOME or put nvcc on PATH")


def sources() -> list[Path]:
    return sorted(SRC_DIR.glob("*.cu")) + [TORCH_SRC] + headers()


def headers() -> list[Path]:
    return sorted(SRC_DIR.glob("*.cuh")) + sorted(SRC_DIR.glob("*.h")) + [INCLUDE_DIR / "fp8ops.h"]


def torch_library_fits(torch_version: str, path: Path | None = None) -> bool:
    """Whether the library of torch operators is there and was built for this torch (it says so in a string of its own,
    TORCH_MARK and the version; torch's C++ interface changes from version to version)."""
    path = TORCH_LIB_PATH if path is None else path
    return path.exists() and (TORCH_MARK + torch_version).encode() + b"\0" in path.read_bytes()


def needs_rebuild() -> bool:
    import torch

    if not LIB_PATH.exists() or not torch_library_fits(torch.__version__):
        return True
    mtime = min(LIB_PATH.stat().st_mtime, TORCH_LIB_PATH.stat().st_mtime)
    return any(p.stat().st_mtime > mtime for p in sources())


def _compile(src: Path, obj: Path, verbose: bool) -> None:
    cmd = [_nvcc(), *NVCC_FLAGS, f"-I{INCLUDE_DIR}", "-c", "-o", str(obj), str(src)]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)


def _compile_torch_ops(obj: Path, verbose: bool) -> None:
    import torch
    from torch.utils.cpp_extension import include_paths

    cuda_include = Path(_nvcc()).resolve().parent.parent / "include"
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-c", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DFP8_TORCH_MARK="{TORCH_MARK}{torch.__version__}"', f"-I{INCLUDE_DIR}", *(f"-isystem{p}" for p in (*include_paths(), cuda_include)), "-o", str(obj), str(TORCH_SRC)]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)


def _link_torch_ops(obj: Path) -> None:
    import torch

    torch_lib = Path(torch.__file__).resolve().parent / "lib"
    tmp = TORCH_LIB_PATH.with_suffix(".so.tmp")
    subprocess.run(["g++", "-shared", "-o", str(tmp), str(obj), f"-L{torch_lib}", "-ltorch", "-ltorch_cpu", "-lc10",
                    "-lc10_cuda", f"-L{PKG_DIR}", f"-l:{LIB_NAME}", "-Wl,-rpath,$ORIGIN"], check=True)
    os.replace(tmp, TORCH_LIB_PATH)


def build_library(force: bool = False, verbose: bool = False) -> Path:
    """Compile every csrc/*.cu (side by side) and link libfp8ops.so for sm_100a; returns its path.

    An object file in ``_build/`` is kept while it is newer than its source and every header."""
    import torch

    if not force and not needs_rebuild():
        return LIB_PATH
    OBJ_DIR.mkdir(exist_ok=True)
    newest_header = max(p.stat().st_mtime for p in headers())
    jobs = []
    for src in sorted(SRC_DIR.glob("*.cu")):
        obj = OBJ_DIR / (src.stem + ".o")
        if force or not obj.exists() or obj.stat().st_mtime <= max(newest_header, src.stat().st_mtime):
            jobs.append((src, obj))
    torch_obj = OBJ_DIR / (TORCH_SRC.stem + ".o")
    torch_newest = max(TORCH_SRC.stat().st_mtime, (INCLUDE_DIR / "fp8ops.h").stat().st_mtime)
    keep_torch_obj = not force and torch_obj.exists() and torch_obj.stat().st_mtime > torch_newest \
        and torch_library_fits(torch.__version__, torch_obj)
    with ThreadPoolExecutor() as pool:
        running = [pool.submit(_compile, src, obj, verbose) for src, obj in jobs]
        if not keep_torch_obj:
            running.append(pool.submit(_compile_torch_ops, torch_obj, verbose))
        for done in running:
            done.result()
    tmp = LIB_PATH.with_suffix(".so.tmp")
    objs = [str(OBJ_DIR / (src.stem + ".o")) for src in sorted(SRC_DIR.glob("*.cu"))]
    subprocess.run([_nvcc(), *NVCC_FLAGS, "-shared", "-o", str(tmp), *objs], check=True)
    os.replace(tmp, LIB_PATH)
    _link_torch_ops(torch_obj)
    return LIB_PATH


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv, verbose="-v" in sys.argv))
