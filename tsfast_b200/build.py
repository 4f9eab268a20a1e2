"""Build ``libb200scan.so`` (the C-ABI CUDA library) in-tree with nvcc for sm_100a.

``python -m tsfast_b200.build`` compiles every ``csrc/*.cu`` into ``tsfast_b200/lib/`` and links
them into one shared library; ``build_host`` compiles the block operators' host path beside it.  nvcc cross-compiles,
so no GPU is needed to build.  Objects are rebuilt only when a source or header is newer.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "lib"
LIB = LIBDIR / "libb200scan.so"
INCLUDE = PKG.parent / "include"
HOST_SRC = CSRC / "host" / "block_host.cpp"
HOST_LIB = LIBDIR / "_block_host.so"

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-ccbin", "/usr/bin/g++",
]
# Approximate division / flush-to-zero only where the reference's own GPU kernels use fast
# transcendentals (the Mamba section and its conv + SiLU); the diagonal, all-pole, projection and
# glue kernels keep IEEE arithmetic.
FAST_MATH_SOURCES = {"mamba_scan.cu", "conv_silu.cu"}


def _nvcc() -> str:
    exe = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(exe).exists():
        raise RuntimeError("nvcc not found: cannot build libb200scan.so")
    return exe


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    mt = target.stat().st_mtime
    return any(d.stat().st_mtime > mt for d in deps)


def build(verbose: bool = False, force: bool = False, extra_flags: list[str] | None = None,
          out: Path | None = None) -> Path:
    """Compile the library; returns its path. ``extra_flags``/``out`` serve tuning builds."""
    LIBDIR.mkdir(exist_ok=True)
    out = Path(out) if out else LIB
    objdir = LIBDIR if out == LIB else out.parent / (out.stem + "_obj")
    objdir.mkdir(parents=True, exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted(INCLUDE.glob("*.h"))
    sources = sorted(CSRC.glob("*.cu"))
    nvcc = _nvcc()
    flags = NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + (extra_flags or [])

    def compile_one(src: Path):
        obj = objdir / (src.stem + ".o")
        if force or _stale(obj, [src, *headers]):
            extra = ["--use_fast_math"] if src.name in FAST_MATH_SOURCES else []
            r = subprocess.run([nvcc, *flags, *extra, "-c", str(src), "-o", str(obj)], capture_output=True, text=True)
            if r.returncode != 0:
                raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
            if verbose:
                sys.stderr.write(r.stderr)
            return obj, True
        return obj, False

    with ThreadPoolExecutor(max_workers=min(8, os.cpu_count() or 1)) as ex:
        results = list(ex.map(compile_one, sources))
    objs = [o for o, _ in results]
    if force or any(ch for _, ch in results) or _stale(out, objs):
        r = subprocess.run([nvcc, "-shared", "-o", str(out), *map(str, objs), "-ccbin", "/usr/bin/g++"],
                           capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    return out


def host_tag() -> str:
    """What the host path has to be built for; it stands in the built file."""
    import torch

    return f"b200 host path for torch {torch.__version__}, Python {sys.version_info.major}.{sys.version_info.minor}"


def host_is_current() -> bool:
    """Whether the built host path belongs to this torch and this Python."""
    return HOST_LIB.exists() and host_tag().encode() + b"\0" in HOST_LIB.read_bytes()


def build_host(force: bool = False) -> Path:
    """Compile the block operators' host path (a PyTorch extension module in C++, no CUDA code) with g++; returns its path."""
    import sysconfig

    import torch

    LIBDIR.mkdir(exist_ok=True)
    if not force and host_is_current() and not _stale(HOST_LIB, [HOST_SRC, INCLUDE / "b200scan.h"]):
        return HOST_LIB
    root = Path(torch.__file__).resolve().parent
    cuda = Path(_nvcc()).resolve().parent.parent
    cmd = ["/usr/bin/g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_block_host",
           "-DTORCH_API_INCLUDE_EXTENSION_H", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DB200_HOST_TAG="{host_tag()}"']
    for inc in (root / "include", root / "include" / "torch" / "csrc" / "api" / "include", cuda / "include"):
        cmd += ["-isystem", str(inc)]
    cmd += ["-I" + sysconfig.get_paths()["include"], str(HOST_SRC), "-o", str(HOST_LIB), "-L" + str(root / "lib"), "-lc10", "-lc10_cuda",
            "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on {HOST_SRC.name}:\n{r.stdout}\n{r.stderr}")
    return HOST_LIB


if __name__ == "__main__":
    p = build(verbose="-v" in sys.argv, force="-f" in sys.argv)
    build_host(force="-f" in sys.argv)
    print(p)
