"""Builds libw4a8.so (the C-ABI CUDA library) in-tree for sm_100a, and the
small torch module _w4a8_torch.so beside it.

Usage: python build_native.py [--force] [--library]   (--library: libw4a8.so alone)

The library is self-contained (static CUDA runtime, no torch linkage); the
Python module ``int4_int8_ext`` loads it with ctypes. _w4a8_torch.so holds the
argument checks of the 4-bit cache operators, against the installed torch.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
LIB = HERE / "libw4a8.so"
BINDING = HERE / "_w4a8_torch.so"
BINDING_SOURCE = "torch_binding.cpp"
SOURCES = ["gemm_conv.cu", "aux_kernels.cu", "kv_cache.cu", "attn_int4.cu"]
# Sources compiled once for each head size, with -DW4A8_HEAD_DIM.
DIM_SOURCES = ["attn_int4_dim.cu"]
HEAD_DIMS = (64, 96, 128, 192, 256)
HEADERS = ["ptx.cuh", "launch.cuh", "mma_kernel.cuh", "gemm_w4_kernel.cuh", "gemv_w4.cuh", "tensormap.cuh",
           "kv_cache.cuh", "kv_host.cuh", "attn_int4.cuh", "attn_int4_host.cuh",
           "prefill_int4.cuh"]

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC",
    "-Xcompiler", "-fvisibility=hidden",
]


def _nvcc() -> str:
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    cand = Path(cuda_home) / "bin" / "nvcc"
    return str(cand) if cand.exists() else "nvcc"


def _built_for() -> str:
    """What a torch module fits: one torch and one Python."""
    import torch

    return f"torch {torch.__version__}, C++11 ABI {int(torch._C._GLIBCXX_USE_CXX11_ABI)}, {sysconfig.get_config_var('SOABI')}"


def _note() -> Path:
    """The file that says what the torch module was built for."""
    return HERE / "_build" / (BINDING.stem + ".txt")


def _fits() -> bool:
    try:
        return _note().read_text() == _built_for()
    except (OSError, ImportError):
        return False


def _build_binding(verbose: bool) -> None:
    """Compiles _w4a8_torch.so against the installed torch."""
    import torch

    root = Path(torch.__file__).resolve().parent
    cuda_home = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    includes = [sysconfig.get_paths()["include"], root / "include", root / "include/torch/csrc/api/include",
                Path(cuda_home) / "include", INCLUDE]
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
           f"-DTORCH_EXTENSION_NAME={BINDING.stem}", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           *[f"-I{i}" for i in includes], str(CSRC / BINDING_SOURCE), "-o", str(tmp), f"-L{root / 'lib'}", "-lc10",
           "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    _note().parent.mkdir(exist_ok=True)
    _note().write_text(_built_for())


def _stale(target: Path, deps) -> bool:
    """Whether target is missing or older than what it is made from."""
    if not target.exists():
        return True
    at = target.stat().st_mtime
    return any(d.stat().st_mtime > at for d in [*deps, INCLUDE / "w4a8.h", Path(__file__)] if d.exists())


def _build_library(pool: ThreadPoolExecutor, verbose: bool) -> None:
    """Compiles every CUDA source for sm_100a and links libw4a8.so."""
    objdir = HERE / "_build"
    objdir.mkdir(exist_ok=True)
    nvcc = _nvcc()
    units = [(src, Path(src).stem, []) for src in SOURCES]
    units += [(src, f"{Path(src).stem}{d}", [f"-DW4A8_HEAD_DIM={d}"]) for src in DIM_SOURCES for d in HEAD_DIMS]

    def compile_unit(unit) -> str:
        src, stem, defines = unit
        obj = objdir / (stem + ".o")
        cmd = [nvcc, *NVCC_FLAGS, *defines, "-I", str(INCLUDE), "-c", str(CSRC / src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
        return str(obj)

    objs = list(pool.map(compile_unit, units))
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-o", str(tmp), *objs,
           "-Xcompiler", "-fPIC"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)


def build(force: bool = False, verbose: bool = False, torch_module: bool = True) -> Path:
    """Builds libw4a8.so and, unless torch_module is False, the torch module beside it, where they are missing or older than
    their sources, the module also where it was built for another torch or Python. The library needs nvcc alone and is in place before a failure of the module is raised."""
    library = force or _stale(LIB, [CSRC / s for s in SOURCES + DIM_SOURCES + HEADERS])
    module = torch_module and (force or not _fits() or _stale(BINDING, [CSRC / BINDING_SOURCE]))
    with ThreadPoolExecutor(max_workers=max(1, os.cpu_count() or 1)) as pool:
        binding = pool.submit(_build_binding, verbose) if module else None
        if library:
            _build_library(pool, verbose)
        if binding and binding.exception():
            raise RuntimeError(f"libw4a8.so is built, the torch module {BINDING.name} is not: {binding.exception()}"
                               ) from binding.exception()
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True, torch_module="--library" not in sys.argv)
    print(LIB)
