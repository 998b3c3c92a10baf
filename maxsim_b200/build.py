"""Build recipe for libmaxsim_b200.so (sm_100a) -- in-tree, no JIT cache.

    python -m maxsim_b200.build            # or: from maxsim_b200.build import build; build()

Compiles every ``csrc/*.cu`` with nvcc for ``sm_100a`` into
``maxsim_b200/libmaxsim_b200.so`` (static cudart, so the library does not
depend on which libcudart torch bundles).  nvcc cross-compiles without a GPU.
``csrc/generation_binding.cpp`` becomes ``maxsim_b200/_generation.so``, the
Python module between torch and the library's cache and weight operators
(g++, torch's own headers and libraries).  Where torch is not installed only
the library is built; another torch than the module was built for makes the
module stale.
"""

from __future__ import annotations

import importlib.metadata
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIB = PKG / "libmaxsim_b200.so"
BINDING_SRC = CSRC / "generation_binding.cpp"
BINDING = PKG / "_generation.so"
ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-lineinfo", "-std=c++17", "--expt-relaxed-constexpr", "-Xcompiler", "-fPIC",
              "-Xptxas", "-warn-spills"]


def nvcc_path() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; set NVCC or install the CUDA toolkit")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def torch_build() -> str | None:
    """What the Python module depends on of torch and Python (without importing torch), None without torch."""
    spec = importlib.util.find_spec("torch")
    if spec is None:
        return None
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:
        version = "unknown"
    return f"{version} {spec.origin} {sysconfig.get_config_var('SOABI')}"


def _older(target: Path, deps: list[Path]) -> bool:
    return not target.exists() or any(p.stat().st_mtime > target.stat().st_mtime for p in deps if p.exists())


def _header() -> Path:
    return PKG.parent / "include" / "maxsim_b200.h"


def _stamp() -> Path:
    return PKG / "_build" / "generation.torch"


def library_stale() -> bool:
    return _older(LIB, sources() + sorted(CSRC.glob("*.cuh")) + [_header()])


def binding_stale() -> bool:
    torch = torch_build()
    if torch is None:
        return False
    return _older(BINDING, [BINDING_SRC, _header()]) or not _stamp().exists() or _stamp().read_text() != torch


def needs_build() -> bool:
    return library_stale() or binding_stale()


def build(force: bool = False, verbose: bool = False) -> Path:
    if force or library_stale():
        build_library(verbose)
    if torch_build() is None:
        sys.stderr.write("torch is not installed: _generation.so (Int4KVCache, Int4Linear) is not built\n")
    elif force or binding_stale():
        build_binding()
    return LIB


def build_library(verbose: bool = False) -> Path:
    nvcc = nvcc_path()
    objdir = PKG / "_build"
    objdir.mkdir(exist_ok=True)
    objs = []
    procs = []
    for src in sources():
        obj = objdir / (src.stem + ".o")
        cmd = [nvcc, *ARCH_FLAGS, *NVCC_FLAGS, "-dc" if False else "-c", str(src), "-o", str(obj)]
        procs.append((src, cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
        objs.append(obj)
    failed = False
    for src, cmd, p in procs:
        out, _ = p.communicate()
        text = out.decode(errors="replace")
        if p.returncode != 0:
            failed = True
            sys.stderr.write(f"nvcc failed for {src.name}:\n{text}\n")
        elif verbose and text.strip():
            sys.stderr.write(text)
    if failed:
        raise RuntimeError("CUDA build failed")
    tmp = LIB.with_suffix(".so.tmp")
    cmd = [nvcc, *ARCH_FLAGS, "-shared", "-o", str(tmp), *map(str, objs), "-cudart", "static"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, LIB)
    return LIB


def build_binding() -> Path:
    import torch

    base = Path(torch.__file__).resolve().parent
    cuda = Path(nvcc_path()).resolve().parent.parent
    tmp = BINDING.with_suffix(".so.tmp")
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}", f"-I{base / 'include'}",
           f"-I{base / 'include/torch/csrc/api/include'}", f"-I{cuda / 'include'}",
           f"-I{sysconfig.get_paths()['include']}", str(BINDING_SRC), "-o", str(tmp), f"-L{base / 'lib'}", f"-L{PKG}",
           "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda", "-lc10", "-lc10_cuda", f"-l:{LIB.name}", "-Wl,-rpath,$ORIGIN"]
    subprocess.run(cmd, check=True)
    os.replace(tmp, BINDING)
    _stamp().parent.mkdir(exist_ok=True)
    _stamp().write_text(torch_build())
    return BINDING


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
