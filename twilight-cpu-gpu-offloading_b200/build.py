"""Build recipe of the sm_100a extension (libtwilight_b200.so, in-tree).

    python twilight-cpu-gpu-offloading_b200/build.py

nvcc cross-compiles for sm_100a without a GPU.  The shared library exports
the C ABI declared in include/twilight_b200.h; _binding.so calls it with torch
tensors where a call through ctypes would take the host too long.
"""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
REPO = PKG.parent
CSRC = PKG / "csrc"
LIB = PKG / "libtwilight_b200.so"
BINDING = PKG / "_binding.so"  # Python calls with torch tensors (csrc/binding.cpp)
SOURCES = ["quest.cu", "int4.cu", "topp_union.cu", "gather.cu", "attention.cu", "frontend.cu",
           "capi.cu", "paged.cu", "paged_attention.cu",
           "paged_token.cu", "paged_chunk.cu", "rope.cu", "paged_weights.cu", "paged_evict.cu"]
NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a",
    "-O3", "-lineinfo", "-std=c++17",
    "-Xcompiler", "-fPIC", "-shared",
    "--expt-relaxed-constexpr",
]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), "/usr/local/cuda/bin/nvcc", shutil.which("nvcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found; the sm_100a extension cannot be built")


def sources() -> list[Path]:
    return [CSRC / s for s in SOURCES]


def binding_command() -> list[str]:
    """g++ against the headers and libraries of the installed torch."""
    import torch
    from torch.utils import cpp_extension

    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"],
               str(Path(nvcc()).resolve().parents[1] / "include")]
    lib = Path(torch.__file__).resolve().parent / "lib"
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared",
            f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *[f"-I{p}" for p in include], str(CSRC / "binding.cpp"), "-o",
            str(BINDING.with_suffix(".so.tmp")), f"-L{PKG}", f"-l:{LIB.name}",
            "-Wl,-rpath,$ORIGIN", f"-L{lib}", "-lc10", "-lc10_cuda", "-ltorch", "-ltorch_cpu",
            "-ltorch_python"]


def needs_build() -> bool:
    if not LIB.exists() or not BINDING.exists():
        return True
    mtime = min(LIB.stat().st_mtime, BINDING.stat().st_mtime)
    deps = sources() + list(CSRC.glob("*.cuh")) + [CSRC / "binding.cpp"] + [REPO / "include" / "twilight_b200.h"]
    return any(d.stat().st_mtime > mtime for d in deps)


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compiles every source to an object in parallel (one nvcc per file),
    then links the shared library."""
    if not force and not needs_build():
        return LIB
    obj_dir = PKG / "_build"
    obj_dir.mkdir(exist_ok=True)
    compile_flags = [f for f in NVCC_FLAGS if f != "-shared"]
    jobs = []
    for src in sources():
        obj = obj_dir / (src.stem + ".o")
        jobs.append((obj, [nvcc(), *compile_flags, "-c", str(src), "-o", str(obj)]))
    if verbose:
        for _, cmd in jobs:
            print(" ".join(cmd))
    workers = max(1, min(len(jobs), os.cpu_count() or 1))
    with ThreadPoolExecutor(max_workers=workers) as pool:
        results = list(pool.map(lambda j: subprocess.run(j[1]).returncode, jobs))
    if any(results):
        raise RuntimeError(f"nvcc failed for {[str(j[0].name) for j, r in zip(jobs, results) if r]}")
    tmp = LIB.with_suffix(".so.tmp")
    link = [nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-shared", "-Xcompiler", "-fPIC",
            *[str(o) for o, _ in jobs], "-o", str(tmp)]
    if verbose:
        print(" ".join(link))
    subprocess.run(link, check=True)
    tmp.replace(LIB)
    cmd = binding_command()
    if verbose:
        print(" ".join(cmd))
    subprocess.run(cmd, check=True)
    BINDING.with_suffix(".so.tmp").replace(BINDING)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv, verbose=True)
    print(LIB)
