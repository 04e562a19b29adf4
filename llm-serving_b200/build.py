"""Build recipe for the sm_100a paged-decode library (``libpaged_decode.so``).

The library is a plain shared object with the C ABI of ``include/paged_decode.h``; Python
binds it with ctypes (``model/_native.py``). Every translation unit is compiled with
``nvcc -gencode arch=compute_100a,code=sm_100a`` in parallel, then linked with the static
CUDA runtime, so the .so only needs the driver (``libcuda.so.1``) at run time and can be
loaded (not used) on a host without a GPU.

The Python binding of the newer operators, ``pd_ops.so``, is compiled beside it with g++ against
torch's headers; it calls the library through addresses it is handed and links to nothing of it. Where
torch or g++ is missing, the library is built without it.

Usage: ``python llm-serving_b200/build.py [--force] [--verbose]``. The output lands next to
this file and is rebuilt only when a source is newer than it.
"""

from __future__ import annotations

import argparse
import importlib.metadata
import importlib.util
import os
import re
import shutil
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

HERE = Path(__file__).resolve().parent
CSRC = HERE / "csrc"
INCLUDE = HERE.parent / "include"
BUILD = HERE / "_build"
LIB = HERE / "libpaged_decode.so"
#: The Python binding of the newer operators (csrc/py_ops.cpp): a CPython extension over torch's
#: C++ API that calls the library's C ABI. Compiled by the host compiler, no device code.
OPS = HERE / "pd_ops.so"
#: The torch and interpreter it was compiled for: another of either rebuilds it.
OPS_STAMP = BUILD / "pd_ops.stamp"

SOURCES = [
    "pd_api.cu",
    "pd_append.cu",
    "pd_merge.cu",
    "pd_decode_bf16.cu",
    "pd_decode_f16.cu",
    "pd_decode_f32.cu",
    "pd_decode_mma_bf16.cu",
    "pd_decode_mma_f16.cu",
    "pd_decode_var_bf16.cu",
    "pd_decode_var_f16.cu",
    "pd_decode_var_f32.cu",
    "pd_decode_var_mma_bf16.cu",
    "pd_decode_var_mma_f16.cu",
    "pd_weights.cu",
    "pd_decode_cluster_bf16.cu",
    "pd_decode_cluster_f16.cu",
    "pd_decode_cluster_f32.cu",
    "pd_prefill.cu",
    "pd_prefill_tc.cu",
    "pd_ops_api.cu",
    "pd_norm_rope.cu",
    "pd_fp4_rows.cu",
    "pd_fp4_attend.cu",
    "pd_fp4_prefill.cu",
    "pd_block_copy.cu",
    "pd_evict.cu",
    "pd_window_prefill.cu",
]
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = [
    "-O3",
    "-std=c++17",
    "-lineinfo",
    "-Xcompiler",
    "-fPIC",
    "-Xptxas",
    "-O3",
    f"-I{INCLUDE}",
    f"-I{CSRC}",
]


def _nvcc() -> str:
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    path = Path(cuda) / "bin" / "nvcc"
    return str(path) if path.exists() else "nvcc"


def _headers(src: Path, seen: set[Path] | None = None) -> set[Path]:
    """The repository's headers that ``src`` includes, directly or through another."""
    seen = set() if seen is None else seen
    for name in re.findall(r'^#include "([^"]+)"', src.read_text(), flags=re.M):
        for folder in (CSRC, INCLUDE):
            header = folder / name
            if header.exists() and header not in seen:
                seen.add(header)
                _headers(header, seen)
    return seen


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    mtime = target.stat().st_mtime
    return any(dep.stat().st_mtime > mtime for dep in deps)


def _torch_root() -> Path | None:
    """Where torch is installed, without importing it; None where it is not."""
    spec = importlib.util.find_spec("torch")
    return Path(spec.origin).resolve().parent if spec is not None and spec.origin else None


def _ops_missing() -> str | None:
    """What the binding's build lacks on this host, or None."""
    root = _torch_root()
    if root is None:
        return "torch is not installed"
    if not (root / "include" / "ATen").is_dir():
        return f"torch's headers are not in {root / 'include'}"
    return None if shutil.which("g++") else "g++ is not on PATH"


def _ops_stamp() -> str:
    """What the binding was compiled against besides its sources: torch and the interpreter."""
    try:
        version = importlib.metadata.version("torch")
    except importlib.metadata.PackageNotFoundError:  # a source tree: its location has to do
        version = "?"
    return f"torch {version} in {_torch_root()}, {sysconfig.get_config_var('SOABI')}"


def _ops_stale() -> bool:
    source = CSRC / "py_ops.cpp"
    if _stale(OPS, [source, *_headers(source)]):
        return True
    return not OPS_STAMP.exists() or OPS_STAMP.read_text() != _ops_stamp()


def _ops_command() -> list[str]:
    import torch

    root = _torch_root()
    cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
    includes = [INCLUDE, CSRC, root / "include", root / "include/torch/csrc/api/include",
                sysconfig.get_paths()["include"], Path(cuda) / "include"]
    libs = ["torch_python", "torch", "torch_cpu", "torch_cuda", "c10", "c10_cuda"]
    return ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}",
            *[f"-I{p}" for p in includes], str(CSRC / "py_ops.cpp"), "-o", str(OPS), f"-L{root / 'lib'}",
            *[f"-l{name}" for name in libs]]


def build(force: bool = False, verbose: bool = False, ptxas_verbose: bool = False) -> Path:
    """Compile and link the library, and the Python binding beside it; returns the library's path.

    Raises on a compiler error. The library needs nvcc alone: on a host without what the binding needs
    (torch with its headers, g++) it is built all the same, and a line on stderr says what is missing."""
    BUILD.mkdir(exist_ok=True)
    nvcc = _nvcc()
    objects = []
    jobs = []
    for name in SOURCES:
        src = CSRC / name
        obj = BUILD / (Path(name).stem + ".o")
        objects.append(obj)
        if force or _stale(obj, [src, *_headers(src)]):
            cmd = [nvcc, *ARCH, *NVCC_FLAGS, "-c", str(src), "-o", str(obj)]
            if ptxas_verbose:
                cmd[1:1] = ["-Xptxas", "-v"]
            jobs.append(cmd)
    compile_jobs = len(jobs)
    missing = _ops_missing()
    if missing is not None:
        OPS.unlink(missing_ok=True)  # what is there may be for another torch
        sys.stderr.write(f"{OPS.name} is not built: {missing}\n")
    elif force or _ops_stale():
        OPS_STAMP.unlink(missing_ok=True)
        jobs.append(_ops_command())

    def run(cmd):
        if verbose:
            print(" ".join(cmd), flush=True)
        return cmd, subprocess.run(cmd, capture_output=True, text=True)

    def checked(cmd, proc):
        if proc.returncode != 0 or verbose or ptxas_verbose:
            sys.stderr.write(proc.stdout + proc.stderr)
        if proc.returncode != 0:
            raise RuntimeError(f"{Path(cmd[0]).name} failed ({proc.returncode}): {' '.join(cmd)}")

    with ThreadPoolExecutor(max_workers=max(1, min(len(jobs), os.cpu_count() or 1))) as pool:
        done = list(pool.map(run, jobs))
    for cmd, proc in done[:compile_jobs]:
        checked(cmd, proc)
    if force or compile_jobs or _stale(LIB, objects):
        checked(*run([nvcc, *ARCH, "-shared", "-cudart", "static", "-o", str(LIB), *map(str, objects)]))
    for cmd, proc in done[compile_jobs:]:  # the binding, after the library stands
        checked(cmd, proc)
        OPS_STAMP.write_text(_ops_stamp())
    return LIB


def main(argv: list[str] | None = None) -> int:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--force", action="store_true")
    parser.add_argument("--verbose", action="store_true")
    parser.add_argument("--ptxas-verbose", action="store_true", help="print registers/spills")
    args = parser.parse_args(argv)
    path = build(force=args.force, verbose=args.verbose, ptxas_verbose=args.ptxas_verbose)
    print(path)
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
