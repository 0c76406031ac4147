"""Builds the sm_100a kernel library `foidfinder_b200/_lib/libfoidfinder_b200.so` with nvcc.

Same role as the reference's loader/build step (foidfinder/backends/cuda/kernels.py:22-35,
`foidfinder build-kernels`), but ahead of time, in-tree and for `compute_100a` only: each `.cu` in
`csrc/` is compiled to an object in parallel and linked into one shared library that exports the C ABI
declared in `include/foidfinder_b200.h`. The CUDA runtime is linked statically, so the library needs
only the driver at run time.

`csrc/calls.cpp`, the short way from torch tensors into the calls that are made once per layer, becomes the extension
module `foidfinder_b200._calls` (host code only, g++ against torch's headers). Every call works without it, so a machine
that cannot build it still gets the library, and a warning. It is built again for another version of torch.

    python -m foidfinder_b200.build [--force] [--jobs N]
"""

from __future__ import annotations

import argparse
import concurrent.futures as cf
import os
import shutil
import subprocess
import sys
import sysconfig
from importlib.metadata import PackageNotFoundError, version
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
INCLUDE = ROOT / "include"
BUILD = ROOT / "_build"
LIB_DIR = PKG / "_lib"
LIB = LIB_DIR / "libfoidfinder_b200.so"
CALLS = PKG / ("_calls" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))

ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "-Xcompiler", "-fvisibility=hidden", f"-I{INCLUDE}"]


def nvcc() -> str:
    path = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not Path(path).exists():
        raise RuntimeError("nvcc not found; the CUDA 12.9 toolkit is required to build foidfinder_b200")
    return path


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def _stale(target: Path, deps: list[Path]) -> bool:
    if not target.exists():
        return True
    t = target.stat().st_mtime
    return any(d.stat().st_mtime > t for d in deps)


def build(force: bool = False, jobs: int | None = None, verbose: bool = False) -> Path:
    """Compiles (incrementally) and links the library; returns its path."""
    BUILD.mkdir(exist_ok=True)
    LIB_DIR.mkdir(exist_ok=True)
    headers = sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.h")) + sorted(INCLUDE.glob("*.h"))
    cc = nvcc()
    todo = []
    objects = []
    for src in sources():
        obj = BUILD / (src.stem + ".o")
        objects.append(obj)
        if force or _stale(obj, [src, *headers]):
            todo.append((src, obj))

    def compile_one(item: tuple[Path, Path]) -> tuple[Path, str]:
        src, obj = item
        cmd = [cc, *ARCH, *FLAGS, "-c", str(src), "-o", str(obj)]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        return src, r.stderr

    with cf.ThreadPoolExecutor(max_workers=jobs or os.cpu_count() or 4) as ex:
        for src, log in ex.map(compile_one, todo):
            if verbose:
                print(f"compiled {src.name}", log, file=sys.stderr)
    if force or todo or _stale(LIB, objects):
        tmp = LIB.with_suffix(".so.tmp")
        cmd = [cc, *ARCH, "-shared", "-o", str(tmp), *map(str, objects), "-cudart", "static"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, LIB)
    try:
        build_calls(force)
    except (RuntimeError, ImportError, OSError, PackageNotFoundError) as e:
        CALLS.unlink(missing_ok=True)  # an older one would not fit the sources or torch
        print(f"foidfinder_b200: {CALLS.name} was not built, calls from Python take their longer way: {e}", file=sys.stderr)
    return LIB


def build_calls(force: bool = False) -> Path:
    """The extension module of csrc/calls.cpp, for the installed torch; returns its path."""
    src, stamp, torch_version = CSRC / "calls.cpp", BUILD / "calls.torch", version("torch")
    if force or _stale(CALLS, [src, *INCLUDE.glob("*.h")]) or not stamp.exists() or stamp.read_text() != torch_version:
        import torch
        from torch.utils import cpp_extension as torch_paths

        cxx = shutil.which("g++") or shutil.which("c++")
        if cxx is None:
            raise RuntimeError("no C++ compiler found for foidfinder_b200/csrc/calls.cpp")
        include = [f"-I{p}" for p in (*torch_paths.include_paths("cuda"), sysconfig.get_paths()["include"], INCLUDE)]
        libs = [*(f"-L{p}" for p in torch_paths.library_paths("cuda")), "-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch_python"]
        tmp = CALLS.with_name(CALLS.name + ".tmp")
        cmd = [cxx, "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", f'-DFF_TORCH_VERSION="{torch.__version__}"', *include, str(src), "-o", str(tmp), *libs]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"{cxx} failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        os.replace(tmp, CALLS)
        stamp.write_text(torch_version)
    return CALLS


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--force", action="store_true")
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args()
    print(build(force=args.force, jobs=args.jobs, verbose=True))


if __name__ == "__main__":
    main()
