"""Builds the CUDA backend in-tree: llaccel_b200/csrc/*.cu -> llaccel_b200/_lib/libllx.so, and where
a torch with CUDA is installed the binding of the paged calls, csrc/torch_calls.cpp -> _lib/torch_calls.so.

    python -m llaccel_b200.build [--force]

Compiled for sm_100a only (B200).  nvcc cross-compiles without a GPU, so this runs on any
host with the CUDA toolkit.  The build is skipped when the library is newer than every
source file.
"""
from __future__ import annotations

import argparse
import fcntl
import importlib.util
import os
import shutil
import subprocess
import sys
import sysconfig
from pathlib import Path

PKG = Path(__file__).resolve().parent
CSRC = PKG / "csrc"
LIBDIR = PKG / "_lib"
LIB = LIBDIR / "libllx.so"
CALLS = LIBDIR / "torch_calls.so"
INCLUDE = PKG.parent / "include"

ARCH_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a"]
NVCC_FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC,-O3", "--expt-relaxed-constexpr",
              "-Xptxas", "-warn-spills"]


def nvcc() -> str:
    for cand in (os.environ.get("NVCC"), shutil.which("nvcc"), "/usr/local/cuda/bin/nvcc"):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("nvcc not found: the CUDA toolkit is required to build llaccel_b200")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.cu"))


def deps() -> list[Path]:
    return sources() + sorted(CSRC.glob("*.h")) + sorted(CSRC.glob("*.cuh")) + sorted(CSRC.glob("*.hpp")) + \
        sorted(INCLUDE.glob("*.h"))


def _newer(lib: Path, sources: list[Path]) -> bool:
    if not lib.exists():
        return False
    t = lib.stat().st_mtime
    return all(p.stat().st_mtime <= t for p in sources)


def lib_up_to_date() -> bool:
    return _newer(LIB, deps())


def cuda_torch() -> Path | None:
    """The folder of the installed torch if that is built with CUDA (looked up without importing it).
    Any other has no CUDA tensors to bind, nor the libraries to link with."""
    spec = importlib.util.find_spec("torch")
    root = Path(spec.origin).parent if spec is not None and spec.origin else None
    return root if root is not None and (root / "lib" / "libc10_cuda.so").exists() else None


def _made_for(root: Path) -> str:
    """What the binding depends on besides its sources: the torch in `root` and this Python."""
    return f"{(root / 'version.py').read_text()}{sysconfig.get_config_var('EXT_SUFFIX')}\n"


def calls_up_to_date() -> bool:
    root = cuda_torch()
    if root is None:
        return True
    note = CALLS.with_suffix(".torch")
    return _newer(CALLS, [CSRC / "torch_calls.cpp", *INCLUDE.glob("*.h")]) and note.exists() and note.read_text() == _made_for(root)


def up_to_date() -> bool:
    return lib_up_to_date() and calls_up_to_date()


def build(force: bool = False, verbose: bool = False) -> Path:
    """Compile if any source is newer than the library.  Processes that start together (one
    per GPU rank) serialise on a lock file: the first rebuilds, the others find the library
    up to date once they hold the lock."""
    if not force and up_to_date():
        return LIB
    LIBDIR.mkdir(exist_ok=True)
    with open(LIBDIR / ".build.lock", "w") as lock:
        fcntl.flock(lock, fcntl.LOCK_EX)
        try:
            if not force and up_to_date():
                return LIB
            if force or not lib_up_to_date():
                _compile(verbose)
            if force or not calls_up_to_date():
                _compile_calls(verbose)
            return LIB
        finally:
            fcntl.flock(lock, fcntl.LOCK_UN)


def _compile(verbose: bool) -> Path:
    objdir = PKG / "_build" / str(os.getpid())
    objdir.mkdir(parents=True, exist_ok=True)
    objs = []
    for src in sources():
        obj = objdir / (src.stem + ".o")
        cmd = [nvcc(), *ARCH_FLAGS, *NVCC_FLAGS, "-I", str(INCLUDE), "-I", str(CSRC), "-c", str(src), "-o", str(obj)]
        if verbose:
            print(" ".join(cmd))
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"nvcc failed on {src.name}:\n{r.stdout}\n{r.stderr}")
        if verbose and (r.stdout or r.stderr):
            print(r.stdout + r.stderr)
        objs.append(str(obj))
    tmp = LIB.with_suffix(f".so.{os.getpid()}.tmp")
    cmd = [nvcc(), *ARCH_FLAGS, "-shared", "-o", str(tmp), *objs, "-lcuda", "-ldl"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"link failed:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, LIB)
    shutil.rmtree(objdir, ignore_errors=True)
    return LIB


def _compile_calls(verbose: bool) -> None:
    root = cuda_torch()
    if root is None:
        return
    import torch

    tmp = CALLS.with_suffix(f".so.{os.getpid()}.tmp")
    cuda = Path(nvcc()).resolve().parent.parent
    cmd = ["g++", "-O2", "-std=c++17", "-fPIC", "-shared", f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           "-I", str(root / "include"), "-I", str(root / "include/torch/csrc/api/include"), "-I", str(cuda / "include"),
           "-I", sysconfig.get_paths()["include"], str(CSRC / "torch_calls.cpp"), "-o", str(tmp), "-L", str(root / "lib"),
           "-ltorch_python", "-ltorch_cpu", "-lc10_cuda", "-lc10"]
    if verbose:
        print(" ".join(cmd))
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"g++ failed on torch_calls.cpp:\n{r.stdout}\n{r.stderr}")
    os.replace(tmp, CALLS)
    CALLS.with_suffix(".torch").write_text(_made_for(root))


def main(argv=None) -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--force", action="store_true")
    ap.add_argument("-v", "--verbose", action="store_true")
    a = ap.parse_args(argv)
    print(build(a.force, a.verbose))


if __name__ == "__main__":
    main(sys.argv[1:])
