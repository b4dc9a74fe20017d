"""The serving calls' host code on the CPU: `serve_host_check.cpp` runs the real runtime.cu over a fake CUDA
runtime and makes every operation of a step, a fork and a compaction fail in turn.  A call that fails after
it began to change slots must not leave them open, nor say that nothing was changed."""
from __future__ import annotations

import re
import subprocess
from pathlib import Path

import pytest

from conftest import GOLDEN, REPO
from llaccel_b200 import build as B

HERE = REPO / "tests"


def run(*cmd, **kw):
    r = subprocess.run([str(c) for c in cmd], capture_output=True, text=True, **kw)
    assert r.returncode == 0, r.stdout[-3000:] + r.stderr[-3000:]
    return r.stdout


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    try:
        nvcc = B.nvcc()
    except RuntimeError:
        pytest.skip("nvcc not available")
    tmp = tmp_path_factory.mktemp("serve_host")
    run(nvcc, *B.ARCH_FLAGS, "-std=c++17", "-O1", "--expt-relaxed-constexpr", "-I", B.INCLUDE, "-I", B.CSRC, "-c", B.CSRC / "runtime.cu",
        "-o", tmp / "runtime.o")
    run("g++", "-std=c++17", "-O1", "-I", B.INCLUDE, "-I", Path(nvcc).resolve().parent.parent / "include", "-c", HERE / "serve_host_check.cpp",
        "-o", tmp / "check.o")
    # what neither file has: launches of kernels can fail, the rest says 0
    names = lambda f, *kind: set(re.findall(r"\b(\S+)$", run("nm", *kind, f), re.M))  # noqa: E731
    missing = names(tmp / "runtime.o", "-u") - names(tmp / "check.o", "--defined-only")
    stubs = [".text"]
    for n in sorted(m for m in missing if re.match(r"_ZN3llx|_?_?cuda", m)):
        fails = re.match(r"_ZN3llx\d+launch_|cudaLaunchKernel", n)
        stubs += [f".globl {n}", f"{n}:", " jmp fake_launch" if fails else " xor %eax, %eax\n ret"]
    (tmp / "stubs.s").write_text("\n".join([*stubs, '.section .note.GNU-stack,"",@progbits', ""]))
    run("g++", tmp / "check.o", tmp / "runtime.o", tmp / "stubs.s", "-no-pie", "-ldl", "-o", tmp / "check")
    return tmp / "check"


@pytest.mark.parametrize("graph", ["c1_v2", "qwen3_tiny"])
def test_failing_calls(check, graph):
    assert run(check, GOLDEN / graph, timeout=300).splitlines()[-1] == "0 failures"
