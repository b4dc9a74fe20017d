"""The order in which kernels take tensor memory and let their dependents launch, from the sources."""
from __future__ import annotations

import re

import pytest

from conftest import REPO

SOURCES = sorted((REPO / "llaccel_b200" / "csrc").glob("*.cu"))


def kernels(text: str):
    """(name, body) of each __global__ function."""
    for m in re.finditer(r"__global__ void(?:\s+__launch_bounds__\([^)]*\))?\s+(\w+)\(", text):
        at = text.index("{", text.index(")", m.end()))
        end = re.compile(r"^}", re.M).search(text, at)
        yield m.group(1), re.sub(r"//[^\n]*", "", text[at : end.end()])


def test_every_tcgen05_kernel_is_found():
    found = [n for p in SOURCES for n, body in kernels(p.read_text()) if "tcgen05.alloc" in body]
    assert len(found) == sum(p.read_text().count("tcgen05.alloc.") for p in SOURCES) >= 4


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_tensor_memory_is_taken_before_dependents_launch(source):
    """A dependent takes its columns before it waits for this grid.  Were it on the SM first, a CTA of this
    grid could wait for columns that it gives back only after this grid is done."""
    for name, body in kernels(source.read_text()):
        if "tcgen05.alloc" in body and "pdl_trigger()" in body:
            assert body.index("tcgen05.alloc") < body.index("pdl_trigger()"), name
