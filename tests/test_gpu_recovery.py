"""What follows a call that failed for want of memory, on the GPU."""
from __future__ import annotations

import pytest

from conftest import GOLDEN

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from llaccel_b200 import build  # noqa: E402

build.build()
from llaccel_b200.cuda_backend import LLX_ERR_OOM, CudaModel, CudaServe, LlxError  # noqa: E402


@pytest.mark.parametrize("graph", ["c1_v2", "qwen3_tiny"])
def test_a_cache_too_large_for_the_device_is_only_refused(graph):
    """The allocation that failed is reported once, not again by the next launch."""
    with CudaModel(GOLDEN / graph) as m:
        want = m.generate([1, 2, 3], 4)["generated"]
        for use in (lambda: m.generate([1, 2, 3], 4)["generated"], lambda: CudaServe(m, max_seqs=2, n_pages=4).generate([[1, 2, 3]], 4)[0]):
            with pytest.raises(LlxError) as e:
                CudaServe(m, max_seqs=2, n_pages=2 ** 31 - 1, page_size=256)  # terabytes
            assert e.value.code == LLX_ERR_OOM
            assert use() == want
