"""The paged-serving calls at the ends of what their arguments can say."""
from __future__ import annotations

import subprocess

import numpy as np
import pytest

from conftest import REPO

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from llaccel_b200 import build
    build.build()
    from llaccel_b200 import paged
    return paged


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_page_counts_add_up_in_64_bits(tmp_path):
    from llaccel_b200 import build as B
    r = subprocess.run([B.nvcc(), "-std=c++17", *B.ARCH_FLAGS, "--expt-relaxed-constexpr", "-I", str(B.INCLUDE), "-I", str(B.CSRC), "-c",
                        str(REPO / "tests" / "paged_plan_check.cu"), "-o", str(tmp_path / "check.o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]


@gpu
def test_requests_beyond_32_bits_of_pages_are_refused(paged):
    """128 slots of 2^24 pages each: 2^31 pages, of a cache that has four."""
    W, P, N = 1 << 24, 16, 4
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs a page table of 8 GB")
    table = torch.full((129, W), -1, dtype=torch.int32, device="cuda")
    length, refs = torch.zeros(129, dtype=torch.int32, device="cuda"), ints([0, 1, 0, 0])
    status = ints([0])
    paged.reserve(table, length, refs, ints(range(1, 129)), torch.full((128,), W * P, dtype=torch.int32, device="cuda"), P, status=status)
    assert int(status.item()) == 8
    assert not length.any() and refs.tolist() == [0, 1, 0, 0] and int(table.max()) == -1
    status.zero_()
    length[0], table[0] = W * P, 1
    k, v = (torch.zeros((N, 1, P, 16), dtype=torch.int8, device="cuda") for _ in "kv")
    paged.fork(k, v, table, length, refs, torch.zeros(128, dtype=torch.int32, device="cuda"), ints(range(1, 129)), share=False,
               status=status)
    assert int(status.item()) == 8
    assert not length[1:].any() and refs.tolist() == [0, 1, 0, 0] and int(table[1:].max()) == -1


@gpu
@pytest.mark.parametrize("share", [True, False])
@pytest.mark.parametrize("bad", [-1, 9, 1 << 30])
def test_a_fork_of_a_page_that_is_not_there_changes_nothing(paged, share, bad):
    """Among good pairs; the page of the copy used to be some former owner's."""
    rng = np.random.default_rng(0)
    N, P, status = 9, 16, ints([0])
    k, v = (torch.from_numpy(rng.integers(-128, 128, (2, N, 2, P, 32)).astype(np.int8)).cuda() for _ in "kv")
    table = ints([[4, 0, -1], [7, -1, -1], [bad if not share else 5, bad if share else 6, -1], [2, 8, -1], [-1] * 3])
    length, refs = ints([20, 16, 20, 30, 0]), ints([1, 0, 1, 0, 1, 1, 1, 1, 1])
    before = [t.clone() for t in (k, v, table, length, refs)]
    paged.fork(k, v, table, length, refs, ints([0, 2]), ints([3, 4]), share=share, status=status)
    assert int(status.item()) == 1
    assert all(torch.equal(x, y) for x, y in zip(before, (k, v, table, length, refs)))
    paged.fork(k, v, table, length, refs, ints([0, 1]), ints([3, 4]), share=share, status=status.zero_())
    assert int(status.item()) == 0 and length.tolist() == [20, 16, 20, 20, 16]
    new = table[3, 1].long()
    assert torch.equal(k[:, new, :, :4], before[0][:, 0, :, :4])


@pytest.mark.parametrize("name", ["llx_paged_append", "llx_paged_attention", "llx_pages_fork", "llx_sample"])
def test_a_device_that_is_not_there_is_refused(paged, name):
    """Not run on the current one instead."""
    from test_paged_host import call
    lib = paged.load_library()
    for device in (1000, 1 << 31, (1 << 32) + 1):
        assert call(lib, name, device=device) in (1, 3)  # LLX_ERR_INVALID, LLX_ERR_CUDA
        assert lib.llx_last_error().decode().startswith(name + ": ")


@gpu
def test_a_call_for_a_device_that_is_not_there_changes_nothing(paged):
    lib = paged.load_library()
    table, length, refs, slots = ints([[0, 1], [2, -1]]), ints([20, 3]), ints([1, 1, 1]), ints([0, 1])

    def free(device):
        pack = (0, 0, 0, 256, 1, 3, 1, 16, 16, table.data_ptr(), 2, 2, 2, length.data_ptr(), refs.data_ptr(), slots.data_ptr(), 0, 2,
                0, 0, 0, 0, 0, device)
        code = lib.llx_pages_free(paged._PAGES.pack(*pack), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return code

    assert free(torch.cuda.device_count()) == 3 and length.tolist() == [20, 3] and refs.tolist() == [1, 1, 1]
    assert torch.cuda.current_device() == 0
    assert free(0) == 0 and length.tolist() == [0, 0] and refs.tolist() == [0, 0, 0]


@gpu
def test_lengths_end_at_31_bits(paged):
    """A table row of 2^24 pages of 256 holds more positions than an int32 length can count."""
    W, P, status = 1 << 24, 256, ints([0])
    table = torch.full((1, W), -1, dtype=torch.int32, device="cuda")
    table[0, (2 ** 31 - 10) // P] = 0
    length, refs = ints([2 ** 31 - 10]), ints([1, 0])
    paged.reserve(table, length, refs, ints([0]), ints([10]), P, status=status)
    assert int(status.item()) == 2 and length.tolist() == [2 ** 31 - 10] and refs.tolist() == [1, 0]
    paged.reserve(table, length, refs, ints([0]), ints([9]), P, status=status.zero_())
    assert int(status.item()) == 0 and length.tolist() == [2 ** 31 - 1] and refs.tolist() == [1, 0]


@gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows", [[1, 1], [3, 40]])
def test_the_lowest_length_has_no_keys(paged, rows, D):
    """-2^31 less the launch's rows does not become a long context."""
    from test_paged_ops import attention_case
    assert attention_case(np.random.default_rng(D), 4, 2, D, 16, rows, [-2 ** 31, 40]) == 2


@gpu
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("rows", [[0, 1, 0], [0, 40, 0]])
def test_bounds_are_those_of_sequences_with_rows(paged, rows, D):
    """A slot that brings none may be longer than max_len (or hold a length of no sense): nothing of it is computed."""
    from test_paged_ops import attention_case
    assert attention_case(np.random.default_rng(D), 4, 2, D, 16, rows, [100, 50, -7], max_len=50) == 0
    assert attention_case(np.random.default_rng(D), 4, 2, D, 16, rows, [100, 50, -7], max_len=49) == 4


@gpu
@pytest.mark.parametrize("D", [32, 64])
def test_launches_without_rows(paged, D):
    """No rows (of no sequence, or of two that bring none), no slots, nothing to sample: nothing to do."""
    from llaccel_b200 import sampling
    H, Hkv, P = 4, 2, 16
    pages = [torch.full((3, Hkv, P, D), 5, dtype=torch.int8, device="cuda") for _ in "kv"]
    table, length, status = ints([[0], [1]]), ints([3, 0]), ints([0])
    cos, sin = (torch.zeros((20, D // 2), dtype=torch.int16, device="cuda") for _ in "cs")
    for q_start, seqs in (([0], None), ([0, 0, 0], None), ([0, 0, 0], ints([1, 0])), ([0], ints([]))):
        new = [torch.zeros((0, h, D), dtype=t, device="cuda") for h, t in ((H, torch.int16), (Hkv, torch.int16), (Hkv, torch.int8))]
        q8 = paged.append(*new, *pages, table, length, ints(q_start), cos, sin, (1 << 30, 33), (1 << 30, 33), seqs=seqs, status=status)
        o = paged.attention(q8, *pages, table, length, ints(q_start), (1 << 30, 33), (1 << 30, 33), max_rows=0, max_len=3, seqs=seqs,
                            status=status)
        assert q8.shape == o.shape == (0, H, D) and o.dtype == torch.int8
    with pytest.raises(ValueError, match="must be"):
        paged.attention(q8, *pages, table, length, ints([0]).long(), (1, 33), (1, 33), max_rows=0, max_len=3)
    refs = ints([1, 0, 0])
    paged.reserve(table, length, refs, ints([]), ints([]), P, status=status)
    paged.fork(*pages, table, length, refs, ints([]), ints([]), status=status)
    paged.free(table, length, refs, ints([]), status=status)
    token, prob = sampling.sample(torch.zeros((0, 9), dtype=torch.int16, device="cuda"), torch.zeros(0, dtype=torch.float64, device="cuda"),
                                  exponent=-3)
    assert len(token) == len(prob) == 0
    assert int(status.item()) == 0 and length.tolist() == [3, 0] and refs.tolist() == [1, 0, 0] and all(int(p.min()) == 5 for p in pages)
