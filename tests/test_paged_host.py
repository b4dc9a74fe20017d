"""What the paged-serving calls refuse, and their argument layout: on the CPU.  The C entry points
check before they touch CUDA, so bad arguments are refused the same way without a device."""
from __future__ import annotations

import re
import struct

import numpy as np
import pytest

from conftest import REPO
from oracle import paged_oracle as PO

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lib():
    from llaccel_b200 import build, cuda_backend
    build.build()
    return cuda_backend.load_library()


def fields(name: str) -> list[str]:
    text = re.sub(r"/\*.*?\*/", "", (REPO / "include" / "llx.h").read_text(), flags=re.S)
    body = text[: text.index("} " + name + ";")]
    body = body[body.rindex("typedef struct {") + len("typedef struct {"):]
    return [re.sub(r"[*\s]", "", part.split()[-1] if i == 0 else part) for line in body.split(";") if line.strip()
            for i, part in enumerate(line.strip().split(","))]


GOOD = {
    "llx_paged_append": dict(q=16, k=16, v=16, q8=16, q_stride=256, k_stride=128, v_stride=128, q8_stride=256, rows=0, n_heads=4,
                             n_kv_heads=2, head_dim=64, cos=16, sin=16, n_positions=9, q_M=1, k_M=1, k_pages=16, v_pages=16,
                             page_stride=2048, n_pages=4, page_size=16, table=16, table_stride=2, max_seqs=3, max_pages=2,
                             length=16, q_start=16, n_seqs=0),
    "llx_paged_attention": dict(q8=16, out=16, q8_stride=256, out_stride=256, rows=0, n_heads=4, n_kv_heads=2, head_dim=64,
                                k_pages=16, v_pages=16, page_stride=2048, n_pages=4, page_size=16, table=16, table_stride=2,
                                max_seqs=3, max_pages=2, length=16, q_start=16, n_seqs=0, max_rows=1, max_len=9, Ms=1, Ss=33, Mo=1,
                                So=33, prob_bits=15),
    "llx_pages_fork": dict(k=16, v=16, layer_stride=8192, page_stride=2048, n_layers=2, n_pages=4, n_kv_heads=2, page_size=16,
                           head_dim=64, table=16, table_stride=2, max_seqs=3, max_pages=2, length=16, refs=16, list_a=16,
                           list_b=16, n=0, share=1, scratch=16),
    "llx_sample": dict(logits=16, logits_stride=100, rows=0, vocab=100, exponent=-10, random=16, token=16),
}
STRUCTS = {"llx_paged_append": "llx_paged_append_args", "llx_paged_attention": "llx_paged_attention_args",
           "llx_pages_fork": "llx_pages_args", "llx_sample": "llx_sample_args"}


def call(lib, name, **change):
    values = dict(GOOD[name], **change)
    names = fields(STRUCTS[name])
    assert set(values) <= set(names), set(values) - set(names)
    return getattr(lib, name)(struct.pack(f"={len(names)}q", *(values.get(n, 0) for n in names)), None)


def test_packed_structs_have_the_headers_fields(lib):
    from llaccel_b200 import paged, sampling
    for packed, name in ((paged._APPEND, "llx_paged_append_args"), (paged._ATTENTION, "llx_paged_attention_args"),
                         (paged._PAGES, "llx_pages_args"), (sampling._SAMPLE, "llx_sample_args")):
        assert packed.size == 8 * len(fields(name)), name


@pytest.mark.parametrize("name,change,text", [
    ("llx_paged_append", dict(head_dim=72), "head_dim"), ("llx_paged_append", dict(head_dim=272), "head_dim"),
    ("llx_paged_append", dict(page_size=24), "page_size"), ("llx_paged_append", dict(page_size=8), "page_size"),
    ("llx_paged_append", dict(page_stride=2032), "page_stride"), ("llx_paged_append", dict(page_stride=2056), "page_stride"),
    ("llx_paged_append", dict(n_heads=3), "n_heads"), ("llx_paged_append", dict(rows=-1), "rows"),
    ("llx_paged_append", dict(q=0), "null"), ("llx_paged_append", dict(table=0), "page table"),
    ("llx_paged_append", dict(table_stride=1), "stride"), ("llx_paged_append", dict(max_seqs=0), "max_seqs"),
    ("llx_paged_append", dict(q_stride=255), "stride"), ("llx_paged_append", dict(q_M=-1), "requantization"),
    ("llx_paged_append", dict(k_S=64), "requantization"), ("llx_paged_append", dict(k_M=1 << 32), "requantization"),
    ("llx_paged_append", dict(q_gamma=16, q_C=1 << 40), "norm"), ("llx_paged_append", dict(k_gamma=16, k_eps=-1), "norm"),
    ("llx_paged_append", dict(n_positions=0), "position"), ("llx_paged_append", dict(device=-1), "device"),
    ("llx_paged_attention", dict(prob_bits=16), "prob_bits"), ("llx_paged_attention", dict(Ss=64), "score"),
    ("llx_paged_attention", dict(Mo=-3), "output"), ("llx_paged_attention", dict(q8=8), "aligned"),
    ("llx_paged_attention", dict(q8_stride=260), "aligned"), ("llx_paged_attention", dict(out_stride=128), "stride"),
    ("llx_paged_attention", dict(max_rows=-1), "max_rows"), ("llx_paged_attention", dict(v_pages=0), "null"),
    ("llx_paged_attention", dict(n_pages=0), "n_pages"), ("llx_paged_attention", dict(n_seqs=-1), "n_seqs"),
    ("llx_pages_fork", dict(n=4), "slot"), ("llx_pages_fork", dict(n=-1), "slot"), ("llx_pages_fork", dict(k=8), "aligned"),
    ("llx_pages_fork", dict(scratch=0), "null"), ("llx_pages_fork", dict(refs=0), "refs"),
    ("llx_pages_fork", dict(n_layers=0), "n_layers"), ("llx_pages_fork", dict(layer_stride=8), "layer_stride"),
    ("llx_pages_fork", dict(max_seqs=(1 << 18) + 1), "max_seqs"), ("llx_pages_fork", dict(n=2, list_b=0), "null"),
    ("llx_sample", dict(vocab=0), "vocabulary"), ("llx_sample", dict(vocab=101), "stride"),
    ("llx_sample", dict(exponent=-32), "exponent"), ("llx_sample", dict(exponent=16), "exponent"),
    ("llx_sample", dict(rows=1, random=0), "null"), ("llx_sample", dict(rows=-1), "rows"),
])
def test_refused_arguments(lib, name, change, text):
    assert call(lib, name, **change) == 1  # LLX_ERR_INVALID
    message = lib.llx_last_error().decode()
    assert message.startswith(name + ": ") and text in message


def test_a_null_struct_and_a_huge_vocabulary_are_refused(lib):
    assert lib.llx_sample(None, None) == 1
    assert call(lib, "llx_sample", vocab=1 << 19, logits_stride=1 << 19) == 6  # LLX_ERR_UNSUPPORTED
    assert lib.llx_pages_scratch(10) == 4 * 34 and lib.llx_pages_scratch(-1) == 0


def test_calls_refuse_host_tensors():
    from llaccel_b200 import paged, sampling
    i8, i16, i32 = (torch.zeros(2, 2, 64, dtype=t) for t in (torch.int8, torch.int16, torch.int32))
    pages = torch.zeros(3, 2, 16, 64, dtype=torch.int8)
    ints = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged.append(i16, i16, i8, pages, pages, table, ints, ints, i16, i16, (1, 1), (1, 1))
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged.attention(i8, pages, pages, table, ints, ints, (1, 1), (1, 1), max_rows=1, max_len=1)
    with pytest.raises(ValueError, match="CUDA tensor"):
        paged.fork(pages, pages, table, ints, ints, ints, ints)
    with pytest.raises(ValueError, match="CUDA tensor"):
        sampling.sample(i16[0], torch.zeros(2, dtype=torch.float64), exponent=-10)


def test_pool_and_row_layouts():
    from llaccel_b200 import paged
    five = torch.zeros(2, 3, 2, 16, 64, dtype=torch.int8)
    assert paged._pool(five, five.clone()) == (6144, 2048, 2, 3, 2, 16, 64)
    with pytest.raises(ValueError, match="dense"):
        paged._pool(five[..., ::2], five[..., ::2])
    with pytest.raises(ValueError, match="alike"):
        paged._pool(five, five[0])
    x = torch.zeros(5, 300)
    assert paged._rows(x[:, 40:168].unflatten(1, (2, 64)), "x", 2, 64, 5) == 300
    with pytest.raises(ValueError, match="dense"):
        paged._rows(x[:, :256].unflatten(1, (4, 64))[:, ::2], "x", 2, 64, 5)
    with pytest.raises(ValueError, match=r"\[5, 2, 64\]"):
        paged._rows(x[:, :128], "x", 2, 64, 5)


def test_sampling_weights_fall_monotonically():
    """Every kept set is a prefix of the order (gap, index) because no weight grows with the gap;
    relative to 2^-x a weight above 2^10 is off by less than 2^-20 and the shift's rounding."""
    e = np.arange(1 << 20, dtype=np.uint64)
    b = np.array(PO.POW2, np.uint64)[(e >> np.uint64(10)).astype(np.int64)]
    w = b - ((b * ((e & np.uint64(1023)) * np.uint64(2839))) >> np.uint64(32))
    assert w[0] == 1 << 31 and np.all(w[1:] <= w[:-1]) and w[-1] >= 1 << 30
    want = 2.0 ** 31 * 2.0 ** (-e.astype(np.float64) / 2 ** 20)
    assert np.max(np.abs(w - want) / want) < 2.0 ** -20


def test_oracle_attention_of_pages_is_the_dense_oracles():
    """Pages in any order give the dense attention of the golden oracle."""
    from oracle import golden_oracle as O
    rng = np.random.default_rng(0)
    H, Hkv, D, P, T = 4, 2, 32, 16, 40
    q = rng.integers(-90, 90, (3, H, D)).astype(np.int8)
    kc, vc = (rng.integers(-128, 128, (Hkv, 48, D)).astype(np.int8) for _ in "kv")
    table = np.array([[2, 0, 3]], np.int32)
    kp, vp = (np.zeros((4, Hkv, P, D), np.int8) for _ in "kv")
    for j, p in enumerate(table[0]):
        kp[p], vp[p] = kc[:, j * P : (j + 1) * P], vc[:, j * P : (j + 1) * P]
    out = np.zeros((3, H, D), np.int8)
    rq = ((1900000000, 34), (1717986918, 37))
    PO.attention(q, kp, vp, table, np.array([T]), np.array([0, 3]), *rq, 15, None, 3, T, out)
    want = O.attention_rows(q.reshape(3, -1), kc, vc, H, Hkv, D, T - 3, *rq[0], *rq[1], 15)
    assert np.array_equal(out.reshape(3, -1), want)
