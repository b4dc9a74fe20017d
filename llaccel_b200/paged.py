"""Serving ragged batches from a paged int8 KV cache: the calls of include/llx.h on torch CUDA
tensors.

A layer's cache is two int8 tensors `[n_pages, n_kv_heads, page_size, head_dim]`.  Position t of
the sequence in slot s lies in page `table[s, t // page_size]`, row `t % page_size`; `length[s]`
counts its positions.  A launch brings new rows: sequence i has the rows
`q_start[i] <= r < q_start[i + 1]`, the newest positions of slot `seqs[i]` (default: slot i), from
one row (a decode step) to a whole prompt.  A step of a model is

    reserve(table, length, refs, slots, counts, page_size)           # pages and positions for the new rows
    q8 = append(q, k, v, k_pages, v_pages, table, length, q_start, ...)   # per layer
    o8 = attention(q8, k_pages, v_pages, table, length, q_start, ...)     # per layer

and `llaccel_b200.sampling.sample` picks the next tokens.  `fork` lets answers share their
prompt's pages, `free` gives a sequence's pages back, `compact` moves the live pages to the front.

Every call enqueues on torch's current stream of its tensors' device, allocates only what it
returns (and, for the page calls, scratch) from torch's allocator, and can be captured into a CUDA
graph.  What the host can check raises ValueError; what only the device can see (page ids,
lengths) is skipped and noted in `status`, an int32 tensor of one value that `check` reads.
Calls that change the same cache, table or counts have to be ordered by the caller, as on one
stream.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import importlib.util
import struct
from pathlib import Path

import torch

from .cuda_backend import _check as _check_code
from .cuda_backend import load_library

STATUS = {1: "a position's page id lies outside the cache",
          2: "a position below 0, or beyond the rotation tables or the page table",
          4: "a sequence with more rows or positions than the call was told",
          8: "too few free pages",
          16: "a slot outside the table, listed twice, or both parent and child",
          32: "new positions would fall into a page that other sequences share",
          64: "a bounded wait of a kernel ran out: the call's results are void"}

_APPEND = struct.Struct("=42q")
_ATTENTION = struct.Struct("=30q")
_PAGES = struct.Struct("=24q")


_I8, _I16, _I32 = torch.int8, torch.int16, torch.int32
_stream = torch._C._cuda_getCurrentRawStream


_lib = _calls = None


def _load():
    """libllx.so, and the binding that packs a call's tensors (torch_calls.cpp) with the calls' addresses."""
    global _lib, _calls, _append_at, _attention_at
    _lib = load_library()
    path = Path(__file__).resolve().parent / "_lib" / "torch_calls.so"
    if not path.exists():
        raise RuntimeError(f"binding missing: {path} (build it with `python -m llaccel_b200.build`)")
    spec = importlib.util.spec_from_file_location("torch_calls", path)
    _calls = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(_calls)
    _append_at, _attention_at = (ctypes.cast(f, ctypes.c_void_p).value for f in (_lib.llx_paged_append, _lib.llx_paged_attention))
    return _lib


def _refuse(dev: int, dtype, **tensors) -> None:
    """Says which tensor (None allowed) is not on CUDA device `dev` or has another type."""
    for name, t in tensors.items():
        if t is not None and t.dtype is not dtype:
            raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{name} must be on cuda:{dev}, not {t.device}")


def _cuda(t, name: str) -> int:
    dev = t.get_device()
    if dev < 0:
        raise ValueError(f"{name} must be a CUDA tensor: there is no CPU path")
    return dev


def _rows(t, name: str, heads: int, dim: int, rows: int) -> int:
    """Row stride (in elements) of a [rows, heads, dim] tensor whose rows are dense."""
    if t.shape != (rows, heads, dim):
        raise ValueError(f"{name} must be [{rows}, {heads}, {dim}], not {list(t.shape)}")
    s = t.stride()
    if (s[2] != 1 or s[1] != dim) and rows and ((dim > 1 and s[2] != 1) or (heads > 1 and s[1] != dim)):
        raise ValueError(f"{name}: the heads of a row must be dense")
    return s[0] if rows > 1 else heads * dim


def _pool(k, v) -> tuple:
    """(layer stride, page stride, layers, pages, heads, page size, head dim) of k and v pages."""
    s, n = k.stride(), k.shape
    if n != v.shape or s != v.stride() or len(n) not in (4, 5):
        raise ValueError("k_pages and v_pages must be alike: [n_pages, n_kv_heads, page_size, head_dim], "
                         "page calls also with a layer axis in front")
    if s[-1] != 1 or s[-2] != n[-1] or s[-3] != n[-1] * n[-2]:
        raise ValueError("the heads, rows and channels of a page must be dense")
    return (s[0] if len(n) == 5 else 0, s[-4], n[0] if len(n) == 5 else 1, *n[-4:])


def _table(table, length) -> tuple:
    n, s = table.shape, table.stride()
    if len(n) != 2 or (n[1] > 1 and s[1] != 1):
        raise ValueError("table must be [slots, pages] with dense rows")
    if length is not None and (length.shape != (n[0],) or (n[0] > 1 and length.stride(0) != 1)):
        raise ValueError("length must be a dense vector with an entry per slot of the table")
    return table.data_ptr(), s[0] if n[0] > 1 else n[1], n[0], n[1]


def _vector(t, name: str, n: int | None = None) -> int:
    m = t.shape
    if len(m) != 1 or (n is not None and m[0] != n) or (m[0] > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a dense vector" + (f" of {n} values" if n is not None else ""))
    return t.data_ptr()


def _launch(q_start, seqs) -> tuple:
    n = q_start.shape[0] - 1
    if n < 0:
        raise ValueError("q_start needs an entry per sequence and one more")
    _vector(q_start, "q_start")
    return q_start.data_ptr(), _vector(seqs, "seqs", n) if seqs is not None else 0, n


def _need_slots(seqs, n: int, table) -> None:
    if seqs is None and n > table.shape[0]:
        raise ValueError(f"{n} sequences, but the table has {table.shape[0]} slots")


def _norm(x, name: str, dev: int, dim: int) -> tuple:
    if x is None:
        return 0, 0, 0, 0
    gamma, eps, C, sh = x
    if gamma.dtype is not _I16 or gamma.get_device() != dev:
        _refuse(dev, _I16, **{name: gamma})
    return _vector(gamma, name, dim), eps, C, sh


def append(q, k, v, k_pages, v_pages, table, length, q_start, cos, sin, q_rq, k_rq, *, q_norm=None, k_norm=None,
           seqs=None, out=None, status=None):
    """Queries, keys and values of a launch on their way into a layer's cache.

    q `[rows, n_heads, head_dim]` and k `[rows, n_kv_heads, head_dim]` int16, v int8 like k: per
    query and key head an RMSNorm (`q_norm` / `k_norm` = (gamma int16 [head_dim], eps_t, C,
    sh_post), or None), the rotation at the row's position (`cos`, `sin` int16 Q1.14
    [positions, head_dim / 2]) and requantization by `q_rq` / `k_rq` = (M, S).  Keys and values go
    to the pages of their positions; a slot may be listed once.  Returns the int8 queries, in `out` if given; rows behind
    `q_start[-1]` are left as they were."""
    lib = _lib or _load()
    if out is None:
        out = torch.zeros(q.shape, dtype=_I8, device=q.device)
    code = _calls.append(_append_at, q, k, v, k_pages, v_pages, table, length, q_start, cos, sin, q_rq, k_rq, q_norm, k_norm, seqs,
                         out, status)
    if code is None:  # something unusual, or wrong
        code = _append_checked(q, k, v, k_pages, v_pages, table, length, q_start, cos, sin, q_rq, k_rq, q_norm, k_norm, seqs, out,
                               status)
    if code:
        _check_code(lib, code)
    return out


def _append_checked(q, k, v, k_pages, v_pages, table, length, q_start, cos, sin, q_rq, k_rq, q_norm, k_norm, seqs, out, status) -> int:
    dev = _cuda(q, "q")
    _refuse(dev, _I16, q=q, k=k, cos=cos, sin=sin)
    _refuse(dev, _I8, v=v, k_pages=k_pages, v_pages=v_pages, out=out)
    _refuse(dev, _I32, table=table, length=length, q_start=q_start, seqs=seqs, status=status)
    if len(q.shape) != 3 or len(k_pages.shape) != 4:
        raise ValueError("q must be [rows, n_heads, head_dim], k_pages [n_pages, n_kv_heads, page_size, head_dim]")
    R, H, D = q.shape
    _, page_stride, _, n_pages, Hkv, P, Dk = _pool(k_pages, v_pages)
    if D != Dk:
        raise ValueError(f"q has heads of {D}, the cache of {Dk}")
    rot = cos.shape
    if len(rot) != 2 or rot != sin.shape or rot[1] != D // 2 or not (cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError(f"cos and sin must be dense [positions, {D // 2}]")
    starts, slots, n = _launch(q_start, seqs)
    _need_slots(seqs, n, table)
    qg, qe, qC, qsh = _norm(q_norm, "q_norm", dev, D)
    kg, ke, kC, ksh = _norm(k_norm, "k_norm", dev, D)
    args = _APPEND.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _rows(q, "q", H, D, R),
                        _rows(k, "k", Hkv, D, R), _rows(v, "v", Hkv, D, R), _rows(out, "out", H, D, R), R, H, Hkv, D, qg, kg,
                        qe, qC, qsh, ke, kC, ksh, cos.data_ptr(), sin.data_ptr(), rot[0], *q_rq, *k_rq,
                        k_pages.data_ptr(), v_pages.data_ptr(), page_stride, n_pages, P, *_table(table, length),
                        length.data_ptr(), starts, slots, n, status.data_ptr() if status is not None else 0, dev)
    # a launch without rows is nothing to do, and its tensors have no addresses to check
    return (_lib or _load()).llx_paged_append(args, _stream(dev)) if R else 0


def attention(q8, k_pages, v_pages, table, length, q_start, score_rq, out_rq, *, prob_bits=15, max_rows, max_len,
              seqs=None, out=None, status=None):
    """Causal attention of a launch's rows over their sequences' pages, int8 `[rows, n_heads,
    head_dim]` to the same shape (in `out` if given).

    `score_rq` = (Ms, Ss), `out_rq` = (Mo, So) and `prob_bits` are the graph's attention constants.
    `max_rows` and `max_len` bound the new rows and the length of every sequence that has rows: what is
    beyond them is not computed.  They also size the launch and choose its kernel, so bounds near the
    true ones are faster.  Keys whose page id lies outside the cache count as absent; a row without keys
    gets zeros."""
    lib = _lib or _load()
    if out is None:
        out = torch.zeros(q8.shape, dtype=_I8, device=q8.device)
    code = _calls.attention(_attention_at, q8, k_pages, v_pages, table, length, q_start, score_rq, out_rq, prob_bits, max_rows, max_len,
                            seqs, out, status)
    if code is None:  # something unusual, or wrong
        code = _attention_checked(q8, k_pages, v_pages, table, length, q_start, score_rq, out_rq, prob_bits, max_rows, max_len, seqs,
                                  out, status)
    if code:
        _check_code(lib, code)
    return out


def _attention_checked(q8, k_pages, v_pages, table, length, q_start, score_rq, out_rq, prob_bits, max_rows, max_len, seqs, out,
                       status) -> int:
    dev = _cuda(q8, "q8")
    _refuse(dev, _I8, q8=q8, k_pages=k_pages, v_pages=v_pages, out=out)
    _refuse(dev, _I32, table=table, length=length, q_start=q_start, seqs=seqs, status=status)
    if len(q8.shape) != 3 or len(k_pages.shape) != 4:
        raise ValueError("q8 must be [rows, n_heads, head_dim], k_pages [n_pages, n_kv_heads, page_size, head_dim]")
    R, H, D = q8.shape
    _, page_stride, _, n_pages, Hkv, P, Dk = _pool(k_pages, v_pages)
    if D != Dk:
        raise ValueError(f"q8 has heads of {D}, the cache of {Dk}")
    starts, slots, n = _launch(q_start, seqs)
    _need_slots(seqs, n, table)
    args = _ATTENTION.pack(q8.data_ptr(), out.data_ptr(), _rows(q8, "q8", H, D, R), _rows(out, "out", H, D, R), R, H, Hkv, D,
                           k_pages.data_ptr(), v_pages.data_ptr(), page_stride, n_pages, P, *_table(table, length),
                           length.data_ptr(), starts, slots, n, max_rows, max_len, *score_rq, *out_rq, prob_bits,
                           status.data_ptr() if status is not None else 0, dev)
    # a launch without rows is nothing to do, and its tensors have no addresses to check
    return (_lib or _load()).llx_paged_attention(args, _stream(dev)) if R else 0


def _page_call(name, pool, table, length, refs, list_a, list_b, share, new_table, new_refs, status) -> None:
    k, v, shape = pool
    dev = _cuda(table, "table")
    _refuse(dev, _I32, table=table, length=length, refs=refs, list_a=list_a, list_b=list_b, new_table=new_table,
            new_refs=new_refs, status=status)
    _refuse(dev, _I8, k_pages=k, v_pages=v)
    layer_stride, page_stride, L, n_pages, Hkv, P, D = shape
    refs_ptr = _vector(refs, "refs", n_pages)
    n = list_a.shape[0] if list_a is not None else 0
    a = _vector(list_a, "the first list") if list_a is not None else 0
    b = _vector(list_b, "the second list", n) if list_b is not None else 0
    scratch = torch.empty(3 * n_pages + 4, dtype=_I32, device=table.device)
    args = _PAGES.pack(k.data_ptr() if k is not None else 0, v.data_ptr() if v is not None else 0, layer_stride, page_stride,
                       L, n_pages, Hkv, P, D, *_table(table, length), length.data_ptr() if length is not None else 0,
                       refs_ptr, a, b, n, int(share), new_table.data_ptr() if new_table is not None else 0,
                       new_refs.data_ptr() if new_refs is not None else 0, scratch.data_ptr(),
                       status.data_ptr() if status is not None else 0, dev)
    lib = _lib or _load()
    code = getattr(lib, name)(args, _stream(dev))
    if code:
        _check_code(lib, code)


def _no_pool(refs, page_size):
    return None, None, (0, 16 * page_size, 1, refs.shape[0], 1, page_size, 16)


def reserve(table, length, refs, slots, counts, page_size, *, status=None) -> None:
    """`counts[i]` new positions for slot `slots[i]`: takes the pages they need (the free ones with
    the lowest ids) and adds them to `length`.  All or nothing; a slot may be listed once."""
    _page_call("llx_pages_reserve", _no_pool(refs, page_size), table, length, refs, slots, counts, 0, None, None, status)


def free(table, length, refs, slots, *, status=None) -> None:
    """Gives the slots' pages back and sets their lengths to 0.  Slots outside the table are skipped and
    noted in `status`, the others freed all the same."""
    _page_call("llx_pages_free", _no_pool(refs, 16), table, length, refs, slots, None, 0, None, None, status)


def fork(k_pages, v_pages, table, length, refs, parents, children, *, share=True, status=None) -> None:
    """Slot `children[i]` becomes a copy of slot `parents[i]`; its old pages are released first.

    With `share` full pages are shared and a part-filled last page is copied; without, every page
    is copied.  Pages may carry a layer axis in front, `[n_layers, n_pages, ...]`: one id stands for
    a page of every layer.  A parent may be listed often, a child once, and no child is a parent.
    All or nothing."""
    _page_call("llx_pages_fork", (k_pages, v_pages, _pool(k_pages, v_pages)), table, length, refs, parents, children, share,
               None, None, status)


def compact(k_pages, v_pages, table, refs, *, out=None, status=None):
    """Brings the live pages (refs > 0) to the lowest ids and renames them in the table: of n live pages
    those with an id from n on move, in order, into the free ids below n, the others stay.  `out` = (table, refs) receives the renamed ones; default: in place.  Returns them."""
    new_table, new_refs = (table, refs) if out is None else out
    if new_table.shape != table.shape or new_table.stride() != table.stride():
        raise ValueError("the new table must be laid out like the table")
    _vector(new_refs, "new refs", refs.shape[0])
    _page_call("llx_pages_compact", (k_pages, v_pages, _pool(k_pages, v_pages)), table, None, refs, None, None, 0, new_table,
               new_refs, status)
    return new_table, new_refs


def check(status) -> None:
    """Raises ValueError if a call noted something in `status` (waits for the stream), and clears it."""
    code = int(status.item())
    if code:
        status.zero_()
        raise ValueError("; ".join(t for bit, t in STATUS.items() if code & bit))
