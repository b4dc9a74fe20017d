"""What is closed before a model's weights are freed, on the CPU with a library that notes its calls."""
from __future__ import annotations

import gc

import pytest

from llaccel_b200 import cuda_backend as cb


class Library:
    def __init__(self):
        self.calls, self.last = [], 0

    def __getattr__(self, name):
        def call(*args):
            if name in ("llx_model_load", "llx_session_create", "llx_serve_create"):
                self.last += 1
                args[-1]._obj.value = self.last
                self.calls.append((name, self.last))
            elif name.endswith("destroy"):
                self.calls.append((name, args[0].value))
            return 0
        return call

    def destroyed(self):
        return [c for c in self.calls if c[0].endswith("destroy")]


@pytest.fixture
def lib(monkeypatch):
    lib = Library()
    monkeypatch.setattr(cb, "load_library", lambda: lib)
    return lib


def test_a_closed_model_closes_its_servers_first(lib):
    m = cb.CudaModel("x")
    a, b = cb.CudaServe(m, max_seqs=1, n_pages=1), cb.CudaServe(m, max_seqs=1, n_pages=1)
    a.close()
    m.close()
    assert lib.destroyed() == [("llx_serve_destroy", 3), ("llx_serve_destroy", 4), ("llx_session_destroy", 2), ("llx_model_destroy", 1)]
    b.close()
    m.close()
    for use in (lambda: b.step([0], [[1]]), lambda: b.free([0]), lambda: b.fork([0], [1]), b.compact, b.usage):
        with pytest.raises(ValueError, match="closed"):
            use()
    del a, b, m
    gc.collect()
    assert len(lib.destroyed()) == 4


def test_a_closed_model_closes_the_sessions_that_share_its_weights(lib):
    m = cb.CudaModel("x")
    lane = cb.CudaModel("x", share=m)
    s = cb.CudaServe(lane, max_seqs=1, n_pages=1)
    m.close()
    names = [n for n, _ in lib.destroyed()]
    assert names.index("llx_model_destroy") == 3 and sorted(names[:3]) == ["llx_serve_destroy", "llx_session_destroy", "llx_session_destroy"]
    lane.close()
    s.close()
    assert len(lib.destroyed()) == 4
    with pytest.raises(ValueError, match="closed"):
        cb.CudaModel("x", share=m)


def test_a_server_outlives_nothing_it_needs(lib):
    s = cb.CudaServe(cb.CudaModel("x"), max_seqs=1, n_pages=1)
    gc.collect()
    assert lib.destroyed() == []
    del s
    gc.collect()
    assert [n for n, _ in lib.destroyed()] == ["llx_serve_destroy", "llx_session_destroy", "llx_model_destroy"]
