"""Serving a model over a paged cache: ragged steps, forks and sampled tokens in the model's own path,
against the dense sessions, the golden records and the CPU oracle -- bit for bit."""
from __future__ import annotations

import json

import numpy as np
import pytest

from conftest import GOLDEN
from oracle import golden_oracle as O
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from llaccel_b200 import build  # noqa: E402

build.build()
from llaccel_b200.cuda_backend import LLX_ERR_OOM, LLX_ERR_UNSUPPORTED, CudaModel, CudaServe, LlxError  # noqa: E402

GRAPHS = ["c1_v2", "qwen2_tiny", "qwen3_tiny", "d128_tiny", "fx_v2"]


def prompts(model, rng, n):
    top = model.max_seq * 2 // 3
    return [rng.integers(0, model.vocab, rng.integers(1, top)).tolist() for _ in range(n)]


@pytest.mark.parametrize("graph", GRAPHS)
@pytest.mark.parametrize("page_size,chunk", [(16, None), (64, 5)])
def test_ragged_generation_is_each_sequence_alone(graph, page_size, chunk):
    with CudaModel(GOLDEN / graph) as m:
        rng = np.random.default_rng(len(graph) + page_size)
        P = prompts(m, rng, 7)
        n = min(12, m.max_seq - max(map(len, P)) - 1)
        with CudaServe(m, max_seqs=9, n_pages=9 * (m.max_seq // page_size + 1), page_size=page_size, max_rows=64) as s:
            got = s.generate(P, n, chunk=chunk)
            assert s.usage()[1] == 0
        for p, g in zip(P, got):
            assert g == m.generate(p, n)["generated"]


@pytest.mark.parametrize("graph", ["c1_v2", "qwen3_tiny"])
def test_golden_record_through_pages(graph):
    rec = json.loads((GOLDEN / graph / "golden.json").read_text())
    prompt, want = rec["prompt_tokens"], rec["generated"]
    n = min(len(want), 10)
    with CudaModel(GOLDEN / graph) as m, CudaServe(m, max_seqs=2, n_pages=8, page_size=16) as s:
        assert s.generate([prompt], n) == [want[:n]]


@pytest.mark.parametrize("graph", ["qwen3_tiny", "d128_tiny"])
def test_step_logits_are_the_oracles(graph):
    """Two sequences, one in two chunks, in the same steps; logits of the last rows."""
    with CudaModel(GOLDEN / graph) as m, CudaServe(m, max_seqs=3, n_pages=12, page_size=16) as s:
        rng = np.random.default_rng(3)
        a, b = rng.integers(0, m.vocab, 21), rng.integers(0, m.vocab, 18)
        first = s.step([2, 0], [a[:9], b], with_logits=True)["logits"]
        second = s.step([0, 2], [[5], a[9:]], with_logits=True)["logits"]
        oracle = O.OracleModel(GOLDEN / graph)

        def last(tokens):
            oracle.reset()
            return oracle.run_chunk(oracle.embed[np.asarray(tokens)].astype(np.int64), 0)[-1]

        assert np.array_equal(first[0], last(a[:9])) and np.array_equal(first[1], last(b))
        assert np.array_equal(second[0], last([*b, 5])) and np.array_equal(second[1], last(a))


def test_forks_go_on_alone():
    with CudaModel(GOLDEN / "c1_v2") as m, CudaServe(m, max_seqs=6, n_pages=24, page_size=16) as s:
        rng = np.random.default_rng(4)
        prompt = rng.integers(0, m.vocab, 37).tolist()  # two full pages and a part-filled one
        s.step([0], [prompt])
        used = s.usage()[1]
        s.fork([0, 0], [1, 2])
        s.fork([0], [3], share=False)
        assert s.usage()[1] == used + 2 + 3  # a part page each, and the copy's three
        seqs = {i: list(prompt) for i in range(4)}
        for t in range(6):
            feed = {i: int(rng.integers(0, m.vocab)) for i in seqs}
            got = s.step(list(seqs), [[feed[i]] for i in seqs])["next"]
            for i, g in zip(list(seqs), got):
                seqs[i].append(feed[i])
                assert g == m.generate(seqs[i], 1)["generated"][0], (t, i)
            if t == 2:
                s.free([0])  # the shared pages live on in the children
                del seqs[0]
                s.compact()
        lengths, used = s.usage()
        assert lengths.tolist() == [0, 43, 43, 43, 0, 0] and used <= 9
        s.free([1, 2, 3])
        assert s.usage()[1] == 0


def test_sampled_steps_are_the_samplers():
    with CudaModel(GOLDEN / "c1_v2") as m, CudaServe(m, max_seqs=5, n_pages=20, page_size=16) as s:
        rng = np.random.default_rng(5)
        how = dict(temperature=np.float32([0.002, 0.0, 0.01, 1.0, 0.004]), top_k=np.int32([0, 0, 9, 40, 0]),
                   top_p=np.float32([0.9, 1.0, 1.0, 0.5, 0.99]), min_p=np.float32([0.0, 0.0, 0.1, 0.0, 0.01]))
        feed = [rng.integers(0, m.vocab, k).tolist() for k in (3, 17, 1, 30, 16)]
        for _ in range(4):
            u = rng.random(5)
            got = s.step(range(5), feed, random=u, with_logits=True, **how)
            for i in range(5):
                row = got["logits"][i, : m.vocab]
                want, p = PO.sample(row, float(u[i]), m.E_LOGIT, **{k: v[i].item() for k, v in how.items()})
                assert got["next"][i] == want
                # one division rounded to float32
                assert abs(float(got["prob"][i]) - p) <= p * (np.finfo(np.float32).eps / 2 + 2.0 ** -52)
            feed = [[int(t)] for t in got["next"]]
        a = s.generate([[1, 2, 3], [7]], 5, rng=np.random.default_rng(1), temperature=0.01)
        b = s.generate([[1, 2, 3], [7]], 5, rng=np.random.default_rng(1), temperature=0.01)
        assert a == b and all(len(x) == 5 for x in a)


def test_refusals_change_nothing():
    with CudaModel(GOLDEN / "c1_v2") as m, CudaServe(m, max_seqs=4, n_pages=4, page_size=16, max_rows=60) as s:
        s.step([0, 1], [[1] * 20, [2] * 10])  # three pages
        before = s.usage()[0].tolist()
        with pytest.raises(LlxError) as e:
            s.step([0, 2], [[3] * 20, [4]])
        assert e.value.code == LLX_ERR_OOM
        with pytest.raises(LlxError) as e:
            s.fork([0, 0], [2, 3])
        assert e.value.code == LLX_ERR_OOM
        for bad in (lambda: s.step([0, 0], [[1], [1]]), lambda: s.step([4], [[1]]), lambda: s.step([0], [[m.vocab]]),
                    lambda: s.step([0], [[-1]]), lambda: s.step([0], [[]]), lambda: s.step([0], [[1] * 61]),
                    lambda: s.step([2], [[1] * (m.max_seq + 1)]), lambda: s.step([], []), lambda: s.step([0, 1], [[1]]),
                    lambda: s.step([0], [[1]], top_p=0.5), lambda: s.fork([0], [0]), lambda: s.fork([0, 1], [2, 2]),
                    lambda: s.fork([0, 2], [2, 3]), lambda: s.fork([9], [2]), lambda: s.free([-1]), lambda: s.free([1, 1])):
            with pytest.raises(ValueError):
                bad()
        assert s.usage()[0].tolist() == before
        s.fork([1], [3])  # one page is still there
        follow = s.step([3, 1], [[9], [9]])["next"]
        assert follow[0] == follow[1] == m.generate([2] * 10 + [9], 1)["generated"][0]


def test_unfused_graphs_are_refused():
    for graph, kw in (("c1_v1", {}), ("c1_v2", dict(fuse=False))):
        with CudaModel(GOLDEN / graph, **kw) as m:
            try:
                s = CudaServe(m, max_seqs=2, n_pages=4)
            except LlxError as e:
                assert e.code == LLX_ERR_UNSUPPORTED
            else:  # a v1 graph whose rotations were grouped all the same has to be right
                assert s.generate([[1, 2, 3]], 4) == [m.generate([1, 2, 3], 4)["generated"]]
                s.close()


def test_bad_sizes_are_refused():
    with CudaModel(GOLDEN / "c1_v2") as m:
        for kw in (dict(max_seqs=0, n_pages=4), dict(max_seqs=2, n_pages=0), dict(max_seqs=2, n_pages=4, page_size=24),
                   dict(max_seqs=2, n_pages=4, page_size=512), dict(max_seqs=2, n_pages=4, max_rows=0)):
            with pytest.raises(ValueError):
                CudaServe(m, **kw)
