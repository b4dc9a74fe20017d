"""The paged-serving calls as a program uses them: chained, on a side stream, captured into CUDA graphs that
share a cache, over many sequences, and at addresses past 32 bits.  Whole numbers against the CPU oracle."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from llaccel_b200 import build  # noqa: E402

build.build()
from llaccel_b200 import paged, sampling  # noqa: E402

Q_RQ, K_RQ, SCORE, OUT = (1142505715, 37), (1142505715, 36), (1900000000, 35), (1717986918, 37)


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Steps:
    """Steps of one layer and a head of `V` logits, on the GPU and in the oracle.  The logits of a row are its
    attention output's products with a fixed matrix, formed by the test in exact integers."""

    def __init__(self, rng, H, Hkv, D, P, slots, pages, V=333, norm=True):
        self.rng, self.H, self.Hkv, self.D, self.P, self.V = rng, H, Hkv, D, P, V
        N = slots * pages
        self.o = PO.Pages(np.full((slots, pages), -1, np.int32), np.zeros(slots, np.int32), np.zeros(N, np.int32), P)
        self.k, self.v = (np.zeros((N, Hkv, P, D), np.int8) for _ in "kv")
        self.tk, self.tv = dev(self.k), dev(self.v)
        self.table, self.length, self.refs = dev(self.o.table), dev(self.o.length), dev(self.o.refs)
        ang = np.arange(pages * P)[:, None] * 1e4 ** (-np.arange(D // 2)[None] / (D // 2))
        self.cos, self.sin = (np.round(f(ang) * 16384).astype(np.int16) for f in (np.cos, np.sin))
        self.norm = (rng.integers(3000, 16000, D).astype(np.int16), 343597, 759250125, 28) if norm else None
        self.head = rng.integers(-8, 9, (H * D, V)).astype(np.int32)
        self.t = dict(cos=dev(self.cos), sin=dev(self.sin), norm=(dev(self.norm[0]), *self.norm[1:]) if norm else None,
                      head=dev(self.head.astype(np.float32)), st=torch.zeros(1, dtype=torch.int32, device="cuda"))

    def inputs(self, rows, slots):
        """One step's tensors; their contents may be replaced between replays."""
        R = sum(rows)
        i16 = lambda h: self.rng.integers(-20000, 20000, (R, h, self.D)).astype(np.int16)  # noqa: E731
        x = dict(q=i16(self.H), k=i16(self.Hkv), v=self.rng.integers(-128, 128, (R, self.Hkv, self.D)).astype(np.int8),
                 u=self.rng.random(len(rows)), q_start=np.concatenate([[0], np.cumsum(rows)]).astype(np.int32),
                 slots=np.array(slots, np.int32), counts=np.array(rows, np.int32), top_k=self.rng.integers(0, 60, len(rows)).astype(np.int32),
                 temperature=self.rng.uniform(0.3, 2.0, len(rows)).astype(np.float32),
                 top_p=self.rng.uniform(0.3, 1.0, len(rows)).astype(np.float32))
        return x, {n: dev(a) for n, a in x.items()}

    def enqueue(self, t, max_rows, max_len):
        paged.reserve(self.table, self.length, self.refs, t["slots"], t["counts"], self.P, status=self.t["st"])
        q8 = paged.append(t["q"], t["k"], t["v"], self.tk, self.tv, self.table, self.length, t["q_start"], self.t["cos"],
                          self.t["sin"], Q_RQ, K_RQ, q_norm=self.t["norm"], k_norm=self.t["norm"], seqs=t["slots"],
                          status=self.t["st"])
        o = paged.attention(q8, self.tk, self.tv, self.table, self.length, t["q_start"], SCORE, OUT, max_rows=max_rows,
                            max_len=max_len, seqs=t["slots"], status=self.t["st"])
        # whole numbers below 2^24: fp32 products are exact in any order
        last = o.flatten(1)[(t["q_start"][1:] - 1).long()].float()
        logits = (last @ self.t["head"]).clamp(-32768, 32767).to(torch.int16)
        return q8, o, logits, sampling.sample(logits, t["u"], exponent=-11, temperature=t["temperature"], top_k=t["top_k"], top_p=t["top_p"])

    def expect(self, x, max_rows, max_len):
        assert self.o.reserve(x["slots"].tolist(), x["counts"].tolist()) == 0
        R = len(x["q"])
        q8, o = (np.zeros((R, self.H, self.D), np.int8) for _ in "qo")
        PO.append(x["q"], x["k"], x["v"], self.k, self.v, self.o.table, self.o.length, x["q_start"], self.cos, self.sin, Q_RQ, K_RQ,
                  self.norm, self.norm, x["slots"], q8)
        PO.attention(q8, self.k, self.v, self.o.table, self.o.length, x["q_start"], SCORE, OUT, 15, x["slots"], max_rows, max_len, o)
        last = o.reshape(R, -1)[x["q_start"][1:] - 1].astype(np.int64)
        assert np.abs(last).max() * 8 * self.H * self.D < 2 ** 24
        logits = np.clip(last @ self.head, -32768, 32767).astype(np.int16)
        token = [PO.sample(logits[i], float(x["u"][i]), -11, **{n: x[n][i].item() for n in ("temperature", "top_k", "top_p")})[0]
                 for i in range(len(x["slots"]))]
        return q8, o, logits, token

    def same(self, got, want):
        for name, g, w in zip(("q8", "attention", "logits"), got, want):
            assert np.array_equal(g.cpu().numpy(), w), name
        assert got[3][0].tolist() == want[3]
        assert np.array_equal(self.tk.cpu().numpy(), self.k) and np.array_equal(self.tv.cpu().numpy(), self.v)
        assert np.array_equal(self.length.cpu().numpy(), self.o.length)
        assert np.array_equal(self.table.cpu().numpy(), self.o.table) and np.array_equal(self.refs.cpu().numpy(), self.o.refs)
        assert int(self.t["st"].item()) == 0


@pytest.mark.parametrize("H,Hkv,D", [(8, 2, 64), (4, 2, 128), (4, 1, 32)])
def test_steps_on_a_side_stream(H, Hkv, D):
    """Prompts, then single tokens, then both kinds in one launch, without a wait in between."""
    s = Steps(np.random.default_rng(D), H, Hkv, D, 16, 6, 8)
    side = torch.cuda.Stream()
    plan = [([5, 33, 1], [4, 0, 2]), ([1, 1, 1], [0, 2, 4]), ([1, 40, 1], [2, 5, 0]), ([1, 1], [5, 4])]
    steps = [s.inputs(*p) for p in plan]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [s.enqueue(t, 40, 128) for _, t in steps]
    side.synchronize()
    want = [s.expect(x, 40, 128) for x, _ in steps]
    for g, w in zip(got, want):
        s.same(g, w)


@pytest.mark.parametrize("D", [64, 128])
def test_two_graphs_of_one_cache(D):
    """A graph of a chunk step and one of a token step take turns over the same pages, with new inputs each time."""
    s = Steps(np.random.default_rng(D), 4, 2, D, 16, 4, 16)
    kinds = {"chunk": ([20, 1, 7], [3, 0, 1]), "token": ([1, 1, 1], [1, 3, 0])}
    held = {n: s.inputs(*p)[1] for n, p in kinds.items()}
    warm = Steps(np.random.default_rng(0), 4, 2, D, 16, 4, 16)
    for n, p in kinds.items():  # a first call outside any capture
        warm.enqueue(warm.inputs(*p)[1], 20, 256)
    torch.cuda.synchronize()
    graphs, outs = {}, {}
    for n in kinds:
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[n]):
            outs[n] = s.enqueue(held[n], 20, 256)
    assert int(s.length.sum()) == 0  # capture runs nothing
    for n in ("chunk", "token", "token", "chunk", "token"):
        x, t = s.inputs(*kinds[n])
        for name, a in t.items():
            held[n][name].copy_(a)
        graphs[n].replay()
        torch.cuda.synchronize()
        s.same(outs[n], s.expect(x, 20, 256))


def test_two_streams_with_a_cache_each():
    steps = [Steps(np.random.default_rng(i), 8, 4, 64, 32, 3, 8) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in steps]
    plan = [([60, 9, 31], [0, 1, 2])] + [([1, 1, 1], [2, 0, 1])] * 4
    ins = [[s.inputs(*p) for p in plan] for s in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for j in range(len(plan)):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                got[i].append(s.enqueue(ins[i][j][1], 60, 256))
    torch.cuda.synchronize()
    for i, s in enumerate(steps):
        want = [s.expect(x, 60, 256) for x, _ in ins[i]]
        for g, w in zip(got[i], want):
            s.same(g, w)


@pytest.mark.parametrize("n", [33, 1025, 1100])
@pytest.mark.parametrize("D", [64, 128, 16])
def test_many_sequences(n, D):
    """Searches over more than 32 and 1024 starts, empty sequences among them."""
    rng = np.random.default_rng(n)
    s = Steps(rng, 2, 1, D, 16, n, 1, V=17, norm=False)
    rows = rng.integers(0, 4, n)
    rows[[0, 31, -1]] = 0, 5, 2
    x, t = s.inputs(rows.tolist(), rng.permutation(n).tolist())
    assert s.o.reserve(x["slots"].tolist(), x["counts"].tolist()) == 0
    R = len(x["q"])
    q8, o = (np.zeros((R, 2, D), np.int8) for _ in "qo")
    PO.append(x["q"], x["k"], x["v"], s.k, s.v, s.o.table, s.o.length, x["q_start"], s.cos, s.sin, Q_RQ, K_RQ, None, None, x["slots"], q8)
    PO.attention(q8, s.k, s.v, s.o.table, s.o.length, x["q_start"], SCORE, OUT, 15, x["slots"], 5, 16, o)
    paged.reserve(s.table, s.length, s.refs, t["slots"], t["counts"], 16, status=s.t["st"])
    g8 = paged.append(t["q"], t["k"], t["v"], s.tk, s.tv, s.table, s.length, t["q_start"], s.t["cos"], s.t["sin"], Q_RQ, K_RQ,
                      seqs=t["slots"], status=s.t["st"])
    # bounds wider than the launch's rows are no other than its rows
    for most in (5, 1 << 40):
        g = paged.attention(g8, s.tk, s.tv, s.table, s.length, t["q_start"], SCORE, OUT, max_rows=most, max_len=16, seqs=t["slots"],
                            status=s.t["st"])
        assert np.array_equal(g.cpu().numpy(), o)
    assert np.array_equal(g8.cpu().numpy(), q8) and np.array_equal(s.tk.cpu().numpy(), s.k)
    assert int(s.t["st"].item()) == 0


def test_one_slot_read_by_many_sequences():
    """Attention only reads: a slot may be listed often, here by more sequences than a grid axis holds."""
    rng = np.random.default_rng(3)
    H, D, P, n = 2, 64, 16, 65600
    k, v = (rng.integers(-100, 101, (8, 1, P, D)).astype(np.int8) for _ in "kv")
    table, length = np.arange(8, dtype=np.int32).reshape(4, 2), np.array([20, 32, 1, 16], np.int32)
    q = rng.integers(-100, 101, (64, H, D)).astype(np.int8)
    want = np.zeros((64, H, D), np.int8)
    PO.attention(q, k, v, table, length, np.arange(65, dtype=np.int32), SCORE, OUT, 15, np.arange(64, dtype=np.int32) % 4, 1, 32, want)
    got = paged.attention(dev(q).repeat(n // 64, 1, 1), dev(k), dev(v), dev(table), dev(length), dev(np.arange(n + 1, dtype=np.int32)),
                          SCORE, OUT, max_rows=1, max_len=32, seqs=dev(np.arange(n, dtype=np.int32) % 4))
    assert torch.equal(got, dev(want).repeat(n // 64, 1, 1))


@pytest.mark.parametrize("D", [64, 128, 32])
def test_pages_past_32_bits(D):
    """The same steps in a small cache and with their pages at the end of one of 4.5 GB."""
    rng = np.random.default_rng(D)
    s = Steps(rng, 4, 1, D, 64, 3, 4)
    N = (9 << 29) // (64 * D)
    big = [torch.empty((N, 1, 64, D), dtype=torch.int8, device="cuda") for _ in "kv"]
    for rows, slots in (([70, 9, 1], [0, 1, 2]), ([1, 1, 1], [2, 1, 0]), ([1, 50, 1], [0, 2, 1])):
        x, t = s.inputs(rows, slots)
        got = s.enqueue(t, 70, 256)
        s.same(got, s.expect(x, 70, 256))
        table = torch.where(s.table >= 0, N - 1 - s.table, s.table)
        q8 = paged.append(t["q"], t["k"], t["v"], *big, table, s.length, t["q_start"], s.t["cos"], s.t["sin"], Q_RQ, K_RQ,
                          q_norm=s.t["norm"], k_norm=s.t["norm"], seqs=t["slots"], status=s.t["st"])
        o = paged.attention(q8, *big, table, s.length, t["q_start"], SCORE, OUT, max_rows=70, max_len=256, seqs=t["slots"],
                            status=s.t["st"])
        assert torch.equal(q8, got[0]) and torch.equal(o, got[1])
    # a copied sequence, compaction to the front, and the attention of what lies there then
    refs = torch.zeros(N, dtype=torch.int32, device="cuda")
    wide = torch.full((4, 4), -1, dtype=torch.int32, device="cuda")
    wide[:3] = table
    refs[table[table >= 0].long()] = 1
    length = torch.zeros(4, dtype=torch.int32, device="cuda")
    length[:3] = s.length
    paged.fork(*big, wide, length, refs, dev(np.array([0], np.int32)), dev(np.array([3], np.int32)), share=False, status=s.t["st"])
    paged.compact(*big, wide, refs, status=s.t["st"])
    assert int(wide.max()) < 16 and int(s.t["st"].item()) == 0
    o2 = paged.attention(q8, *big, wide, length, t["q_start"], SCORE, OUT, max_rows=70, max_len=256, seqs=t["slots"])
    assert torch.equal(o2, o)
    copied = t["slots"].clone()
    copied[copied == 0] = 3
    assert torch.equal(paged.attention(q8, *big, wide, length, t["q_start"], SCORE, OUT, max_rows=70, max_len=256, seqs=copied), o)


def test_chunk_over_a_long_context():
    """More than 65536 keys under a chunk: sums of weights and of weighted values that need all of 32 bits."""
    rng = np.random.default_rng(5)
    H, D, P, T = 4, 64, 256, 70001
    n = -(-T // P)
    table = rng.permutation(n).astype(np.int32)[None]
    q = rng.integers(-128, 128, (10, H, D)).astype(np.int8)
    for flat in (False, True):
        k = np.full((n, 1, P, D), 3, np.int8) if flat else rng.integers(-128, 128, (n, 1, P, D)).astype(np.int8)
        v = np.full((n, 1, P, D), -128, np.int8) if flat else rng.integers(-128, 128, (n, 1, P, D)).astype(np.int8)
        want = np.zeros_like(q)
        rq = (1 << 30, 30) if flat else SCORE
        args = (table, np.array([T], np.int32), np.array([0, 10], np.int32))
        PO.attention(q, k, v, *args, rq, (1717986918, 36), 15, None, 10, T, want)
        got = paged.attention(dev(q), dev(k), dev(v), *map(dev, args), rq, (1717986918, 36), max_rows=10, max_len=T)
        assert np.array_equal(got.cpu().numpy(), want)


def test_numbers_of_other_types_and_refusals():
    """numpy numbers and lists are looked at in Python: the same results, and the same words for what is wrong."""
    s = Steps(np.random.default_rng(1), 4, 2, 64, 16, 2, 4)
    x, t = s.inputs([9, 1], [0, 1])
    paged.reserve(s.table, s.length, s.refs, t["slots"], t["counts"], 16, status=s.t["st"])
    args = [t["q"], t["k"], t["v"], s.tk, s.tv, s.table, s.length, t["q_start"], s.t["cos"], s.t["sin"]]
    norm = (s.t["norm"][0], *(np.int64(n) for n in s.t["norm"][1:]))
    q8 = [paged.append(*args, Q_RQ, K_RQ, q_norm=s.t["norm"], k_norm=s.t["norm"], seqs=t["slots"], status=s.t["st"]),
          paged.append(*args, list(Q_RQ), np.array(K_RQ), q_norm=norm, k_norm=list(norm), seqs=t["slots"])]
    assert torch.equal(*q8) and int(q8[0].abs().max()) > 0
    args = [q8[0], s.tk, s.tv, s.table, s.length, t["q_start"]]
    o = [paged.attention(*args, SCORE, OUT, max_rows=9, max_len=64, seqs=t["slots"], status=s.t["st"]),
         paged.attention(*args, list(SCORE), np.array(OUT), prob_bits=np.int32(15), max_rows=np.int64(9), max_len=np.int64(64),
                         seqs=t["slots"])]
    assert torch.equal(*o) and int(o[0].abs().max()) > 0
    for i, wrong, words in ((0, q8[0].short(), "q8 must be torch.int8"), (1, s.tk[:, :, :8], "alike"), (2, s.tv.cpu(), "must be on cuda"),
                            (3, s.table.t(), "dense rows"), (4, s.length[:1], "entry per slot"), (5, t["q_start"][::2], "dense vector"),
                            (0, q8[0][..., ::2], "heads of 32"), (0, q8[0].transpose(0, 1), "must be|dense")):
        bad = list(args)
        bad[i] = wrong
        with pytest.raises(ValueError, match=words):
            paged.attention(*bad, SCORE, OUT, max_rows=9, max_len=64, seqs=t["slots"], out=torch.zeros_like(q8[0]))
    with pytest.raises(ValueError, match="prob_bits"):
        paged.attention(*args, SCORE, OUT, prob_bits=9, max_rows=9, max_len=64, seqs=t["slots"])
    with pytest.raises(ValueError, match="outside M"):
        paged.attention(*args, (-1, 3), OUT, max_rows=9, max_len=64, seqs=t["slots"])
    assert int(s.t["st"].item()) == 0
