"""The paged-serving calls on the GPU against the CPU oracle: whole numbers, so equality."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import golden_oracle as O
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from llaccel_b200 import build  # noqa: E402

build.build()
from llaccel_b200 import paged, sampling  # noqa: E402


def dev(x, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(x))
    return (t.to(dtype) if dtype else t).cuda()


def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def launch(rng, rows, lens, P, *, slots=None, spare=3, extra_pages=0):
    """Shuffled pages for sequences of `lens` positions, with `rows` new rows each."""
    need = [-(-max(n, 0) // P) for n in lens]
    S = (max(slots) + 1 if slots else len(lens)) + 1
    W = max(max(need), 1) + extra_pages
    N = sum(need) + spare
    ids = rng.permutation(N)
    table = np.full((S, W), -1, np.int32)
    length = np.zeros(S, np.int32)
    at = 0
    for i, n in enumerate(lens):
        s = slots[i] if slots else i
        table[s, : need[i]] = ids[at : at + need[i]]
        length[s] = n
        at += need[i]
    q_start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    return dict(table=table, length=length, q_start=q_start, N=N, seqs=None if slots is None else np.array(slots, np.int32))


# ---- append -------------------------------------------------------------------------------
def append_case(rng, H, Hkv, D, P, rows, lens, norm, *, pad=0, slots=None, positions=None, sd=6000.0, edit=None):
    L = launch(rng, rows, lens, P, slots=slots)
    R = int(L["q_start"][-1]) + pad
    i16 = lambda shape, s: np.clip(np.round(rng.normal(0, s, shape)), -32768, 32767).astype(np.int16)  # noqa: E731
    q, k = i16((R, H, D), sd), i16((R, Hkv, D), sd)
    v = rng.integers(-128, 128, (R, Hkv, D)).astype(np.int8)
    half, n_pos = D // 2, positions or max(max(lens), 1)
    ang = np.arange(n_pos)[:, None] * 1e4 ** (-np.arange(half)[None] / half)
    cos, sin = (np.round(f(ang) * 16384).astype(np.int16) for f in (np.cos, np.sin))
    qn = (i16((D,), 3000) + 9000, 343597, 759250125, 28) if norm else None
    kn = (i16((D,), 3000) + 9000, 68719, 268435456, 26) if norm else None
    kp, vp = (rng.integers(-128, 128, (L["N"], Hkv, P, D)).astype(np.int8) for _ in "kv")
    out = rng.integers(-128, 128, (R, H, D)).astype(np.int8)
    if edit:
        edit(L, q, k)
    want = [x.copy() for x in (out, kp, vp)]
    PO.append(q, k, v, want[1], want[2], L["table"], L["length"], L["q_start"], cos, sin, (1142505715, 37), (2128689551, 38), qn,
              kn, L["seqs"], want[0])
    got = [dev(x) for x in (out, kp, vp)]
    st = status()
    norms = [None if n is None else (dev(n[0]), *n[1:]) for n in (qn, kn)]
    paged.append(dev(q), dev(k), dev(v), got[1], got[2], dev(L["table"]), dev(L["length"]), dev(L["q_start"]), dev(cos), dev(sin),
                 (1142505715, 37), (2128689551, 38), q_norm=norms[0], k_norm=norms[1],
                 seqs=None if slots is None else dev(L["seqs"]), out=got[0], status=st)
    for g, w, name in zip(got, want, ("q8", "k pages", "v pages")):
        assert np.array_equal(g.cpu().numpy(), w), name
    return int(st.item())


@pytest.mark.parametrize("H,Hkv,D", [(16, 8, 128), (14, 2, 64), (4, 2, 32), (3, 1, 16), (2, 2, 256), (5, 5, 80), (1, 1, 48)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(H, Hkv, D, norm):
    rng = np.random.default_rng(H * D + norm)
    assert append_case(rng, H, Hkv, D, 16, [1, 17, 0, 40, 1], [1, 17, 5, 100, 33], norm, pad=3) == 0


def test_append_slots_in_any_order():
    rng = np.random.default_rng(1)
    assert append_case(rng, 4, 2, 64, 32, [3, 1, 64], [35, 64, 64], True, slots=[5, 0, 2]) == 0


def test_append_one_norm_only_and_extremes():
    """Full-range values: saturation in the norm, the rotation and the requantization; a zero head."""
    rng = np.random.default_rng(2)

    def edit(L, q, k):
        q[0], k[0] = -32768, 32767
        q[1, 0], k[1] = 0, 0

    assert append_case(rng, 4, 4, 128, 64, [5], [70], True, sd=30000.0, edit=edit) == 0


@pytest.mark.parametrize("D", [16, 64, 128, 48])
def test_append_rotation_at_the_ends_of_16_bits(D):
    """x2 c + x1 s from -2^31 + 2^16 to 2^31, which 32 bits hold only one by one."""
    H, Hkv, P, ends = 4, 2, 16, np.array([-32768, 32767], np.int16)
    rng = np.random.default_rng(D)
    L = launch(rng, [64], [64], P)
    q, k = (rng.choice(ends, (64, h, D)) for h in (H, Hkv))
    v = np.zeros((64, Hkv, D), np.int8)
    cos, sin = (rng.choice(ends, (64, D // 2)) for _ in "cs")
    rq = (1142505715, 38)
    want = [np.zeros((64, H, D), np.int8)] + [np.zeros((L["N"], Hkv, P, D), np.int8) for _ in "kv"]
    got = [dev(w) for w in want]
    PO.append(q, k, v, want[1], want[2], L["table"], L["length"], L["q_start"], cos, sin, rq, rq, None, None, None, want[0])
    paged.append(dev(q), dev(k), dev(v), got[1], got[2], dev(L["table"]), dev(L["length"]), dev(L["q_start"]), dev(cos), dev(sin), rq,
                 rq, out=got[0])
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)
    assert len(np.unique(want[0])) > 2


def test_append_skips_rows_without_a_place():
    rng = np.random.default_rng(3)

    def edit(L, q, k):
        L["table"][0, 1] = L["N"]  # outside the cache
        L["table"][1, 0] = -7
        L["length"][2] = 2  # four rows, two positions

    assert append_case(rng, 4, 2, 64, 16, [20, 3, 4], [30, 3, 4], True, edit=edit) == 1 | 2


def test_append_positions_beyond_the_tables():
    rng = np.random.default_rng(4)
    assert append_case(rng, 2, 1, 64, 16, [6], [40], False, positions=37) == 2


def test_append_reads_strided_rows():
    """q, k, v as column ranges of one fused projection's rows; q8 into a wider buffer."""
    rng = np.random.default_rng(5)
    H, Hkv, D, P = 4, 2, 64, 16
    L = launch(rng, [9, 1], [25, 16], P)
    wide = rng.integers(-9000, 9000, (10, (H + Hkv) * D + 8)).astype(np.int16)
    q, k = wide[:, : H * D].reshape(10, H, D), wide[:, H * D : (H + Hkv) * D].reshape(10, Hkv, D)
    vw = rng.integers(-128, 128, (10, Hkv * D + 16)).astype(np.int8)
    cos, sin = (rng.integers(-16384, 16385, (30, D // 2)).astype(np.int16) for _ in "cs")
    kp, vp = (np.zeros((L["N"], Hkv, P, D), np.int8) for _ in "kv")
    out = np.zeros((10, H, D), np.int8)
    want = [out.copy(), kp.copy(), vp.copy()]
    PO.append(q, k, vw[:, : Hkv * D].reshape(10, Hkv, D), want[1], want[2], L["table"], L["length"], L["q_start"], cos, sin,
              (1142505715, 37), (1142505715, 36), None, None, None, want[0])
    tw, tv, to = dev(wide), dev(vw), torch.zeros((10, H * D + 32), dtype=torch.int8, device="cuda")
    view = lambda t, a, b, h: t[:, a:b].unflatten(1, (h, D))  # noqa: E731
    gk, gv = dev(kp), dev(vp)
    o = view(to, 0, H * D, H)
    paged.append(view(tw, 0, H * D, H), view(tw, H * D, (H + Hkv) * D, Hkv), view(tv, 0, Hkv * D, Hkv), gk, gv, dev(L["table"]),
                 dev(L["length"]), dev(L["q_start"]), dev(cos), dev(sin), (1142505715, 37), (1142505715, 36), out=o)
    assert np.array_equal(o.cpu().numpy(), want[0])
    assert np.array_equal(gk.cpu().numpy(), want[1]) and np.array_equal(gv.cpu().numpy(), want[2])
    assert int(to[:, H * D :].abs().sum()) == 0


# ---- attention ----------------------------------------------------------------------------
def attention_case(rng, H, Hkv, D, P, rows, lens, *, bits=15, score_rq=None, out_rq=(1717986918, 37), pad=0, slots=None, max_rows=None,
                   max_len=None, edit=None, sd=32.0, page_gap=0, check=True):
    L = launch(rng, rows, lens, P, slots=slots)
    R = int(L["q_start"][-1]) + pad
    i8 = lambda shape, s: np.clip(np.round(rng.normal(0, s, shape)), -128, 127).astype(np.int8)  # noqa: E731
    q = i8((R, H, D), sd)
    kp, vp = i8((L["N"], Hkv, P, D), sd), i8((L["N"], Hkv, P, D), 40.0)
    out = rng.integers(-128, 128, (R, H, D)).astype(np.int8)
    if score_rq is None:
        step = 640.0 / (1024.0 * D ** 0.5)
        Ss = 30 - int(np.floor(np.log2(step)))
        score_rq = (int(step * 2.0 ** Ss), Ss)
    if edit:
        edit(L, q, kp, vp)
    mr = max(max(rows), 1) if max_rows is None else max_rows
    ml = max(max(lens), 1) if max_len is None else max_len
    want = out.copy()
    PO.attention(q, kp, vp, L["table"], L["length"], L["q_start"], score_rq, out_rq, bits, L["seqs"], mr, ml, want)
    got, st = dev(out), status()
    tk, tv = dev(kp), dev(vp)
    if page_gap:  # pages further apart than their size
        wide = [torch.zeros((L["N"], Hkv * P * D + page_gap), dtype=torch.int8, device="cuda") for _ in "kv"]
        for w, t in zip(wide, (tk, tv)):
            w[:, : Hkv * P * D] = t.flatten(1)
        tk, tv = (w[:, : Hkv * P * D].unflatten(1, (Hkv, P, D)) for w in wide)
    paged.attention(dev(q), tk, tv, dev(L["table"]), dev(L["length"]), dev(L["q_start"]), score_rq, out_rq, prob_bits=bits,
                    max_rows=mr, max_len=ml, seqs=None if slots is None else dev(L["seqs"]), out=got, status=st)
    g = got.cpu().numpy()
    bad = np.argwhere(g != want)
    assert not len(bad), (len(bad), bad[:5].tolist(), [(int(g[tuple(b)]), int(want[tuple(b)])) for b in bad[:5]])
    return int(st.item())


GEOMETRIES = [(14, 2, 64), (16, 8, 128), (32, 8, 128), (8, 8, 64), (9, 3, 64), (5, 1, 128), (4, 2, 32), (3, 1, 16), (2, 1, 256),
              (6, 2, 80), (20, 1, 64), (33, 1, 128)]


@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
@pytest.mark.parametrize("P", [16, 64])
def test_attention_of_single_tokens(H, Hkv, D, P):
    rng = np.random.default_rng(H * 1000 + D + P)
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1]
    assert attention_case(rng, H, Hkv, D, P, [1] * len(lens), lens, pad=2) == 0


@pytest.mark.parametrize("H,Hkv,D", GEOMETRIES)
@pytest.mark.parametrize("P,bits", [(32, 15), (128, 8)])
def test_attention_of_chunks(H, Hkv, D, P, bits):
    rng = np.random.default_rng(H * 1000 + D + P)
    assert attention_case(rng, H, Hkv, D, P, [1, 33, 0, 70, 5, 129, 2], [40, 33, 9, 200, 5, 300, 128], bits=bits, pad=5) == 0


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_page_sizes(P, D):
    rng = np.random.default_rng(P + D)
    assert attention_case(rng, 8, 2, D, P, [1, 20, 1, 60], [P + 1, 2 * P + 7, 5 * P, 517], slots=[3, 1, 0, 6]) == 0


def test_attention_long_context():
    """More keys than a block's on-chip scores, on one and on two sequences."""
    rng = np.random.default_rng(7)
    assert attention_case(rng, 8, 2, 64, 128, [1, 1], [40001, 20000]) == 0
    assert attention_case(rng, 4, 1, 128, 64, [1], [70001]) == 0
    assert attention_case(rng, 4, 1, 128, 64, [40, 3], [9003, 12345]) == 0


@pytest.mark.parametrize("rq", [(1, 0), (1, 3), (0, 10), (4000000000, 40), (3000000000, 33), (2000000000, 32), (7, 63), (1900000000, 31)])
@pytest.mark.parametrize("rows", [[1, 1], [30, 17]])
def test_attention_score_scaling(rq, rows):
    """Every form of the score shift; flat and one-hot softmax; output saturation."""
    rng = np.random.default_rng(rq[0] % 1000 + rq[1])
    assert attention_case(rng, 4, 2, 64, 16, rows, [200, 77], score_rq=rq, out_rq=(1717986918, 33)) == 0
    assert attention_case(rng, 2, 1, 128, 64, rows, [200, 77], score_rq=rq, out_rq=(1, 0), bits=8) == 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [[1, 1, 1], [9, 40, 140]])
def test_attention_extreme_values(D, rows):
    """All -128: the largest scores and value sums; equal keys: a flat softmax."""
    rng = np.random.default_rng(D)

    def edit(L, q, kp, vp):
        q[:], kp[:], vp[:] = -128, -128, -128

    lens = [max(r, n) for r, n in zip(rows, (700, 64, 333))]
    for bits in (8, 15):
        assert attention_case(rng, 4, 2, D, 32, rows, lens, bits=bits, edit=edit, out_rq=(1717986918, 31 + bits // 2)) == 0


@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [0, 40, -3]), ([20, 50, 9], [12, 50, 0])])
@pytest.mark.parametrize("D", [64, 128, 32])
def test_attention_rows_without_keys_are_zero(rows, lens, D):
    """More rows than positions: the first rows see nothing."""
    rng = np.random.default_rng(D)
    assert attention_case(rng, 4, 2, D, 16, rows, lens) == 2


@pytest.mark.parametrize("D", [64, 128, 32])
@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 40, 40], [2, 90, 100]])
def test_attention_bad_pages_are_absent(rows, D):
    rng = np.random.default_rng(D)

    def edit(L, q, kp, vp):
        L["table"][0, 2] = L["N"]
        L["table"][1, :] = -1  # nothing left
        L["table"][2, 0] = 1 << 30
        L["table"][2, 3] = -2

    assert attention_case(rng, 4, 2, D, 16, rows, [100, 100, 111], edit=edit) == 1


def test_attention_bounds_cut_rows_and_keys():
    rng = np.random.default_rng(11)
    assert attention_case(rng, 4, 2, 64, 16, [12, 3], [60, 20], max_rows=5) & 4
    assert attention_case(rng, 4, 2, 64, 16, [1, 1], [60, 20], max_len=33) & 4
    assert attention_case(rng, 4, 2, 128, 16, [40, 33], [60, 50], max_len=33) & 4


def test_attention_pages_apart_and_wide_rows():
    rng = np.random.default_rng(12)
    assert attention_case(rng, 4, 2, 64, 16, [1, 30], [50, 61], page_gap=48) == 0
    H, Hkv, D, P = 4, 2, 64, 16
    L = launch(rng, [1, 20], [37, 40], P)
    i8 = lambda *s: rng.integers(-100, 100, s).astype(np.int8)  # noqa: E731
    wide, kp, vp = i8(21, 3 * H * D), i8(L["N"], Hkv, P, D), i8(L["N"], Hkv, P, D)
    q = wide[:, H * D : 2 * H * D].reshape(21, H, D)
    want = np.zeros((21, H, D), np.int8)
    args = ((1900000000, 35), (1717986918, 37))
    PO.attention(q, kp, vp, L["table"], L["length"], L["q_start"], *args, 15, None, 20, 40, want)
    tw, to = dev(wide), torch.zeros((21, 2 * H * D), dtype=torch.int8, device="cuda")
    o = to[:, H * D :].unflatten(1, (H, D))
    paged.attention(tw[:, H * D : 2 * H * D].unflatten(1, (H, D)), dev(kp), dev(vp), dev(L["table"]), dev(L["length"]),
                    dev(L["q_start"]), *args, max_rows=20, max_len=40, out=o)
    assert np.array_equal(o.cpu().numpy(), want) and int(to[:, : H * D].abs().sum()) == 0


# ---- pages --------------------------------------------------------------------------------
class Cache:
    def __init__(self, rng, S=12, W=6, N=40, P=16, layers=3, Hkv=2, D=32):
        self.P, self.rng = P, rng
        self.k, self.v = (rng.integers(-128, 128, (layers, N, Hkv, P, D)).astype(np.int8) for _ in "kv")
        self.o = PO.Pages(np.full((S, W), -1, np.int32), np.zeros(S, np.int32), np.zeros(N, np.int32), P)
        self.tk, self.tv = dev(self.k), dev(self.v)
        self.table, self.length, self.refs, self.status = dev(self.o.table), dev(self.o.length), dev(self.o.refs), status()

    def same(self, code=0):
        assert int(self.status.item()) == code
        self.status.zero_()
        for t, w, n in ((self.table, self.o.table, "table"), (self.length, self.o.length, "length"), (self.refs, self.o.refs, "refs"),
                        (self.tk, self.k, "k"), (self.tv, self.v, "v")):
            assert np.array_equal(t.cpu().numpy(), w), n

    def ints(self, x):
        return dev(np.array(x, np.int32))

    def reserve(self, slots, counts):
        code = self.o.reserve(slots, counts)
        paged.reserve(self.table, self.length, self.refs, self.ints(slots), self.ints(counts), self.P, status=self.status)
        self.same(code)
        return code

    def fork(self, parents, children, share=True):
        code, copies = self.o.fork(parents, children, share)
        for s, d, rows in copies:
            for x in (self.k, self.v):
                x[:, d, :, :rows] = x[:, s, :, :rows]
        paged.fork(self.tk, self.tv, self.table, self.length, self.refs, self.ints(parents), self.ints(children), share=share,
                   status=self.status)
        self.same(code)
        return code

    def free(self, slots):
        self.o.free(slots)
        paged.free(self.table, self.length, self.refs, self.ints(slots), status=self.status)
        self.same()

    def compact(self):
        for s, d in self.o.compact():
            for x in (self.k, self.v):
                x[:, d] = x[:, s]
        paged.compact(self.tk, self.tv, self.table, self.refs, status=self.status)
        self.same()


def test_pages_life():
    c = Cache(np.random.default_rng(0))
    assert c.reserve([3, 0, 7], [40, 0, 16]) == 0
    assert c.reserve([0, 3], [1, 8]) == 0
    assert c.fork([3, 7, 3], [1, 2, 4]) == 0
    assert c.reserve([1, 4], [3, 20]) == 0
    assert c.fork([1, 0], [5, 2], share=False) == 0  # slot 2 held pages
    c.free([3, 7])
    c.compact()
    assert c.reserve([3, 1], [90, 1]) == 0
    c.free([4, 4, 1])
    c.compact()
    c.compact()
    c.free(list(range(12)))
    assert not c.o.refs.any()


def test_pages_refusals_change_nothing():
    c = Cache(np.random.default_rng(1), N=9)
    assert c.reserve([0, 1], [50, 60]) == 0
    assert c.reserve([0], [40]) == 8
    assert c.reserve([0, 1], [1, 97]) == 2
    assert c.reserve([2, 2], [1, 1]) == 16
    assert c.reserve([12], [1]) == 16
    assert c.reserve([-1], [1]) == 16
    assert c.fork([0, 0], [2, 3], share=False) == 8
    assert c.fork([0], [0]) == 16
    assert c.fork([0, 1], [2, 2]) == 16
    assert c.fork([0, 1], [1, 2]) == 16
    assert c.fork([0, 30], [2, 3]) == 16
    c.o.table[4, 0], c.o.length[4] = c.o.table[0, 0], 5  # a part-filled page that two slots name
    c.o.refs[c.o.table[0, 0]] += 1
    c.table, c.length, c.refs = dev(c.o.table), dev(c.o.length), dev(c.o.refs)
    assert c.reserve([4], [1]) == 32


def test_pages_many():
    """More pairs, pages and slots than one block's threads."""
    rng = np.random.default_rng(2)
    c = Cache(rng, S=3000, W=3, N=9000, P=16, layers=1, Hkv=1, D=16)
    order = rng.permutation(3000)
    assert c.reserve(order[:1400].tolist(), rng.integers(0, 49, 1400).tolist()) == 0
    parents = rng.choice(order[:1400], 1500).tolist()
    assert c.fork(parents, order[1400:2900].tolist()) == 0
    c.free(order[:700].tolist())
    c.compact()
    assert c.fork(order[1400:1500].tolist(), order[2900:].tolist(), share=False) == 0


def test_compact_out_of_place():
    rng = np.random.default_rng(3)
    c = Cache(rng)
    c.reserve([0, 1, 2], [30, 40, 90])
    c.free([0])
    before = c.table.clone(), c.refs.clone()
    new = torch.empty_like(c.table), torch.empty_like(c.refs)
    assert paged.compact(c.tk, c.tv, c.table, c.refs, out=new) == new
    assert torch.equal(c.table, before[0]) and torch.equal(c.refs, before[1])
    for s, d in c.o.compact():
        for x in (c.k, c.v):
            x[:, d] = x[:, s]
    c.table, c.refs = new
    c.same()


# ---- sampling -----------------------------------------------------------------------------
def sample_case(rng, x, exponent, **settings):
    R = len(x)
    u = rng.random(R)
    u[0] = 0.0
    u[-1] = 1 - 2.0 ** -53
    kinds = dict(temperature=np.float32, top_k=np.int32, top_p=np.float32, min_p=np.float32)
    cols = {n: np.broadcast_to(np.asarray(s, kinds[n]), (R,)).copy() for n, s in settings.items()}
    token, prob = sampling.sample(dev(x), dev(u), exponent=exponent, **{n: dev(c) for n, c in cols.items()})
    token, prob = token.cpu().numpy(), prob.cpu().numpy()
    for r in range(R):
        want, p = PO.sample(x[r], float(u[r]), exponent, **{n: c[r].item() for n, c in cols.items()})
        assert token[r] == want, (r, int(token[r]), want)
        # one double division, rounded to float32: half a step, relative to the value
        assert abs(float(prob[r]) - p) <= p * (np.finfo(np.float32).eps / 2 + 2.0 ** -52)


def logits(rng, R, V, exponent, sd=2.5):
    return np.clip(np.round(rng.normal(0, sd, (R, V)) * 2.0 ** -exponent), -32768, 32767).astype(np.int16)


@pytest.mark.parametrize("V", [1, 2, 31, 512, 1000, 32003, 151936])
def test_sample_settings(V):
    rng = np.random.default_rng(V)
    R = 16 if V < 100000 else 8
    x = logits(rng, R, V, -10)
    sample_case(rng, x, -10)
    sample_case(rng, x, -10, temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 2.0, 50.0], R), top_k=rng.choice([0, 1, 2, 7, 50, 1000], R),
                top_p=rng.choice([1.0, 0.999, 0.9, 0.5, 0.01, 0.0], R), min_p=rng.choice([0.0, 0.01, 0.3, 1.0], R))


@pytest.mark.parametrize("name,values", [("top_p", [0.3, 0.9, 0.9999, 1e-9]), ("top_k", [1, 3, 40, 700]), ("min_p", [1e-9, 1e-4, 0.2, 1.0]),
                                         ("temperature", [1e-6, 0.01, 1e6, float("inf")])])
def test_sample_one_setting(name, values):
    rng = np.random.default_rng(5)
    for value in values:
        sample_case(rng, logits(rng, 8, 5000, -9, sd=1.0), -9, **{name: value})


def test_sample_ties_and_flat_rows():
    """Equal logits everywhere, two levels, the lowest value as a mask: ties go by index."""
    rng = np.random.default_rng(6)
    x = np.zeros((8, 3001), np.int16)
    x[1] = -32768
    x[2, ::3] = 1
    x[3] = 32767
    x[4] = -32768
    x[4, 17] = 5
    x[5] = rng.integers(0, 2, 3001) * -20000
    x[6, 1500:] = -32768
    x[7, 3000] = 3000
    for s in ({}, dict(top_k=700), dict(top_p=0.37), dict(top_k=2500, top_p=0.6, min_p=0.5), dict(temperature=0.0), dict(min_p=1.0)):
        sample_case(rng, x, -8, **s)


@pytest.mark.parametrize("exponent", [-31, -15, -4, 0, 15])
def test_sample_exponents(exponent):
    rng = np.random.default_rng(7)
    x = rng.integers(-32768, 32768, (6, 700)).astype(np.int16)
    sample_case(rng, x, exponent, top_p=0.8)
    sample_case(rng, x, exponent, temperature=1000.0, top_k=100)


def test_sample_strided_rows_and_padded_vocabulary():
    rng = np.random.default_rng(8)
    x = logits(rng, 5, 1003, -10)
    x[:, 900:] = 32767  # padding columns, never to be drawn
    u = rng.random(5)
    token, _ = sampling.sample(dev(x)[:, :1000], dev(u), exponent=-10, vocab=900)
    assert token.cpu().tolist() == [PO.sample(x[r, :900], float(u[r]), -10)[0] for r in range(5)]


def test_sample_follows_the_distribution():
    """20,000 draws of one row: every count within 5 standard deviations of its expectation."""
    rng = np.random.default_rng(9)
    x = logits(rng, 1, 50, -10, sd=1.0)
    n = 20000
    u = (np.arange(n) + 0.5) / n
    token, _ = sampling.sample(dev(np.repeat(x, n, 0)), dev(u), exponent=-10)
    p = np.exp(x[0].astype(np.float64) / 1024)
    p /= p.sum()
    # stratified u: a count differs from n p by less than one at either end of its interval, and
    # the weights' 2^-21 moves the ends by less than n 2^-20 draws
    assert np.all(np.abs(np.bincount(token.cpu().numpy(), minlength=50) - n * p) < 2 + n * 2.0 ** -20)


# ---- together -----------------------------------------------------------------------------


def test_nan_settings_turn_the_filters_off():
    rng = np.random.default_rng(10)
    x = logits(rng, 4, 300, -10)
    u = dev(np.array([0.1, 0.5, 0.9, 0.3]))
    nan = torch.full((4,), float("nan"), device="cuda")
    a, _ = sampling.sample(dev(x), u, exponent=-10, top_p=nan, min_p=nan)
    b, _ = sampling.sample(dev(x), u, exponent=-10)
    assert torch.equal(a, b)
    a, _ = sampling.sample(dev(x), u, exponent=-10, temperature=nan)
    assert a.cpu().tolist() == [int(np.argmax(r)) for r in x]
