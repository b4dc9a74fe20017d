"""Cases of the paged-serving operators: appending a launch's keys and values to a paged int8
cache (query / key norms and the rotation in the same pass), attention of a chunk of new tokens
over the pages, forking / copying / compacting pages, and sampling from integer logits.

Everything is the framework's integer arithmetic, so the outputs are whole numbers and have one
right value; the one exception is the probability that sampling returns beside a token.
"""
import math
import random

import torch

own = False

I64 = torch.int64
EXPI = [round(65535 * math.exp(-i)) for i in range(16)]
EXPF = [round(65535 * math.exp(-f / 256.0)) for f in range(256)]
# sampling weights: 2^31 * 2^(-j / 1024), and ln(2) 2^-20 in units of 2^-32
POW2 = [round(2.0 ** 31 * 2.0 ** (-j / 1024.0)) for j in range(1024)]
LN2_STEP = 2839


# ---- the cases ----------------------------------------------------------------------------
def listed():
    return [
        # one sequence's next token with query and key norms (Qwen3-0.6B heads), the latency of a batch-1 step
        dict(name="append-1-token-norm", op="append", H=16, Hkv=8, D=128, P=64, norm=True, seqs=1, rows_lo=1, rows_hi=1,
             ctx_lo=900, ctx_hi=900, pad=0, layout=1),
        # prompt chunks of 16 sequences, ragged, with a few pad rows at the end of the launch
        dict(name="append-chunks-norm", op="append", H=16, Hkv=8, D=128, P=64, norm=True, seqs=16, rows_lo=384,
             rows_hi=640, ctx_lo=0, ctx_hi=2000, pad=13, layout=2),
        # one sequence's next token at a short context (Qwen2.5-0.5B heads)
        dict(name="attend-1-token", op="attention", H=14, Hkv=2, D=64, P=64, bits=15, seqs=1, rows_lo=1, rows_hi=1,
             ctx_lo=1000, ctx_hi=1000, mixed=0, layout=3),
        # 64 sequences of ragged lengths decode together (Qwen3-0.6B heads)
        dict(name="attend-64-tokens-ragged", op="attention", H=16, Hkv=8, D=128, P=64, bits=15, seqs=64, rows_lo=1,
             rows_hi=1, ctx_lo=1500, ctx_hi=4200, mixed=0, layout=4),
        # two very long sequences decode (Llama-3-8B heads)
        dict(name="attend-2-tokens-64k", op="attention", H=32, Hkv=8, D=128, P=128, bits=15, seqs=2, rows_lo=1, rows_hi=1,
             ctx_lo=50001, ctx_hi=65003, mixed=0, layout=5),
        # chunks of four prompts over their earlier pages (Llama-3-8B heads)
        dict(name="attend-4-chunks", op="attention", H=32, Hkv=8, D=128, P=64, bits=15, seqs=4, rows_lo=500, rows_hi=512,
             ctx_lo=2100, ctx_hi=4000, mixed=0, layout=6),
        # decode of 30 sequences with two prompt chunks in the same launch (Qwen2.5-0.5B heads)
        dict(name="attend-mixed", op="attention", H=14, Hkv=2, D=64, P=32, bits=15, seqs=32, rows_lo=300, rows_hi=420,
             ctx_lo=200, ctx_hi=2300, mixed=30, layout=7),
        # 48 answers continue 12 prompts: full pages shared, the part-filled last page copied
        dict(name="fork-48", op="pages", kind="fork", L=24, Hkv=2, D=64, P=64, parents=12, children=48, len_lo=500,
             len_hi=1100, pages=2048, layout=8),
        # whole sequences copied, nothing shared
        dict(name="copy-24", op="pages", kind="copy", L=24, Hkv=2, D=64, P=64, parents=8, children=24, len_lo=900,
             len_hi=1500, pages=2048, layout=9),
        # live pages moved to the front of the cache
        dict(name="compact-half", op="pages", kind="compact", L=24, Hkv=2, D=64, P=64, parents=64, children=0, len_lo=600,
             len_hi=1300, pages=2048, layout=10),
        # one sequence's next token
        dict(name="sample-1", op="sample", R=1, V=151936, E=-10, spread=2.5, layout=11),
        # a batch of sequences, each with its own settings
        dict(name="sample-128", op="sample", R=128, V=151936, E=-10, spread=2.5, layout=12),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "pages", "sample"])
    while True:
        layout = rng.randrange(1 << 20)
        heads = rng.choice([(14, 2, 64), (9, 3, 64), (32, 8, 128), (16, 8, 128), (8, 8, 64), (16, 2, 128), (5, 1, 128)])
        P = rng.choice([16, 32, 64, 128])
        if op == "append":
            n = _between(rng, 1, 128)
            lo = _between(rng, 1, 1024)
            c = dict(op=op, H=heads[0], Hkv=heads[1], D=heads[2], P=P, norm=rng.random() < 0.6, seqs=n, rows_lo=lo,
                     rows_hi=lo + rng.randrange(1 + lo), ctx_lo=0, ctx_hi=_between(rng, 1, 4000), pad=rng.randrange(20),
                     layout=layout)
        elif op == "attention":
            n = _between(rng, 1, 96)
            token = rng.random() < 0.5
            lo = 1 if token else _between(rng, 2, 900)
            ctx = _between(rng, 1, 60000)
            c = dict(op=op, H=heads[0], Hkv=heads[1], D=heads[2], P=P, bits=rng.choice([8, 15, 15]), seqs=n, rows_lo=lo,
                     rows_hi=1 if token else lo + rng.randrange(1 + lo // 2), ctx_lo=max(0, ctx - rng.randrange(ctx + 1)),
                     ctx_hi=ctx, mixed=0 if token else rng.randrange(n), layout=layout)
        elif op == "pages":
            kind = rng.choice(["fork", "copy", "compact"])
            L, n = rng.randrange(1, 33), _between(rng, 1, 48)
            lo = _between(rng, 1, 1200)
            hi = lo + rng.randrange(1 + lo)
            c = dict(op=op, kind=kind, L=L, Hkv=heads[1], D=heads[2], P=P, parents=n,
                     children=0 if kind == "compact" else rng.randrange(1, 65), len_lo=lo, len_hi=hi, pages=0, layout=layout)
            c["pages"] = _pages_needed(c) * 3 // 2 + 3
            if c["pages"] * 2 * L * heads[1] * P * heads[2] > 1.7e9:
                continue
        else:
            c = dict(op=op, R=_between(rng, 1, 192), V=rng.choice([512, 32003, 49152, 128256, 151936, rng.randrange(1000, 150000)]),
                     E=rng.randrange(-12, -8), spread=round(rng.uniform(0.8, 4.0), 2), layout=layout)
        most = max(_cost(x) for x in listed() if x["op"] == op)
        if _cost(c) <= most:
            return c


# ---- what a case's layout says: lengths and pages, the same for every seed ------------------
def _rows_and_lengths(c):
    """New rows and whole length (with the new rows) of each sequence of a launch."""
    r = random.Random(c["layout"])
    rows = [r.randint(c["rows_lo"], c["rows_hi"]) for _ in range(c["seqs"])]
    mixed = c.get("mixed", 0)
    rows[:mixed] = [1] * mixed
    return rows, [m + r.randint(c["ctx_lo"], c["ctx_hi"]) for m in rows]


def _page_lengths(c):
    r = random.Random(c["layout"])
    return [r.randint(c["len_lo"], c["len_hi"]) for _ in range(c["parents"])]


def _children(c):
    r = random.Random(c["layout"] + 1)
    return [r.randrange(c["parents"]) for _ in range(c["children"])]


def _pages_needed(c):
    lens, P = _page_lengths(c), c["P"]
    n = sum(-(-x // P) for x in lens)
    for p in _children(c):
        n += 1 if c["kind"] == "fork" else -(-lens[p] // P)
    return n


def _compact_ids(c):
    """Page ids of the sequences' pages, in order, scattered over the cache."""
    n = sum(-(-x // c["P"]) for x in _page_lengths(c))
    return random.Random(c["layout"] + 2).sample(range(c["pages"]), n)


def _cost(c):
    if c["op"] == "attention":
        rows, lens = _rows_and_lengths(c)
        # what the plain form holds: every sequence padded to the longest
        return c["seqs"] * (max(rows) * c["H"] + 2 * c["Hkv"] * c["D"]) * max(lens)
    w = work(c)
    return w["bytes"]


def work(c):
    op = c["op"]
    if op == "append":
        R = sum(_rows_and_lengths(c)[0])
        H, Hkv, D = c["H"], c["Hkv"], c["D"]
        return {"bytes": R * (2 * (H + Hkv) * D + Hkv * D + H * D + 2 * Hkv * D + 2 * D), "flops": R * (H + Hkv) * D * 20}
    if op == "attention":
        rows, lens = _rows_and_lengths(c)
        H, Hkv, D = c["H"], c["Hkv"], c["D"]
        pairs = sum(m * (n - m) + m * (m + 1) // 2 for m, n in zip(rows, lens))
        return {"bytes": 2 * Hkv * D * sum(lens) + 2 * H * D * sum(rows), "flops": 4 * H * D * pairs}
    if op == "pages":
        row = c["L"] * 2 * c["Hkv"] * c["D"]
        lens, P = _page_lengths(c), c["P"]
        if c["kind"] == "compact":
            ids = _compact_ids(c)
            moved = sum(i >= len(ids) for i in ids) * P
        elif c["kind"] == "fork":
            moved = sum(lens[p] % P for p in _children(c))
        else:
            moved = sum(lens[p] for p in _children(c))
        return {"bytes": 2 * row * moved + 8 * c["pages"], "flops": 0}
    return {"bytes": c["R"] * (2 * c["V"] + 36), "flops": c["R"] * c["V"] * 10}


# ---- inputs --------------------------------------------------------------------------------
def _i8(shape, g, sd):
    out = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        part = flat[i : i + (1 << 28)]
        part.copy_((torch.randn(part.numel(), generator=g, device="cuda") * sd).round_().clamp_(-128, 127))
    return out


def _i16(shape, g, sd):
    return (torch.randn(shape, generator=g, device="cuda") * sd).round_().clamp_(-32768, 32767).to(torch.int16)


def _launch(c, g):
    """Page table, lengths and row starts of a launch, pages in shuffled order."""
    rows, lens = _rows_and_lengths(c)
    P = c["P"]
    need = [-(-n // P) for n in lens]
    W, N = max(need), sum(need) + 5
    ids = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device="cuda")
    j = torch.arange(W, device="cuda")
    held = j[None] < torch.tensor(need, device="cuda")[:, None]
    table = torch.where(held, ids[(first[:, None] + j).clamp(max=N - 1)], torch.tensor(-1, dtype=torch.int32, device="cuda"))
    starts = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
    return dict(table=table.contiguous(), length=torch.tensor(lens, dtype=torch.int32, device="cuda"), q_start=starts, N=N,
                R=sum(rows), max_rows=max(rows), max_len=max(lens))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] in ("append", "attention"):
        s.update(_launch(c, g))
        H, Hkv, D, R = c["H"], c["Hkv"], c["D"], s["R"]
        shape = (s["N"], Hkv, c["P"], D)
        if c["op"] == "append":
            R += c["pad"]
            s["q"], s["k"] = _i16((R, H, D), g, 4000.0), _i16((R, Hkv, D), g, 3000.0)
            s["v"] = _i8((R, Hkv, D), g, 30.0)
            # the norms' integer constants as the quantizer picks them for a head of D values
            eps, C, sh = (343597, 759250125, 28) if D == 128 else (68719, 268435456, 26)
            s["q_norm"] = (_i16((D,), g, 1500.0) + 14000, eps, C, sh) if c["norm"] else None
            s["k_norm"] = (_i16((D,), g, 1500.0) + 12000, eps, C, sh) if c["norm"] else None
            s["q_rq"], s["k_rq"] = (1142505715, 37), (1261255548, 37)
            pos = torch.arange(s["max_len"], device="cuda", dtype=torch.float64)
            freq = 1e6 ** (-torch.arange(D // 2, device="cuda", dtype=torch.float64) * 2 / D)
            ang = pos[:, None] * freq[None]
            s["cos"], s["sin"] = ((f(ang) * 16384).round().to(torch.int16) for f in (torch.cos, torch.sin))
            s["k_pages"], s["v_pages"] = (torch.zeros(shape, dtype=torch.int8, device="cuda") for _ in "kv")
            s["out"] = torch.zeros((R, H, D), dtype=torch.int8, device="cuda")
        else:
            s["q"] = _i8((R, H, D), g, 32.0)
            s["k_pages"], s["v_pages"] = _i8(shape, g, 32.0), _i8(shape, g, 40.0)
            # a score gap of sd 32 * 32 * sqrt(D) stands for 2.5 nats: 640 steps of 1/256
            step = 640.0 / (1024.0 * math.sqrt(D))
            Ss = 30 - math.floor(math.log2(step))
            s["score_rq"], s["out_rq"] = (int(step * 2.0 ** Ss), Ss), (1717986918, 37)
            s["out"] = torch.zeros((R, H, D), dtype=torch.int8, device="cuda")
        return s
    if c["op"] == "pages":
        lens, P, N, n = _page_lengths(c), c["P"], c["pages"], c["children"]
        need = [-(-x // P) for x in lens]
        W, slots = max(need) + 1, len(lens) + n
        ids = _compact_ids(c) if c["kind"] == "compact" else list(range(sum(need)))
        rows = [ids[sum(need[:i]) : sum(need[: i + 1])] for i in range(len(need))] + [[] for _ in range(n)]
        s["table"] = torch.tensor([r + [-1] * (W - len(r)) for r in rows], dtype=torch.int32, device="cuda")
        s["length"] = torch.tensor(lens + [0] * n, dtype=torch.int32, device="cuda")
        refs = torch.zeros(N, dtype=torch.int32)
        refs[torch.tensor(ids)] = 1
        s["refs"] = refs.cuda()
        s["parents"] = torch.tensor(_children(c), dtype=torch.int32, device="cuda")
        s["children"] = torch.tensor(list(range(len(lens), slots)), dtype=torch.int32, device="cuda")
        shape = (c["L"], N, c["Hkv"], P, c["D"])
        s["k_pages"], s["v_pages"] = (torch.randint(-128, 128, shape, generator=g, dtype=torch.int8, device="cuda") for _ in "kv")
        if c["kind"] == "compact":
            s["new_table"], s["new_refs"] = torch.empty_like(s["table"]), torch.empty_like(s["refs"])
        return s
    R, V = c["R"], c["V"]
    x = torch.randn((R, V), generator=g, device="cuda") * c["spread"]
    # some rows are sure of a few tokens, others are flat
    lift = torch.rand((R, 1), generator=g, device="cuda") * 10
    at = torch.randint(0, V, (R, 12), generator=g, device="cuda")
    x.scatter_add_(1, at, lift * torch.rand((R, 12), generator=g, device="cuda") + 2 * c["spread"])
    s["logits"] = (x * 2.0 ** -c["E"]).round_().clamp_(-32768, 32767).to(torch.int16)
    r = random.Random(c["layout"])
    pick = lambda v, t: torch.tensor([r.choice(v) for _ in range(R)], dtype=t, device="cuda")  # noqa: E731
    s["temperature"] = pick([0.6, 0.7, 0.8, 1.0, 1.0, 1.3] + ([0.0] if R > 4 else []), torch.float32)
    s["top_k"] = pick([0, 0, 20, 50, 1000], torch.int32)
    s["top_p"] = pick([1.0, 0.95, 0.9, 0.8, 0.5], torch.float32)
    s["min_p"] = pick([0.0, 0.0, 0.02, 0.1], torch.float32)
    if R == 1:
        s["top_k"].zero_()
        s["top_p"].fill_(0.95)
    s["random"] = torch.rand(R, generator=g, device="cuda", dtype=torch.float64)
    return s


# ---- one pass ------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from llaccel_b200 import paged, sampling

        if c["op"] == "append":
            paged.append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["q_start"], s["cos"],
                         s["sin"], s["q_rq"], s["k_rq"], q_norm=s["q_norm"], k_norm=s["k_norm"], out=s["out"])
            return s["out"], s["k_pages"], s["v_pages"]
        if c["op"] == "attention":
            return paged.attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["q_start"], s["score_rq"],
                                   s["out_rq"], prob_bits=c["bits"], max_rows=s["max_rows"], max_len=s["max_len"],
                                   out=s["out"])
        if c["op"] == "pages" and c["kind"] == "compact":
            paged.compact(s["k_pages"], s["v_pages"], s["table"], s["refs"], out=(s["new_table"], s["new_refs"]))
            return s["k_pages"], s["v_pages"], s["new_table"], s["new_refs"]
        if c["op"] == "pages":
            paged.fork(s["k_pages"], s["v_pages"], s["table"], s["length"], s["refs"], s["parents"], s["children"],
                       share=c["kind"] == "fork")
            return s["k_pages"], s["v_pages"], s["table"], s["length"], s["refs"]
        return sampling.sample(s["logits"], s["random"], exponent=c["E"], temperature=s["temperature"], top_k=s["top_k"],
                               top_p=s["top_p"], min_p=s["min_p"])
    if c["op"] == "append":
        return _append(s)
    if c["op"] == "attention":
        return _attention(s)
    if c["op"] == "pages":
        return _compact(s) if c["kind"] == "compact" else _fork(s, c["kind"] == "fork")
    return _sample(s, c["E"])


def _rshr(v, n):
    """Shift right by n, halves up."""
    return v if n == 0 else (v >> n) + ((v >> (n - 1)) & 1)


def _placed(s, R):
    """Sequence, position and validity of each of R launch rows."""
    r = torch.arange(R, device="cuda")
    starts = s["q_start"].to(I64)
    i = torch.searchsorted(starts[1:].contiguous(), r, right=True).clamp(max=starts.numel() - 2)
    pos = s["length"].to(I64)[i] - (starts[i + 1] - r)
    return i, pos, (r < starts[-1]) & (pos >= 0)


def _norm(x, norm):
    if norm is None:
        return x
    gamma, eps, C, sh = norm
    t = (x * x).sum(-1, keepdim=True) + eps
    r = t.to(torch.float64).sqrt().to(I64)
    r = r - (r * r > t).to(I64)
    r = r + ((r + 1) * (r + 1) <= t).to(I64)
    inv = (C // r.clamp(min=1)).clamp(max=65535)
    return _rshr(x * gamma.to(I64) * inv, sh).clamp(-32768, 32767)


def _rotate(x, cos, sin, rq):
    a, b = x.chunk(2, -1)
    y = torch.cat([_rshr(a * cos - b * sin, 14), _rshr(b * cos + a * sin, 14)], -1).clamp(-32768, 32767)
    return _rshr(y * rq[0], rq[1]).clamp(-128, 127).to(torch.int8)


def _append(s):
    P = s["k_pages"].shape[2]
    i, pos, ok = _placed(s, s["q"].shape[0])
    at = pos.clamp(0, s["cos"].shape[0] - 1)
    cos, sin = (s[k].to(I64)[at][:, None] for k in ("cos", "sin"))
    q = _rotate(_norm(s["q"].to(I64), s["q_norm"]), cos, sin, s["q_rq"])
    k = _rotate(_norm(s["k"].to(I64), s["k_norm"]), cos, sin, s["k_rq"])
    s["out"][ok] = q[ok]
    page = s["table"].to(I64)[i, at // P]
    s["k_pages"][page[ok], :, (at % P)[ok]] = k[ok]
    s["v_pages"][page[ok], :, (at % P)[ok]] = s["v"][ok]
    return s["out"], s["k_pages"], s["v_pages"]


def _attention(s):
    c = s["case"]
    H, Hkv, D, P, bits = c["H"], c["Hkv"], c["D"], c["P"], c["bits"]
    n, m, T = s["length"].numel(), s["max_rows"], s["max_len"]
    W = -(-T // P)
    ids = s["table"][:, :W].to(I64).clamp(min=0)
    # [n, Hkv, W * P, D]; sums of int8 products stay below 2^24, so 32-bit floats hold them exactly
    k, v = (s[x][ids].permute(0, 2, 1, 3, 4).reshape(n, Hkv, W * P, D).float() for x in ("k_pages", "v_pages"))
    starts, length = s["q_start"].to(I64), s["length"].to(I64)
    j = torch.arange(m, device="cuda")
    rows = (starts[1:] - starts[:-1])[:, None]
    live = j[None] < rows
    at = (starts[:-1, None] + j).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].view(n, m, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(n, Hkv, -1, D).float()
    pos = length[:, None] - rows + j
    seen = (torch.arange(W * P, device="cuda") <= pos[..., None]) & live[..., None]
    seen = seen[:, None, None]
    score = (q @ k.transpose(-1, -2)).to(torch.int32).view(n, Hkv, H // Hkv, m, W * P)
    top = torch.where(seen, score, -(1 << 30)).amax(-1, keepdim=True)
    z = _rshr((top - score).to(I64) * s["score_rq"][0], s["score_rq"][1])
    seen = seen & (z < 4096)
    z = torch.where(seen, z, 0)
    expi, expf = (torch.tensor(t, device="cuda") for t in (EXPI, EXPF))
    p = torch.where(seen, (expi[z >> 8] * expf[z & 255] + 32768) >> 16, 0)
    del z, score
    inv = (1 << 31) // p.sum(-1, keepdim=True).clamp(min=1)
    p = _rshr(p * inv, 31 - bits).clamp(max=(1 << bits) - 1)
    # the normalised weights add up to 2^16 at most, so these sums stay below 2^24 too
    o = (p.float().view(n, Hkv, -1, W * P) @ v).to(I64).view(n, Hkv, H // Hkv, m, D)
    o = _rshr(o, 7) if bits == 15 else o
    o = _rshr(o * s["out_rq"][0], s["out_rq"][1]).clamp(-128, 127).to(torch.int8)
    s["out"][at[live]] = o.permute(0, 3, 1, 2, 4).reshape(n, m, H, D)[live]
    return s["out"]


def _fork(s, share):
    table, length, refs = s["table"], s["length"], s["refs"]
    P = s["k_pages"].shape[3]
    parents, children = s["parents"].to(I64), s["children"].to(I64)
    old = table[children].to(I64)
    refs.index_add_(0, old[old >= 0], -torch.ones_like(old[old >= 0]).to(torch.int32))
    size = length[parents].to(I64)
    src = table[parents].to(I64)
    j = torch.arange(table.shape[1], device="cuda")
    held = j * P < size[:, None]
    kept = held & ((j + 1) * P <= size[:, None]) if share else torch.zeros_like(held)
    fresh = held & ~kept
    new = torch.nonzero(refs == 0).flatten()[: int(fresh.sum())]
    row = torch.where(kept, src, -1)
    row[fresh] = new
    table[children] = row.to(torch.int32)
    length[children] = size.to(torch.int32)
    refs.index_add_(0, src[kept], torch.ones_like(src[kept]).to(torch.int32))
    refs[new] = 1
    # rows of the new pages that the parent has written
    rows = (size[:, None] - j * P)[fresh]
    take = (torch.arange(P, device="cuda") < rows[:, None])[None, :, None, :, None]
    for x in (s["k_pages"], s["v_pages"]):
        x[:, new] = torch.where(take, x[:, src[fresh]], x[:, new])
    return s["k_pages"], s["v_pages"], table, length, refs


def _compact(s):
    refs, table = s["refs"], s["table"].to(I64)
    used = refs > 0
    n = int(used.sum())
    first = torch.arange(refs.numel(), device="cuda") < n
    src, dst = torch.nonzero(used & ~first).flatten(), torch.nonzero(~used & first).flatten()
    for x in (s["k_pages"], s["v_pages"]):
        x[:, dst] = x[:, src]
    to = torch.arange(refs.numel(), device="cuda")
    to[src] = dst
    s["new_table"].copy_(torch.where(table >= 0, to[table.clamp(min=0)], table))
    s["new_refs"].zero_()
    s["new_refs"][to[used]] = refs[used]
    return s["k_pages"], s["v_pages"], s["new_table"], s["new_refs"]


def _times(total, f):
    """total * f / 2^31 as whole part and whether anything is left over, for total < 2^62 and f <= 2^31."""
    low = (total & ((1 << 31) - 1)) * f
    return (total >> 31) * f + (low >> 31), (low & ((1 << 31) - 1)) > 0


def _sample(s, E):
    x = s["logits"].to(I64)
    V = x.shape[1]
    temp = s["temperature"].to(torch.float64)[:, None]
    greedy = ~(temp > 0)
    step = (math.log2(math.e) * 2.0 ** (32 + E) / temp.masked_fill(greedy, 1.0)).round().clamp(max=2.0 ** 47).to(I64)
    gap = x.amax(1, keepdim=True) - x
    e = (gap * step) >> 12
    base = torch.tensor(POW2, device="cuda")[(e >> 10) & 1023]
    w = (base - ((base * ((e & 1023) * LN2_STEP)) >> 32)) >> (e >> 20).clamp(max=62)
    del e, base
    order = torch.sort(gap, dim=1, stable=True).indices
    ranked = w.gather(1, order)
    total = ranked.cumsum(1)
    k = s["top_k"].to(I64)[:, None]
    k = torch.where(greedy, 1, torch.where((k <= 0) | (k > V), V, k))
    top_p = s["top_p"].to(torch.float64)[:, None]
    part = (top_p.clamp(0, 1) * 2.0 ** 31).floor().nan_to_num(0).to(I64)
    need, more = _times(total.gather(1, k - 1), part)
    need = (need + more).clamp(min=1)
    by_p = torch.where(top_p < 1, (total < need).sum(1, keepdim=True) + 1, V)
    least = (s["min_p"].to(torch.float64)[:, None].nan_to_num(0).clamp(0, 1) * 2.0 ** 31).ceil().to(I64)
    by_m = (ranked >= least).sum(1, keepdim=True)
    n = torch.minimum(torch.minimum(k, by_p), by_m).clamp(min=1)
    keep = torch.zeros_like(w, dtype=torch.bool).scatter_(1, order, torch.arange(V, device="cuda") < n)
    w = torch.where(keep, w, 0)
    run_up = w.cumsum(1)
    u = (s["random"][:, None] * 2.0 ** 31).floor().nan_to_num(0).clamp(0, 2.0 ** 31 - 1).to(I64)
    at, _ = _times(run_up[:, -1:], u)
    token = (run_up <= at).sum(1, keepdim=True)
    prob = w.gather(1, token).to(torch.float64) / run_up[:, -1:].to(torch.float64)
    return token[:, 0].to(torch.int32), prob[:, 0].to(torch.float32)


# ---- the definition, sequence by sequence and row by row, in 64 bits -------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "sample" and c["R"] * c["V"] <= 24_000_000:
        return _exact_sample(s, c["E"])
    if c["op"] == "attention" and work(c)["flops"] < 2e10:
        return _exact_attention(s)
    return None


def _exact_attention(s):
    c = s["case"]
    P, D, rep, bits = c["P"], c["D"], c["H"] // c["Hkv"], c["bits"]
    table, starts, lens = s["table"].tolist(), s["q_start"].tolist(), s["length"].tolist()
    out = s["out"].to(I64)
    curve = torch.tensor([(EXPI[z >> 8] * EXPF[z & 255] + 32768) // 65536 for z in range(4096)] + [0], device="cuda")
    for i, n in enumerate(lens):
        ids = torch.tensor(table[i][: -(-n // P)], device="cuda")
        a, b = starts[i], starts[i + 1]
        for h in range(c["H"]):
            k, v = (s[x][ids, h // rep].reshape(-1, D)[:n].to(torch.float64) for x in ("k_pages", "v_pages"))
            sc = (s["q"][a:b, h].to(torch.float64) @ k.T).to(I64)
            hide = torch.arange(n, device="cuda") > torch.arange(n - (b - a), n, device="cuda")[:, None]
            d = sc.masked_fill(hide, -(1 << 40)).amax(1, keepdim=True) - sc
            z = (d * s["score_rq"][0] + (1 << (s["score_rq"][1] - 1))) >> s["score_rq"][1]
            p = curve[z.clamp(0, 4096)].masked_fill(hide, 0)
            pn = (p * (2 ** 31 // p.sum(1, keepdim=True)) + (1 << (30 - bits))) >> (31 - bits)
            o = (pn.clamp(max=2 ** bits - 1).to(torch.float64) @ v).to(I64)
            o = (o + 64) >> 7 if bits == 15 else o
            out[a:b, h] = ((o * s["out_rq"][0] + (1 << (s["out_rq"][1] - 1))) >> s["out_rq"][1]).clamp(-128, 127)
    return out.to(torch.int8)


def _exact_sample(s, E):
    tokens, probs = [], []
    cols = [s[k].tolist() for k in ("temperature", "top_k", "top_p", "min_p", "random")]
    for x, temp, k, top_p, min_p, u in zip(s["logits"], *cols):
        x = x.cpu().to(I64)
        V, top = x.numel(), int(x.max())
        step = min(round(math.log2(math.e) * 2.0 ** (32 + E) / temp), 2 ** 47) if temp > 0 else 0
        # weight of every gap that occurs, once
        levels, which, count = torch.unique(top - x, return_inverse=True, return_counts=True)
        w = []
        for gap in levels.tolist():
            e = gap * step >> 12
            b = POW2[e >> 10 & 1023]
            w.append(b - (b * ((e & 1023) * LN2_STEP) >> 32) >> (e >> 20))
        count = count.tolist()
        k = 1 if not temp > 0 else V if k <= 0 or k > V else k
        all_k, left = 0, k
        for wt, m in zip(w, count):
            all_k += wt * min(m, left)
            left -= min(m, left)
        need = max(1, -(-all_k * math.floor(min(1.0, max(0.0, top_p)) * 2 ** 31) // 2 ** 31)) if top_p < 1 else None
        keep, left, got = [], k, 0
        for wt, m in zip(w, count):
            m = min(m, left)
            if need is not None and wt:
                m = min(m, max(0, -(-(need - got) // wt)))
            elif need is not None and got >= need:
                m = 0
            if wt < math.ceil(min(1.0, max(0.0, min_p)) * 2 ** 31):
                m = 0
            keep.append(m)
            left -= m
            got += wt * m
        kept = torch.zeros(V, dtype=I64)
        for i, (m, wt) in enumerate(zip(keep, w)):
            if m == 0 or wt == 0:
                break
            kept[torch.nonzero(which == i).flatten()[:m]] = wt
        upto = kept.cumsum(0)
        W = int(upto[-1])
        t = W * math.floor(u * 2 ** 31) >> 31
        tok = int(torch.searchsorted(upto, torch.tensor(t), right=True))
        tokens.append(tok)
        probs.append(int(kept[tok]) / W)
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(probs, dtype=torch.float64)
