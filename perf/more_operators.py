"""Measured operators: the paged key/value cache.

A pool of pages holds the keys and values of many sequences in 16 bits, each
page some rows of every key head; a table names the pages of each sequence in
order.  Four operators work on it: the append of new tokens, whose keys (and
queries) are rotated by their positions on the way; the attention over it, of
single tokens, chunks and frames; the attention of a tree of drafted tokens,
each of which sees the cached rows and its own ancestors; and the commit, which
moves the rows of the accepted tokens to the front of the draft, in every layer's
pool at once.

listed() and draw() name the cases, prepare() makes a case's inputs on the GPU
from a seed, run() is one pass: through the library's entry points where `own`
is true, in elementary torch operations otherwise.  work() says what a pass
cannot do without, exact() gives the results in 64 bits.

Appends and commits change the pool in place, in both forms, and a second pass
over the same state writes the same values again.  Sequences' pages lie in the
pool in random order, and table entries past a sequence's pages are -1.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
INF = float("inf")


# ---------------------------------------------------------------- the cases
def listed() -> list:
    return [
        # one new token of each of 16 sequences: the smallest append, made once per
        # layer and generated token
        dict(name="append_token", kind="append", dtype="bf16", src="bf16", B=16, Hq=32, H=8, D=128,
             page=16, T=1, start=2000, ragged=True, rot=128, pairs="halves", theta=500000.0,
             offset=0, width=0),
        # a video model's frame of 1,560 tokens behind seven earlier ones, pairs
        # side by side
        dict(name="append_frame", kind="append", dtype="bf16", src="bf16", B=1, Hq=24, H=24, D=128,
             page=64, T=1560, start=10920, ragged=False, rot=128, pairs="neighbours",
             theta=10000.0, offset=0, width=0),
        # four prompts at once into empty pages, an odd length, fp16 rows
        dict(name="append_prompt", kind="append", dtype="fp16", src="fp16", B=4, Hq=32, H=8, D=128,
             page=16, T=8191, start=0, ragged=False, rot=128, pairs="halves", theta=10000.0,
             offset=0, width=0),
        # one token of one sequence over a short cache: latency
        dict(name="attend_token", kind="attend", dtype="bf16", B=1, Hq=32, H=8, D=128, page=16, Q=1,
             N=4096, ragged=False, causal=False),
        # a serving step: one token of each of 32 sequences of unlike lengths
        dict(name="attend_tokens", kind="attend", dtype="bf16", B=32, Hq=32, H=8, D=128, page=16,
             Q=1, N=16384, ragged=True, causal=False),
        # one token over one long context with few key heads: the only
        # parallelism is along the keys
        dict(name="attend_long", kind="attend", dtype="bf16", B=1, Hq=16, H=2, D=128, page=64, Q=1,
             N=262144, ragged=False, causal=False),
        # the next chunk of two prompts, causal, narrow heads, odd sizes, fp16
        dict(name="attend_prompt", kind="attend", dtype="fp16", B=2, Hq=16, H=4, D=64, page=32,
             Q=1023, N=5001, ragged=True, causal=True),
        # a frame of queries over eight frames of history: the largest call
        dict(name="attend_frame", kind="attend", dtype="bf16", B=1, Hq=24, H=24, D=128, page=64,
             Q=1560, N=12480, ragged=False, causal=False),
        # a draft of 16 tokens of one sequence, four to a level
        dict(name="tree_one", kind="tree", dtype="bf16", B=1, Hq=32, H=8, D=128, page=16, Q=16,
             N=4096, ragged=False, width=4),
        # drafts of 64 tokens of 16 sequences of unlike lengths, eight to a level
        dict(name="tree_batch", kind="tree", dtype="bf16", B=16, Hq=32, H=8, D=128, page=16, Q=64,
             N=8192, ragged=True, width=8),
        # the accepted tokens of one sequence's draft, up to six of 16, in one layer
        dict(name="commit_one", kind="commit", dtype="bf16", B=1, H=8, D=128, page=16, layers=1,
             N=4096, T=16, M=6),
        # those of 32 sequences' drafts, up to 12 of 64, in eight layers at once
        dict(name="commit_batch", kind="commit", dtype="bf16", B=32, H=8, D=128, page=16, layers=8,
             N=1024, T=64, M=12),
    ]


def _logint(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    """One more case: the operators above over the types, head counts, widths, page
    sizes and lengths that their callers use, odd ones among them."""
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "tree", "tree", "commit"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    D = rng.choice([128, 128, 128, 64, 80, 96])
    H = rng.choice([1, 2, 4, 8, 16, 24])
    page = rng.choice([16, 16, 32, 64, 128])
    ragged = rng.random() < 0.5
    if kind == "commit":
        B = _logint(rng, 1, 64)
        M = _logint(rng, 1, 32)
        T = M + _logint(rng, M, 4 * M + 8)
        layers = _logint(rng, 1, 16)
        N = _logint(rng, 2 * T, max(2 * T, min(4096, 2097152 // (B * H * layers))))
        return dict(kind=kind, dtype=dtype, B=B, H=H, D=D, page=page, layers=layers, N=N, T=T, M=M)
    G = rng.choice([1, 1, 2, 4, 7, 8])
    if kind == "append":
        B = _logint(rng, 1, 32)
        T = _logint(rng, 1, max(1, min(8192, 1048576 // (B * H * (G + 2)))))
        rot = rng.choice([D, D, D // 2]) if D % 32 == 0 else D
        return dict(kind=kind, dtype=dtype, src=rng.choice([dtype, dtype, "fp32"]), B=B, Hq=H * G,
                    H=H, D=D, page=page, T=T, start=rng.choice([0, rng.randint(1, 4096)]),
                    ragged=ragged, rot=rot, pairs=rng.choice(["halves", "neighbours"]),
                    theta=rng.choice([10000.0, 500000.0]),
                    offset=rng.choice([0, 0, _logint(rng, 1000, 1000000)]),
                    width=rng.choice([0, 0, rng.randint(1, 10)]) if T <= 256 else 0)
    B = _logint(rng, 1, 32)
    if kind == "tree":
        Q = _logint(rng, 2, 128)
    else:
        Q = _logint(rng, 2, 2048) if rng.random() < 0.5 else 1
    # rows such that the call is no larger than the largest listed ones
    top = int(200e9 / (4 * B * H * G * Q * 128))
    N = max(Q if kind == "tree" else 1, _logint(rng, 1, max(1, min(262144, top, 4194304 // (B * H)))))
    c = dict(kind=kind, dtype=dtype, B=B, Hq=H * G, H=H, D=D, page=page, Q=Q, N=N, ragged=ragged)
    if kind == "tree":
        return dict(c, width=rng.randint(1, 10))
    return dict(c, causal=Q > 1 and rng.random() < 0.5)


def _lengths(c: dict) -> list:
    """Each sequence's rows, a draft's own among them: unlike ones in a ragged
    batch, the last of which is a slot that holds one token."""
    B, N = c["B"], c["N"]
    if not c.get("ragged"):
        return [N] * B
    n = [max(1, N - b * N * 5 // (8 * B)) for b in range(B)]
    if B > 2:
        n[-1] = 1
    return [max(x, c["Q"]) for x in n] if c["kind"] == "tree" else n


def _starts(c: dict) -> list:
    return [max(0, c["start"] - 97 * b) if c["ragged"] else c["start"] for b in range(c["B"])]


def _levels(n: int, width: int) -> list:
    """The depth of each of n drafted tokens: one root, then `width` to a level."""
    return [0 if t == 0 else 1 + (t - 1) // width for t in range(n)]


def _accepted(c: dict) -> list:
    """How many of its draft's tokens each sequence keeps."""
    return [1 + (5 * b + 3) % c["M"] if c["M"] > 1 else 1 for b in range(c["B"])]


# ---------------------------------------------------------------- inputs
def _tables(gen, c: dict, rows: list):
    """A table [B, widest] of the pages that each sequence's rows need, in random
    order, -1 behind them, and the pool's page count, a few more than needed."""
    need = [-(-n // c["page"]) for n in rows]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _pool(gen, c: dict, pages: int, loud: bool) -> torch.Tensor:
    """[pages, H, page, D] random rows whose amplitude differs by channel (loud: a
    few of them many times, as keys have)."""
    H, D = c["H"], c["D"]
    channel = torch.exp(0.4 * torch.randn((H, 1, D), generator=gen, device=DEV))
    if loud:
        channel = channel * (1 + 3 * (torch.rand((H, 1, D), generator=gen, device=DEV) < 0.02))
    x = torch.empty((pages, H, c["page"], D), device=DEV, dtype=TYPE[c["dtype"]])
    step = max(1, (1 << 27) // (H * c["page"] * D))
    for p in range(0, pages, step):
        part = x[p:p + step]
        part.copy_(torch.randn(part.shape, generator=gen, device=DEV).mul_(channel))
    return x


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    c, s = case, {"case": case}
    B, H, D = c["B"], c["H"], c["D"]
    if c["kind"] == "append":
        T, starts = c["T"], _starts(c)
        s["table"], pages = _tables(gen, c, [x + T for x in starts])
        s["k"], s["v"] = _pool(gen, c, pages, True), _pool(gen, c, pages, False)
        # the Q, K and V columns of a projection's output, as a model has them
        qkv = torch.randn((B, T, c["Hq"] + 2 * H, D), generator=gen, device=DEV).to(TYPE[c["src"]])
        s["q"], s["new_k"], s["new_v"] = qkv.split([c["Hq"], H, H], dim=2)
        s["start"] = torch.tensor(starts, device=DEV, dtype=torch.int32)
        half = torch.arange(c["rot"] // 2, device=DEV, dtype=torch.float64)
        s["freqs"] = (c["theta"] ** (-half / (c["rot"] // 2))).to(torch.float32)
        # positions of their own: those of a draft's levels, or of a cache whose
        # first rows were dropped
        s["positions"] = None
        if c["offset"] or c["width"]:
            step = _levels(T, c["width"]) if c["width"] else list(range(T))
            step = torch.tensor(step, device=DEV, dtype=torch.int32)
            s["positions"] = s["start"][:, None] + step + c["offset"]
        return s
    if c["kind"] == "commit":
        T, M = c["T"], c["M"]
        s["table"], pages = _tables(gen, c, [c["N"]] * B)
        s["pools"] = [(_pool(gen, c, pages, True), _pool(gen, c, pages, False))
                      for _ in range(c["layers"])]
        s["start"] = torch.full((B,), c["N"] - T, device=DEV, dtype=torch.int32)
        # the first token stays where it is and the others come from behind all
        # places they go to, so that a second pass moves the same values
        path = torch.rand((B, T - M), generator=gen, device=DEV).argsort(1)[:, :M - 1] + M
        s["rows"] = torch.zeros((B, M), device=DEV, dtype=torch.int32)
        s["rows"][:, 1:] = path.sort(1).values
        s["count"] = torch.tensor(_accepted(c), device=DEV, dtype=torch.int32)
        return s
    lengths = _lengths(c)
    s["table"], pages = _tables(gen, c, lengths)
    s["k"], s["v"] = _pool(gen, c, pages, True), _pool(gen, c, pages, False)
    s["length"] = torch.tensor(lengths, device=DEV, dtype=torch.int32)
    q = torch.randn((B, c["Q"], c["Hq"], D), generator=gen, device=DEV)
    s["q"] = q.to(TYPE[c["dtype"]])
    if c["kind"] == "tree":
        # a parent of each token among those one level up; -1 for the root
        w, level = c["width"], torch.tensor(_levels(c["Q"], c["width"]), device=DEV)
        pick = (torch.rand((B, c["Q"]), generator=gen, device=DEV) * w).long().clamp_max(w - 1)
        s["parents"] = torch.where(level > 1, 1 + (level - 2) * w + pick, level - 1).to(torch.int32)
    return s


# ---------------------------------------------------------------- the plain forms
def _slots(c: dict, table: torch.Tensor, rows: torch.Tensor):
    """Page and row in the page of rows [B, n] of each sequence."""
    page = table.gather(1, (rows // c["page"]).long()).long()
    return page, (rows % c["page"]).long()


def _rotate(c: dict, x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [B, T, heads, D] fp32 by angles [B, T, 1, rot / 2]: pair i is columns i and
    i + rot / 2, or 2 i and 2 i + 1; the columns from rot on stay."""
    rot = c["rot"]
    y = x.clone()
    if c["pairs"] == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2] = a * cos - b * sin
        y[..., rot // 2:rot] = b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2] = a * cos - b * sin
        y[..., 1:rot:2] = b * cos + a * sin
    return y


def _plain_append(s: dict):
    c = s["case"]
    dtype = TYPE[c["dtype"]]
    rows = s["start"][:, None] + torch.arange(c["T"], device=DEV)
    at = rows if s["positions"] is None else s["positions"]
    angle = at.to(torch.float64)[..., None, None] * s["freqs"].to(torch.float64)
    cos, sin = torch.cos(angle).to(torch.float32), torch.sin(angle).to(torch.float32)
    q = _rotate(c, s["q"].to(torch.float32), cos, sin).to(dtype)
    k = _rotate(c, s["new_k"].to(torch.float32), cos, sin).to(dtype)
    page, row = _slots(c, s["table"], rows)
    s["k"][page, :, row] = k
    s["v"][page, :, row] = s["new_v"].to(dtype)
    return q, s["k"], s["v"]


def _gathered(s: dict, pool: torch.Tensor) -> torch.Tensor:
    """fp32 rows [B, H, N, D] of each sequence, zeros where it has no page."""
    c = s["case"]
    page = s["table"].long().clamp_min(0)
    x = pool[page].to(torch.float32)                       # [B, pages, H, page, D]
    x = x.masked_fill_((s["table"] < 0)[:, :, None, None, None], 0.0)
    x = x.permute(0, 2, 1, 3, 4).reshape(c["B"], c["H"], -1, c["D"])
    return x[:, :, :c["N"]]


def _hidden(s: dict, n: int) -> torch.Tensor:
    """[B, Q, n] truth values: the rows that a query does not see."""
    c = s["case"]
    B, Q = c["B"], c["Q"]
    at, length = torch.arange(n, device=DEV), s["length"].view(B, 1, 1)
    if c["kind"] == "attend":
        end = length.expand(B, Q, 1)
        if c["causal"]:
            end = end - Q + 1 + torch.arange(Q, device=DEV).view(1, Q, 1)
        return at >= end
    # a draft: the rows before it, and of its own those on the way to the root
    sees = torch.zeros((B, Q, Q), device=DEV, dtype=torch.bool)
    node = torch.arange(Q, device=DEV).expand(B, Q)
    for _ in range(1 + _levels(Q, c["width"])[-1]):
        sees |= ((node[..., None] == torch.arange(Q, device=DEV)) & (node >= 0)[..., None])
        node = torch.where(node >= 0, s["parents"].long().gather(1, node.clamp_min(0)), -1)
    own_row = (at - length + Q).expand(B, Q, n)
    mine = sees.gather(2, own_row.clamp(0, Q - 1)) & (own_row < Q)
    return ~torch.where(own_row < 0, at < length, mine)


def _plain_attend(s: dict):
    c = s["case"]
    B, H, G, Q, N, D = c["B"], c["H"], c["Hq"] // c["H"], c["Q"], c["N"], c["D"]
    q = s["q"].to(torch.float32).view(B, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Q, D)
    k = _gathered(s, s["k"])
    z = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).view(B, H, G, Q, N)
    del k
    z = z.masked_fill_(_hidden(s, N)[:, None, None], -INF)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - top.clamp_min(-1e30))
    del z
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, H, G * Q, N), _gathered(s, s["v"])).view(B, H, G, Q, D)
    o = o / total.clamp_min(1e-30)
    lse = (top + torch.log(total))[..., 0].reshape(B, c["Hq"], Q)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, c["Hq"], D).to(s["q"].dtype), lse


def _plain_commit(s: dict):
    c = s["case"]
    j = torch.arange(c["M"], device=DEV, dtype=torch.int32)
    kept = j < s["count"][:, None]                          # the others stay
    to = s["start"][:, None] + j
    tp, tr = _slots(c, s["table"], to)
    fp, fr = _slots(c, s["table"], torch.where(kept, s["start"][:, None] + s["rows"], to))
    for pools in s["pools"]:
        for pool in pools:
            pool[tp, :, tr] = pool[fp, :, fr]
    return [x for pools in s["pools"] for x in pools] + [s["start"] + s["count"]]


def run(state: dict):
    s = state
    c = s["case"]
    if own:
        from nanokv_amd import ops
        if c["kind"] == "append":
            q = ops.paged_append(ops.PagedCache(s["k"], s["v"]), s["table"], s["new_k"], s["new_v"],
                                 s["start"], q=s["q"], freqs=s["freqs"], positions=s["positions"],
                                 interleaved=c["pairs"] == "neighbours")
            return q, s["k"], s["v"]
        if c["kind"] == "attend":
            return ops.paged_attend(s["q"], ops.PagedCache(s["k"], s["v"]), s["table"], s["length"],
                                    max_length=c["N"], causal=c["causal"])
        if c["kind"] == "tree":
            return ops.paged_attend(s["q"], ops.PagedCache(s["k"], s["v"]), s["table"], s["length"],
                                    max_length=c["N"], parents=s["parents"])
        length = ops.paged_commit([ops.PagedCache(k, v) for k, v in s["pools"]], s["table"],
                                  s["start"], s["rows"], s["count"])
        return [x for pools in s["pools"] for x in pools] + [length]
    if c["kind"] == "append":
        return _plain_append(s)
    if c["kind"] == "commit":
        return _plain_commit(s)
    return _plain_attend(s)


# ---------------------------------------------------------------- what a pass needs
def work(case: dict) -> dict:
    c = case
    D, H = c["D"], c["H"]
    if c["kind"] == "append":
        rows = c["B"] * c["T"] * (c["Hq"] + 2 * H)
        turned = c["B"] * c["T"] * (c["Hq"] + H) * c["rot"]
        # source rows in, rotated queries and the pool's rows out
        return {"bytes": rows * D * (BYTES[c["src"]] + BYTES[c["dtype"]]), "flops": 3 * turned}
    if c["kind"] == "commit":
        # each moved row in and out, for keys and values in each layer
        moved = sum(n - 1 for n in _accepted(c)) * H * c["layers"]
        return {"bytes": moved * D * 2 * 4 + c["B"] * (c["M"] + 3) * 4, "flops": 0}
    n, Q = _lengths(c), c["Q"]
    if c["kind"] == "tree":
        own_rows = sum(x + 1 for x in _levels(Q, c["width"]))
        pairs = sum((x - Q) * Q + own_rows for x in n) * c["Hq"]
    elif c["causal"]:
        pairs = sum(sum(max(0, x - Q + 1 + t) for t in range(Q)) for x in n) * c["Hq"]
    else:
        pairs = sum(n) * Q * c["Hq"]
    rows = c["B"] * Q * c["Hq"]
    return {"bytes": sum(n) * H * 4 * D + rows * (4 * D + 4), "flops": 4 * pairs * D}


# ---------------------------------------------------------------- 64 bits
def exact(case: dict, seed: int):
    """The results in 64 bits, sequence by sequence and head by head."""
    c = case
    s = prepare(c, seed)
    f64, page = torch.float64, c["page"]
    table = s["table"].tolist()
    if c["kind"] == "commit":
        count, rows = _accepted(c), s["rows"].tolist()
        first = c["N"] - c["T"]
        pools = [x.to(f64) for pair in s["pools"] for x in pair]
        for b in range(c["B"]):
            came = [first + rows[b][j] for j in range(count[b])]
            src = [(table[b][i // page], i % page) for i in came]
            dst = [(table[b][i // page], i % page) for i in range(first, first + count[b])]
            for x in pools:
                held = [x[p, :, r].clone() for p, r in src]
                for (p, r), y in zip(dst, held):
                    x[p, :, r] = y
        return pools + [None]
    if c["kind"] == "append":
        T, rot = c["T"], c["rot"]
        k, v = s["k"].to(f64), s["v"].to(f64)
        q = s["q"].to(f64)
        new = s["new_k"].to(f64)
        for b, first in enumerate(_starts(c)):
            if s["positions"] is None:
                at = torch.arange(first, first + T, device=DEV, dtype=f64)
            else:
                at = s["positions"][b].to(f64)
            turn = torch.polar(torch.ones((), device=DEV, dtype=f64),
                               torch.outer(at, s["freqs"].to(f64)))[:, None]
            for x in (q, new):
                part = x[b, :, :, :rot]
                if c["pairs"] == "halves":
                    z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous())
                    x[b, :, :, :rot] = torch.cat([(z * turn).real, (z * turn).imag], -1)
                else:
                    z = torch.view_as_complex(part.reshape(*part.shape[:2], -1, 2).contiguous())
                    x[b, :, :, :rot] = torch.view_as_real(z * turn).flatten(2)
            t = 0
            while t < T:
                at_page, at_row = table[b][(first + t) // page], (first + t) % page
                n = min(T - t, page - at_row)
                k[at_page, :, at_row:at_row + n] = new[b, t:t + n].transpose(0, 1)
                v[at_page, :, at_row:at_row + n] = s["new_v"][b, t:t + n].to(f64).transpose(0, 1)
                t += n
        return q, k, v
    G, Q, D = c["Hq"] // c["H"], c["Q"], c["D"]
    out = torch.zeros((c["B"], Q, c["Hq"], D), device=DEV, dtype=f64)
    lse = torch.full((c["B"], c["Hq"], Q), -INF, device=DEV, dtype=f64)
    parents = s["parents"].tolist() if c["kind"] == "tree" else None
    for b, n in enumerate(_lengths(c)):
        mask = None
        if parents:
            mask = torch.zeros((Q, n), dtype=torch.bool)
            mask[:, n - Q:] = True
            for t in range(Q):
                a = t
                while a >= 0:
                    mask[t, n - Q + a] = False
                    a = parents[b][a]
            mask = mask.to(DEV)
        elif c["causal"]:
            sees = torch.arange(n - Q + 1, n + 1, device=DEV)
            mask = torch.arange(n, device=DEV)[None] >= sees[:, None]
        pages = torch.tensor(table[b][:-(-n // page)], device=DEV)
        for h in range(c["H"]):
            k = s["k"][pages, h].reshape(-1, D)[:n].to(f64).T.contiguous()
            v = s["v"][pages, h].reshape(-1, D)[:n].to(f64)
            for g in range(h * G, (h + 1) * G):
                z = (s["q"][b, :, g].to(f64) @ k) / math.sqrt(D)
                if mask is not None:
                    z = z.masked_fill(mask, -INF)
                lse[b, g] = torch.logsumexp(z, 1)
                out[b, :, g] = torch.nan_to_num(torch.softmax(z, 1)) @ v
    return out, lse
