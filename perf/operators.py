"""Measured operators: the 8-bit key/value cache.

A cache holds the keys and values of B sequences and H heads in 8 bits (int8
or e4m3), with one fp32 scale for each block of 64 tokens and head.  Four
operators work on it: the write of new tokens, the attention over it, the
attention weight that each key has received, summed over the queries, and the
eviction of the tokens that received least.

listed() and draw() name the cases, prepare() makes a case's inputs on the GPU
from a seed, run() is one pass: through the library's entry points where `own`
is true, in elementary torch operations otherwise.  work() says what a pass
cannot do without, exact() gives the results in 64 bits.

Caches are made here by plain torch, so a case's inputs do not depend on the
library.  8-bit outputs are returned as the numbers that their codes are (to be
multiplied by the returned scales): e4m3 codes as the float8 tensor itself,
int8 codes in fp16, which holds them exactly.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK = 64                       # tokens that share a scale
TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
TINY = 2.0 ** -64                # the least amplitude a block's scale stands for
INF = float("inf")


# ---------------------------------------------------------------- the cases
def listed() -> list:
    return [
        # one new token of each of 16 sequences, somewhere in a block: the
        # smallest call, made once per layer and generated token
        dict(name="write_token", kind="write", fmt="e4m3", dtype="bf16", B=16, H=8, D=128, T=1,
             start=2000, cap=4096, ragged=True),
        # a video model's frame of 1,560 tokens behind seven earlier ones,
        # which end inside a block
        dict(name="write_frame", kind="write", fmt="e4m3", dtype="bf16", B=1, H=24, D=128, T=1560,
             start=10920, cap=12480, ragged=False),
        # four prompts at once into an empty cache, an odd length, fp16 rows
        dict(name="write_prompt", kind="write", fmt="e4m3", dtype="fp16", B=4, H=8, D=128, T=8191,
             start=0, cap=8192, ragged=False),
        # one token of one sequence over a short cache: latency
        dict(name="attend_token", kind="attend", fmt="int8", dtype="bf16", B=1, Hq=32, H=8, D=128,
             Q=1, N=4096, cap=4096, ragged=False, causal=False),
        # a serving step: one token of each of 32 sequences of unlike lengths
        dict(name="attend_tokens", kind="attend", fmt="e4m3", dtype="bf16", B=32, Hq=32, H=8,
             D=128, Q=1, N=16384, cap=16384, ragged=True, causal=False),
        # one token over one long context with few key heads: the only
        # parallelism is along the keys
        dict(name="attend_long", kind="attend", fmt="int8", dtype="bf16", B=1, Hq=16, H=2, D=128,
             Q=1, N=262144, cap=262144, ragged=False, causal=False),
        # a frame of queries over eight frames of history: the largest call
        dict(name="attend_frame", kind="attend", fmt="int8", dtype="bf16", B=1, Hq=24, H=24,
             D=128, Q=1560, N=12480, cap=12480, ragged=False, causal=False),
        # the next chunk of two prompts, causal, narrow heads, odd sizes, fp16
        dict(name="attend_prompt", kind="attend", fmt="e4m3", dtype="fp16", B=2, Hq=16, H=4, D=64,
             Q=1023, N=5001, cap=5056, ragged=True, causal=True),
        # the weight each cached token received from one decoding step
        dict(name="mass_token", kind="mass", fmt="e4m3", dtype="bf16", B=8, Hq=32, H=8, D=128, Q=1,
             N=8192, cap=8192, ragged=True, causal=False),
        # the weight each cached token received from a frame of queries
        dict(name="mass_frame", kind="mass", fmt="int8", dtype="bf16", B=1, Hq=24, H=24, D=128,
             Q=1560, N=12480, cap=12480, ragged=False, causal=False),
        # a short cache back to its budget
        dict(name="evict_short", kind="evict", fmt="e4m3", B=1, H=8, D=128, N=2048, cap=2048,
             keep=1536, sink=4, recent=256, ragged=False),
        # eight long sequences of unlike lengths down to a quarter
        dict(name="evict_long", kind="evict", fmt="e4m3", B=8, H=8, D=128, N=32768, cap=32768,
             keep=8192, sink=16, recent=1024, ragged=True),
    ]


def _logint(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _blocks(n: int) -> int:
    return -(-n // BLOCK) * BLOCK


def draw(rng) -> dict:
    """One more case: the operators above over the formats, types, head counts,
    widths and lengths that their callers use, odd ones among them."""
    kind = rng.choice(["write", "attend", "attend", "attend", "mass", "evict"])
    fmt = rng.choice(["int8", "e4m3"])
    D = rng.choice([128, 128, 128, 64, 80, 96])
    H = rng.choice([1, 2, 4, 8, 16, 24])
    ragged = rng.random() < 0.5
    if kind == "write":
        B = _logint(rng, 1, 32)
        T = _logint(rng, 1, max(1, min(16384, 262144 // (B * H))))
        start = rng.choice([0, rng.randint(1, 4096)])
        return dict(kind=kind, fmt=fmt, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), B=B,
                    H=H, D=D, T=T, start=start, cap=_blocks(start + T + rng.randint(0, 200)),
                    ragged=ragged)
    if kind == "evict":
        B = _logint(rng, 1, 16)
        N = _logint(rng, 64, max(64, min(131072, 2097152 // (B * H))))
        keep = _logint(rng, max(1, N // 16), N)
        sink = rng.randint(0, keep // 4)
        return dict(kind=kind, fmt=fmt, B=B, H=H, D=D, N=N, cap=_blocks(N + rng.randint(0, 200)),
                    keep=keep, sink=sink, recent=rng.randint(0, (keep - sink) // 2),
                    ragged=ragged)
    G = rng.choice([1, 1, 2, 4, 7, 8])
    B = _logint(rng, 1, 32)
    many = rng.random() < 0.5
    Q = _logint(rng, 2, 2048) if many else 1
    # keys such that the call is no larger than the largest listed one
    top = int(200e9 / (4 * B * H * G * Q * 128))
    N = _logint(rng, 1, max(1, min(262144, top, 4194304 // (B * H))))
    return dict(kind=kind, fmt=fmt, dtype=rng.choice(["bf16", "bf16", "fp16"]), B=B, Hq=H * G, H=H,
                D=D, Q=Q, N=N, cap=_blocks(N + rng.randint(0, 200)), ragged=ragged,
                causal=many and rng.random() < 0.5)


def _lengths(c: dict) -> list:
    """Each sequence's length: unlike ones in a ragged batch, the last of which
    is a slot that holds one token."""
    B, N = c["B"], c["N"]
    if not c["ragged"]:
        return [N] * B
    n = [max(1, N - b * N * 5 // (8 * B)) for b in range(B)]
    if B > 2:
        n[-1] = 1
    return n


def _starts(c: dict) -> list:
    return [max(0, c["start"] - 97 * b) if c["ragged"] else c["start"] for b in range(c["B"])]


# ---------------------------------------------------------------- inputs
def _codes(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """x, already divided by its scale, in 8 bits: to the nearest, ties to even."""
    if fmt == "int8":
        return torch.clamp(torch.round(x), -127.0, 127.0).to(torch.int8)
    return torch.clamp(x, -448.0, 448.0).to(torch.float8_e4m3fn)


def _pitch(D: int) -> int:
    return 64 if D <= 64 else 128


def _cache(gen, c: dict, loud: bool):
    """Codes [B, H, cap, pitch] and scales [B, H, cap / 64] of random rows whose
    amplitude differs by channel (loud: a few of them many times, as keys have)
    and from block to block."""
    B, H, cap, D = c["B"], c["H"], c["cap"], c["D"]
    x = torch.randn((B, H, cap, D), generator=gen, device=DEV)
    channel = torch.exp(0.4 * torch.randn((H, 1, D), generator=gen, device=DEV))
    if loud:
        channel = channel * (1 + 3 * (torch.rand((H, 1, D), generator=gen, device=DEV) < 0.02))
    x = x.mul_(channel).view(B, H, cap // BLOCK, BLOCK, D)
    x = x.mul_(torch.exp(0.3 * torch.randn((B, H, cap // BLOCK, 1, 1), generator=gen, device=DEV)))
    scale = x.abs().amax((3, 4)).clamp_min(TINY) / TOP[c["fmt"]]
    codes = _codes(x / scale[..., None, None], c["fmt"]).view(B, H, cap, D)
    if D < _pitch(D):
        wide = torch.zeros((B, H, cap, _pitch(D)), device=DEV, dtype=codes.dtype)
        wide.view(torch.uint8)[..., :D] = codes.view(torch.uint8)
        codes = wide
    return codes, scale


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    c, s = case, {"case": case}
    B, H, D = c["B"], c["H"], c["D"]
    s["k"], s["ks"] = _cache(gen, c, True)
    s["v"], s["vs"] = _cache(gen, c, False)
    if c["kind"] == "write":
        # the K and V columns of a projection's output, as a model has them
        kv = torch.randn((B, c["T"], 2, H, D), generator=gen, device=DEV)
        s["new_k"], s["new_v"] = kv.to(TYPE[c["dtype"]]).unbind(2)
        s["start"] = torch.tensor(_starts(c), device=DEV, dtype=torch.int32)
        return s
    s["length"] = torch.tensor(_lengths(c), device=DEV, dtype=torch.int32)
    if c["kind"] == "evict":
        # a few tokens carry most of the weight; many have received none
        mass = torch.exp(2.5 * torch.randn((B, H, c["cap"]), generator=gen, device=DEV))
        s["mass"] = mass * (torch.rand((B, H, c["cap"]), generator=gen, device=DEV) < 0.9)
        cap = _blocks(c["keep"])
        s["out"] = [torch.zeros((B, H, cap, _pitch(D)), device=DEV, dtype=CODE[c["fmt"]]),
                    torch.zeros((B, H, cap, _pitch(D)), device=DEV, dtype=CODE[c["fmt"]]),
                    torch.zeros((B, H, cap // BLOCK), device=DEV),
                    torch.zeros((B, H, cap // BLOCK), device=DEV),
                    torch.zeros((B, H, cap), device=DEV)]
        return s
    q = torch.randn((B, c["Q"], c["Hq"], D), generator=gen, device=DEV)
    s["q"] = q.to(TYPE[c["dtype"]])
    if c["kind"] == "mass":
        s["lse"] = _lse(s)
        s["mass"] = torch.rand((B, H, c["cap"]), generator=gen, device=DEV)
        s["sum"] = torch.empty_like(s["mass"])
    return s


# ---------------------------------------------------------------- the plain forms
def _values(codes: torch.Tensor, scale: torch.Tensor, n: int, D: int) -> torch.Tensor:
    """fp32 values [B, H, n, D] of a cache's first n rows."""
    per_row = scale.repeat_interleave(BLOCK, dim=2)[:, :, :n, None]
    return codes[:, :, :n, :D].to(torch.float32) * per_row


def _scores(s: dict) -> torch.Tensor:
    """Scaled scores [B, H, G, Q, N], -inf where the query does not see the key."""
    c = s["case"]
    B, H, G, Q, N, D = c["B"], c["H"], c["Hq"] // c["H"], c["Q"], c["N"], c["D"]
    q = s["q"].to(torch.float32).view(B, Q, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * Q, D)
    k = _values(s["k"], s["ks"], N, D)
    z = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).view(B, H, G, Q, N)
    end = s["length"].view(B, 1, 1, 1, 1)
    if c["causal"]:
        end = end - Q + 1 + torch.arange(Q, device=DEV).view(1, 1, 1, Q, 1)
    return z.masked_fill_(torch.arange(N, device=DEV) >= end, -INF)


def _lse(s: dict) -> torch.Tensor:
    """Natural-log row sums [B, Hq, Q], -inf for a row that sees nothing."""
    c = s["case"]
    z = _scores(s)
    top = z.amax(-1, keepdim=True)
    total = torch.exp(z - top.clamp_min(-1e30)).sum(-1)
    return (top[..., 0] + torch.log(total)).reshape(c["B"], c["Hq"], c["Q"])


def _plain_attend(s: dict):
    c = s["case"]
    B, H, G, Q, N, D = c["B"], c["H"], c["Hq"] // c["H"], c["Q"], c["N"], c["D"]
    z = _scores(s)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - top.clamp_min(-1e30))
    total = p.sum(-1, keepdim=True)
    v = _values(s["v"], s["vs"], N, D)
    o = torch.matmul(p.view(B, H, G * Q, N), v).view(B, H, G, Q, D) / total.clamp_min(1e-30)
    lse = (top + torch.log(total))[..., 0].reshape(B, c["Hq"], Q)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, c["Hq"], D).to(s["q"].dtype), lse


def _plain_mass(s: dict):
    c = s["case"]
    B, H, G, Q, N = c["B"], c["H"], c["Hq"] // c["H"], c["Q"], c["N"]
    lse = s["lse"].view(B, H, G, Q, 1)
    p = torch.exp(_scores(s) - lse.masked_fill(lse == -INF, INF))
    mass = s["mass"].clone()
    mass[:, :, :N] += p.sum((2, 3))
    return mass


def _plain_write_one(s: dict, codes, scale, x):
    c = s["case"]
    B, H, D, T, fmt = c["B"], c["H"], c["D"], c["T"], c["fmt"]
    x = x.to(torch.float32).permute(0, 2, 1, 3)                       # [B, H, T, D]
    start = s["start"].to(torch.int64)
    at = (start[:, None] + torch.arange(T, device=DEV))[:, None, :].expand(B, H, T)
    # each touched block's amplitude, and its scale: the larger of what the new
    # rows need and what the rows before them have
    top = torch.zeros_like(scale).scatter_reduce(2, at // BLOCK, x.abs().amax(-1), "amax")
    touched = torch.zeros_like(scale).scatter(2, at // BLOCK, 1.0) > 0
    need = top.clamp_min(TINY) / TOP[fmt]
    first = (start // BLOCK)[:, None, None].expand(B, H, 1)
    kept = (start % BLOCK)[:, None, None]                              # rows before them
    old = scale.gather(2, first)
    grown = torch.maximum(old, need.gather(2, first))
    new = torch.where(touched, need, scale)
    new = new.scatter(2, first, torch.where(kept > 0, grown, new.gather(2, first)))
    # the rows before them, on the grown scale
    out = codes.clone()
    row = first * BLOCK + torch.arange(BLOCK, device=DEV)
    row_w = row[..., None].expand(B, H, BLOCK, out.shape[3])
    raw = out.view(torch.uint8)
    was = raw.gather(2, row_w).view(out.dtype)
    again = _codes(was.to(torch.float32) * (old / grown)[..., None], fmt)
    again = torch.where((torch.arange(BLOCK, device=DEV) < kept)[..., None],
                        again.view(torch.uint8), was.view(torch.uint8))
    raw.scatter_(2, row_w, again)
    # the new rows
    y = _codes(x / new.gather(2, at // BLOCK)[..., None], fmt).view(torch.uint8)
    wide = torch.zeros((B, H, T, out.shape[3]), device=DEV, dtype=torch.uint8)
    wide[..., :D] = y
    raw.scatter_(2, at[..., None].expand_as(wide), wide)
    return out, new


def _plain_evict(s: dict):
    c = s["case"]
    B, H, keep, fmt = c["B"], c["H"], c["keep"], c["fmt"]
    n = s["length"].to(torch.int64)[:, None, None]
    at = torch.arange(c["cap"], device=DEV)
    # the first tokens and the last ones before all others, what is not there last
    rank = s["mass"].masked_fill((at < c["sink"]) | (at >= n - c["recent"]), INF)
    rank = rank.masked_fill(at >= n, -INF)
    best = torch.sort(rank, dim=2, descending=True, stable=True).indices[:, :, :keep]
    there = torch.arange(keep, device=DEV) < n
    rows = best.masked_fill(best >= n, c["cap"]).sort(dim=2).values
    src = rows.clamp_max(c["cap"] - 1)
    cap = _blocks(keep)
    got = []
    for codes, scale, buf in ((s["k"], s["ks"], s["out"][2]), (s["v"], s["vs"], s["out"][3])):
        per_row = scale.gather(2, src // BLOCK) * there
        wide = torch.zeros((B, H, cap), device=DEV)
        wide[:, :, :keep] = per_row
        new = wide.view(B, H, cap // BLOCK, BLOCK).amax(3)
        used = new.repeat_interleave(BLOCK, dim=2)[:, :, :keep]
        row_w = src[..., None].expand(B, H, keep, codes.shape[3])
        was = codes.view(torch.uint8).gather(2, row_w).view(codes.dtype).to(torch.float32)
        y = _codes(was * (per_row / used.clamp_min(1e-38))[..., None], fmt)
        out = torch.zeros((B, H, cap, codes.shape[3]), device=DEV, dtype=torch.uint8)
        out[:, :, :keep] = y.view(torch.uint8) * there[..., None]
        got += [out.view(codes.dtype), new]
    mass = torch.zeros((B, H, cap), device=DEV)
    mass[:, :, :keep] = s["mass"].gather(2, src) * there
    rows = rows.masked_fill(~there, -1).to(torch.int32)
    return got[0], got[2], got[1], got[3], mass, rows, s["length"].clamp_max(keep)


def _numbers(codes: torch.Tensor) -> torch.Tensor:
    return codes.to(torch.float16) if codes.dtype == torch.int8 else codes


def run(state: dict):
    s = state
    c = s["case"]
    if own:
        from nanokv_amd import ops
        cache = ops.Cache8(s["k"], s["v"], s["ks"], s["vs"], c["D"])
        if c["kind"] == "write":
            ops.cache8_write(cache, s["new_k"], s["new_v"], s["start"])
            return _numbers(s["k"]), _numbers(s["v"]), s["ks"], s["vs"]
        if c["kind"] == "attend":
            return ops.cache8_attend(s["q"], cache, s["length"], max_length=c["N"],
                                     causal=c["causal"])
        if c["kind"] == "mass":
            return ops.cache8_mass(s["q"], cache, s["lse"], s["mass"], s["length"], out=s["sum"],
                                   max_length=c["N"], causal=c["causal"])
        out = ops.Cache8(*s["out"][:4], c["D"])
        rows, length = ops.cache8_evict(cache, s["mass"], s["length"], out, s["out"][4],
                                        keep=c["keep"], sink=c["sink"], recent=c["recent"],
                                        max_length=c["N"])
        return (_numbers(out.k), _numbers(out.v), out.k_scale, out.v_scale, s["out"][4], rows,
                length)
    if c["kind"] == "write":
        k, ks = _plain_write_one(s, s["k"], s["ks"], s["new_k"])
        v, vs = _plain_write_one(s, s["v"], s["vs"], s["new_v"])
        return _numbers(k), _numbers(v), ks, vs
    if c["kind"] == "attend":
        return _plain_attend(s)
    if c["kind"] == "mass":
        return _plain_mass(s)
    k, v, *rest = _plain_evict(s)
    return (_numbers(k), _numbers(v), *rest)


# ---------------------------------------------------------------- what a pass needs
def work(case: dict) -> dict:
    c = case
    D, H = c["D"], c["H"]
    if c["kind"] == "write":
        rows = c["B"] * H * c["T"]
        # source rows in, codes and scales out, for keys and values
        return {"bytes": 2 * rows * D * (BYTES[c["dtype"]] + 1) + 8 * (rows / BLOCK + c["B"] * H),
                "flops": 2 * 3 * rows * D}
    n = _lengths(c)
    if c["kind"] == "evict":
        left = sum(min(x, c["keep"]) for x in n) * H
        # every weight in, the kept rows in and out with their weights and indices
        return {"bytes": 4 * sum(n) * H + left * (4 * D + 8 + 8 / BLOCK * 2), "flops": sum(n) * H}
    G, Q = c["Hq"] // H, c["Q"]
    if c["causal"]:
        pairs = sum(sum(max(0, x - Q + 1 + t) for t in range(Q)) for x in n) * c["Hq"]
    else:
        pairs = sum(n) * Q * c["Hq"]
    keys = sum(n) * H
    rows = c["B"] * Q * c["Hq"]
    if c["kind"] == "mass":
        return {"bytes": keys * (D + 4 / BLOCK + 8) + rows * (2 * D + 4), "flops": 2 * pairs * D}
    return {"bytes": keys * 2 * (D + 4 / BLOCK) + rows * (4 * D + 4), "flops": 4 * pairs * D}


# ---------------------------------------------------------------- 64 bits
def exact(case: dict, seed: int):
    """The results in 64 bits, head by head; None in the place of codes and
    indices, which are compared as they are."""
    c = case
    s = prepare(c, seed)
    B, H, D, f64 = c["B"], c["H"], c["D"], torch.float64
    if c["kind"] == "write":
        scales = []
        for old, x in ((s["ks"], s["new_k"]), (s["vs"], s["new_v"])):
            new = old.to(f64)
            for b, first in enumerate(_starts(c)):
                t = 0
                while t < c["T"]:
                    blk = (first + t) // BLOCK
                    n = min(c["T"] - t, (blk + 1) * BLOCK - first - t)
                    top = x[b, t:t + n].to(f64).abs().amax((0, 2)).clamp_min(TINY) / TOP[c["fmt"]]
                    begins = (first + t) % BLOCK == 0
                    new[b, :, blk] = top if begins else torch.maximum(top, new[b, :, blk])
                    t += n
            scales.append(new)
        return None, None, scales[0], scales[1]
    lengths = _lengths(c)
    if c["kind"] == "evict":
        cap, keep = _blocks(c["keep"]), c["keep"]
        ks, vs = (torch.zeros((B, H, cap // BLOCK), dtype=f64) for _ in range(2))
        mass = torch.zeros((B, H, cap), dtype=f64)
        weight, sk, sv = (s[x].cpu().to(f64) for x in ("mass", "ks", "vs"))
        for b in range(B):
            n = lengths[b]
            lo, hi = min(c["sink"], n), max(min(c["sink"], n), n - c["recent"])
            for h in range(H):
                rows = list(range(n))
                if n > keep:
                    w = weight[b, h, lo:hi]
                    order = sorted(range(hi - lo), key=lambda i, w=w.tolist(): (-w[i], i))
                    middle = [lo + i for i in order[:keep - lo - (n - hi)]]
                    rows = sorted(list(range(lo)) + middle + list(range(hi, n)))
                at = torch.tensor(rows)
                mass[b, h, :len(rows)] = weight[b, h, at]
                slot = torch.arange(len(rows)) // BLOCK
                ks[b, h].scatter_reduce_(0, slot, sk[b, h, at // BLOCK], "amax")
                vs[b, h].scatter_reduce_(0, slot, sv[b, h, at // BLOCK], "amax")
        return None, None, ks, vs, mass, None, None
    G, Q = c["Hq"] // H, c["Q"]
    out = torch.zeros((B, Q, c["Hq"], D), device=DEV, dtype=f64)
    lse = torch.full((B, c["Hq"], Q), -INF, device=DEV, dtype=f64)
    mass = s["mass"].to(f64) if c["kind"] == "mass" else None
    for b in range(B):
        n = lengths[b]
        if c["causal"]:
            seen = n - Q + 1 + torch.arange(Q, device=DEV)
            hidden = torch.arange(n, device=DEV)[None] >= seen[:, None]
        for h in range(H):
            per_row = s["ks"][b, h].to(f64).repeat_interleave(BLOCK)[:n, None]
            k = (s["k"][b, h, :n, :D].to(f64) * per_row).T.contiguous()
            if mass is None:
                per_row = s["vs"][b, h].to(f64).repeat_interleave(BLOCK)[:n, None]
                v = s["v"][b, h, :n, :D].to(f64) * per_row
            for g in range(h * G, (h + 1) * G):
                z = (s["q"][b, :, g].to(f64) @ k) / math.sqrt(D)
                if c["causal"]:
                    z = z.masked_fill(hidden, -INF)
                if mass is None:
                    lse[b, g] = torch.logsumexp(z, 1)
                    out[b, :, g] = torch.nan_to_num(torch.softmax(z, 1)) @ v
                else:
                    part = torch.exp(z - s["lse"][b, g].to(f64)[:, None])
                    mass[b, h, :n] += torch.nan_to_num(part).sum(0)
    return (out, lse) if mass is None else mass
