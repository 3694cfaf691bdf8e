"""Rows with gaps between them (slices of a fused projection) that a call of the paged
cache writes: refused where they overlap what the call reads, and taken where they lie
between it.  On the host, against a plain search over the rows; nothing is launched."""
import ctypes
import itertools
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from nanokv_amd import _lib
from tests.test_device_attributes import SHIM
from tests.test_paged import INV, PTR, attend_args, cache, refused, rotated, set_fields

V = PTR + (1 << 24)
ROWS, Q, OUT = PTR + (4 << 24), PTR + (6 << 24), PTR + (7 << 24)
PITCH = 8 * 64                # elements of a token in a fused buffer of 4 + 2 + 2 heads


def at(name, base, sb=4 * PITCH, st=PITCH, sh=64):
    field = {"q_out": "o"}.get(name, name)
    return {name: base, f"{field}_sb": sb, f"{field}_st": st, f"{field}_sh": sh}


def fused(base):
    """q, k and v in one buffer, each token's heads side by side."""
    return {**at("q", base), **at("k", base + 4 * 64 * 2), **at("v", base + 6 * 64 * 2)}


@pytest.mark.parametrize("kw", [
    at("q_out", V - 2 * 1024 + 512),                            # the last token's heads in the pool
    at("q_out", PTR),                                           # over the pool of keys
    at("q_out", PTR + (3 << 24) - 496), at("q_out", PTR + (8 << 24) - 3 * PITCH * 2 - 496),
    {**fused(Q), **at("q_out", Q + 64 * 2)},                    # over queries, one head on
    {**fused(Q), **at("q_out", Q + 4 * 64 * 2)},                # over keys
    {**fused(Q), **at("q_out", Q + 5 * 64 * 2)},                # over a key and values
    {**fused(Q), **at("q_out", Q + (PITCH - 64) * 2)},          # over a value and the next token
    {**fused(Q), **at("q_out", Q), **at("k", Q + 3 * 64 * 2)},  # in place, a key is the last query head
    {**fused(Q), **at("q_out", Q), **at("v", Q + (PITCH - 64) * 2)},
])
def test_append_refuses_queries_with_gaps_over_what_it_reads(kw):
    refused("nkv_paged_append", rotated(**kw), INV, b"overlap")


def attended(**kw):
    return attend_args(**{**dict(G=2, Q=4, lse=PTR + (9 << 24), length=PTR + (10 << 24)), **kw})


def attended_at(name, base, sb=4 * PITCH, st=PITCH, sh=64):
    kw = at(name, base, sb, st, sh)
    return {("o" + k[3:] if k.startswith("out_") else k): v for k, v in kw.items()}


@pytest.mark.parametrize("kw", [
    attended_at("out", PTR + 1024), attended_at("out", V - 512), attended_at("out", PTR + (3 << 24) - 496),
    attended_at("out", PTR + (9 << 24) - 496), attended_at("out", PTR + (10 << 24) - 496),
    {**attended_at("q", Q), **attended_at("out", Q + 128)}, {**attended_at("q", Q), **attended_at("out", Q - 128)},
    {**attended_at("q", Q), **attended_at("out", Q + PITCH * 2 - 128)},
    {**attended_at("q", Q), "lse": Q + PITCH * 2}, {**attended_at("q", Q), "lse": Q - 4},
])
def test_attend_refuses_outputs_with_gaps_over_what_it_reads(kw):
    refused("nkv_paged_attend", attended(**kw), INV, b"overlap", None, 0)


def test_attend_refuses_a_workspace_over_queries_or_outputs_with_gaps():
    c = cache(pages=1 << 10)
    c.v = PTR + (1 << 28)
    far = dict(cache=c, table=1 << 40, lse=(1 << 40) + (1 << 30), length=(1 << 40) + (1 << 31), n=65536,
               table_w=4096, table_sb=4096, B=1)
    a = attended(**far, **attended_at("q", 1 << 41), **attended_at("out", 1 << 42))
    need = _lib.lib().nkv_paged_attend_workspace_size(ctypes.byref(a))
    assert need > 0
    for base in (1 << 41, 1 << 42):
        for t in (0, 3):
            refused("nkv_paged_attend", a, INV, b"workspace overlaps", base + t * PITCH * 2 + 4 * 64 * 2 - 16, need)


CALLS = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # before the library: its symbols come first
sys.path.insert(0, ".")
import random
from nanokv_amd import _lib
from tests import test_paged_overlap_gaps as t
lib = _lib.lib()
shim.shim_device(0)

def taken(name, a, *more):
    rc = getattr(lib, name)(None, ctypes.byref(a), *more)
    return rc == 0, rc, lib.nkv_last_error()

# a fused projection, rotated in place and into a buffer like it, and outputs in the gaps
Q, P = t.Q, t.PITCH
keys_first = {**t.at("k", Q), **t.at("q", Q + 2 * 64 * 2), **t.at("v", Q + 6 * 64 * 2)}
for kw in ({**t.fused(Q), **t.at("q_out", Q)}, {**t.fused(Q), **t.at("q_out", t.OUT)},
           {**keys_first, **t.at("q_out", Q + 2 * 64 * 2)},
           {**t.at("q", Q), **t.at("q_out", Q + 4 * 64 * 2)}):
    ok = taken("nkv_paged_append", t.rotated(**kw))
    assert ok[0], (kw, ok)
for kw in ({**t.attended_at("q", Q), **t.attended_at("out", Q + 4 * 64 * 2)},
           {**t.attended_at("q", Q), **t.attended_at("out", Q - 4 * 64 * 2)},
           {**t.attended_at("q", Q), **t.attended_at("out", Q)},
           {**t.attended_at("q", Q), "lse": Q + 4 * 64 * 2, "B": 1, "Q": 1}):
    ok = taken("nkv_paged_attend", t.attended(**kw), None, 0)
    assert ok[0], (kw, ok)

# rows drawn inside one buffer against a search over all of them
rng = random.Random(5)
counts = [0, 0]
for _ in range(4000):
    a, overlap = t.drawn(rng)
    ok = taken("nkv_paged_append", a)
    assert ok[0] == (not overlap), (ok, overlap, [(f, getattr(a, f)) for f, _ in a._fields_ if f != "cache"])
    assert ok[0] or b"overlap" in ok[2] or b"over q" in ok[2], ok
    counts[overlap] += 1
assert min(counts) > 400, counts
print("ok")
"""


def drawn(rng):
    """An append whose rotated queries, or one of its sources, have gaps, all in one
    buffer; and whether a plain search finds the outputs over a source."""
    B, T, H, Hq, D = rng.choice([1, 2, 3]), rng.choice([1, 2, 3]), rng.choice([1, 2]), rng.choice([1, 2, 3]), 16
    wide, slots = D + rng.choice([0, 0, 8, 24]), rng.randint(3, 9)

    def strides(heads):
        # token after token, or head after head
        n = max(heads, slots)
        st, sh = (n * wide, wide) if order else (wide, T * wide)
        return T * n * wide + gap, st, sh

    order, gap = rng.random() < 0.6, 8 * rng.randint(0, 3)
    base = 1 << 40
    place = lambda: base + 16 * rng.randint(0, 2 * T * slots * wide // 8)
    rows = {}
    for name, heads in (("k", H), ("v", H), ("q", Hq), ("q_out", Hq)):
        rows[name] = (place(), *strides(max(H, Hq)), heads)
    if rng.random() < 0.3:
        rows["q_out"] = (rows["q"][0], *rows["q"][1:])
    if rng.random() < 0.4:
        rows[rng.choice("kv")] = ((1 << 41) + 16 * rng.randint(0, 64), T * H * D, H * D, D, H)
    if rng.random() < 0.3:                    # packed outputs
        rows["q_out"] = (place(), T * Hq * D, Hq * D, D, Hq)
    c = cache(H=H, D=D)
    a = rotated(cache=c, B=B, T=T, Hq=Hq, rot=D, table_w=4)
    for name, (p, sb, st, sh, _) in rows.items():
        set_fields(a, at(name, p, sb, st, sh))

    def starts(name):
        p, sb, st, sh, heads = rows[name]
        return [p + 2 * (b * sb + t * st + h * sh)
                for b, t, h in itertools.product(range(B), range(T), range(heads))]

    out = starts("q_out")
    same = rows["q_out"][:4] == rows["q"][:4]
    overlap = any(abs(x - y) < 2 * D for name in "kvq" if name != "q" or not same
                  for x in out for y in starts(name))
    # (an output at the queries' place with other strides is refused for that)
    overlap = overlap or rows["q_out"][0] == rows["q"][0] and not same
    return a, overlap


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_rows_between_others_are_taken_and_rows_over_others_are_not(tmp_path):
    """Over stand-ins for the HIP calls."""
    src, so = tmp_path / "shim.c", tmp_path / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(src), "-o", str(so)], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(so)], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
