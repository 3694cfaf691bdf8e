"""Refusals of the paged cache's entry points, without a GPU: the C ABI checks every
shape on the host and launches nothing, and the torch wrappers refuse what they cannot
pass on; and the plain forms' own rules."""
import ctypes
import shutil
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import _paged_ref as ref
from nanokv_amd import _lib, ops
from tests.test_device_attributes import SHIM

PTR = 1 << 20      # stands for device memory; never read
INV, UNS = _lib.NKV_ERR_INVALID, _lib.NKV_ERR_UNSUPPORTED


def cache(pages=8, H=2, page=16, D=64, dtype=0, at=PTR):
    return _lib.NkvPagedCache(at, at + (1 << 24), pages, H, page, D, dtype)


def set_fields(a, kw):
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def append_args(**kw):
    a = _lib.NkvPagedAppendArgs()
    a.cache = kw.pop("cache", cache())
    a.table, a.table_sb, a.table_w = PTR + (3 << 24), 4, 4
    a.k, a.v = PTR + (4 << 24), PTR + (5 << 24)
    a.B, a.T, a.start, a.dtype = 2, 4, 0, a.cache.dtype
    D = a.cache.D
    a.k_sb = a.v_sb = 4 * a.cache.H * D
    a.k_st = a.v_st = a.cache.H * D
    a.k_sh = a.v_sh = D
    return set_fields(a, kw)


def rotated(**kw):
    a = append_args(cache=kw.pop("cache", cache()))
    a.q, a.q_out, a.freqs, a.rot = PTR + (6 << 24), PTR + (7 << 24), PTR + (8 << 24), 64
    a.Hq = 4
    a.q_sb, a.q_st, a.q_sh = a.o_sb, a.o_st, a.o_sh = 16 * 64, 4 * 64, 64
    return set_fields(a, kw)


def attend_args(**kw):
    a = _lib.NkvPagedAttendArgs()
    a.cache = kw.pop("cache", cache())
    a.table, a.table_sb, a.table_w, a.B = PTR + (3 << 24), 4, 4, 2
    a.G, a.Q, a.n, a.softmax_scale = 1, 1, 64, 1.0
    a.q, a.out = PTR + (4 << 24), PTR + (5 << 24)
    set_fields(a, kw)
    heads, D = a.cache.H * a.G, a.cache.D
    given = {k: kw[k] for k in ("o_sb", "o_st", "o_sh") if k in kw}
    return set_fields(a, {**dict(o_sb=a.Q * heads * D, o_st=heads * D, o_sh=D), **given})


def commit_args(caches=None, **kw):
    a = _lib.NkvPagedCommitArgs()
    caches = caches or [cache()]
    a.cache = caches[0]
    a._held = (ctypes.c_void_p * (2 * len(caches)))(*(p for c in caches for p in (c.k, c.v)))
    a.pools, a.n_caches = a._held, len(caches)
    a.table, a.table_sb, a.table_w = PTR + (3 << 24), 4, 4
    a.rows, a.rows_sb, a.out_length = PTR + (4 << 24), 3, PTR + (5 << 24)
    a.B, a.M, a.start = 2, 3, 0
    return set_fields(a, kw)


def refused(name, args, code, text, *more):
    lib = _lib.lib()
    assert getattr(lib, name)(None, ctypes.byref(args), *more) == code, lib.nkv_last_error()
    assert text in lib.nkv_last_error(), lib.nkv_last_error()


BAD_CACHES = [
    (dict(D=60), UNS, b"multiple of 8"), (dict(D=136), UNS, b"multiple of 8"), (dict(D=0), INV, b"D >= 1"),
    (dict(H=0), INV, b"H >= 1"), (dict(dtype=2), INV, b"bf16 or fp16"), (dict(page=8), UNS, b"power of two"),
    (dict(page=24), UNS, b"power of two"), (dict(page=2048), UNS, b"power of two"), (dict(pages=0), INV, b"pages"),
    (dict(pages=1 << 31), INV, b"pages"), (dict(at=PTR + 8), INV, b"aligned"),
    (dict(H=65536, D=8), UNS, b"too many heads"), (dict(H=8192, page=1024, D=128), UNS, b"too many heads"),
]


@pytest.mark.parametrize("kw,code,text", BAD_CACHES)
def test_bad_caches(kw, code, text):
    refused("nkv_paged_append", append_args(cache=cache(**kw)), code, text)
    refused("nkv_paged_attend", attend_args(cache=cache(**kw)), code, text, None, 0)
    refused("nkv_paged_commit", commit_args([cache(**kw)]), code, text)
    none = cache()
    none.v = None
    refused("nkv_paged_append", append_args(cache=none), INV, b"required")


BAD_TABLES = [
    (dict(B=-1), INV, b"B >= 0"), (dict(B=65536), UNS, b"too many sequences"), (dict(table_w=-1), INV, b"table_w"),
    (dict(table_w=1 << 31), INV, b"table_w"), (dict(table_sb=-4), INV, b"table_sb"), (dict(table=None), INV, b"table"),
]


@pytest.mark.parametrize("kw,code,text", BAD_TABLES)
def test_bad_tables(kw, code, text):
    refused("nkv_paged_append", append_args(**kw), code, text)
    refused("nkv_paged_attend", attend_args(**kw), code, text, None, 0)
    refused("nkv_paged_commit", commit_args(**kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=-1), INV, b"T must"), (dict(T=1 << 31), INV, b"T must"), (dict(dtype=1), INV, b"cache's type"),
    (dict(start=-1), INV, b"start"), (dict(start=61), INV, b"start"), (dict(start=65, counts=PTR + (9 << 24)), INV, b"start"),
    (dict(k=None), INV, b"required"), (dict(v=PTR + (5 << 24) + 8), INV, b"aligned"), (dict(k_sh=12), INV, b"strides"),
    (dict(k_sb=-64), INV, b"negative"), (dict(k=PTR + 1024), INV, b"overlap"), (dict(table=PTR + 1024), INV, b"overlap"),
    (dict(counts=PTR + (1 << 24)), INV, b"overlap"), (dict(q_out=PTR), INV, b"needs q"),
    (dict(positions=PTR), INV, b"need freqs"), (dict(T=1 << 26, start_dev=PTR + (9 << 24)), UNS, b"too many rows"),
])
def test_append_refusals(kw, code, text):
    refused("nkv_paged_append", append_args(**kw), code, text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(q_out=None), INV, b"q_out"), (dict(Hq=0), INV, b"Hq"), (dict(freqs=None), INV, b"without freqs"),
    (dict(rot=0), INV, b"rot"), (dict(rot=72), INV, b"rot"), (dict(rot=24), UNS, b"multiple of 16"),
    (dict(rot=12, interleaved=1), UNS, b"of 8"), (dict(positions=PTR, pos_sb=-1), INV, b"pos_sb"),
    (dict(o_st=64), INV, b"rows overlap"), (dict(o_sh=0), INV, b"rows overlap"),
    (dict(q_out=PTR + 4096), INV, b"overlap"), (dict(q_out=PTR + (6 << 24) + 1024), INV, b"overlap"),
    (dict(q_out=PTR + (4 << 24)), INV, b"overlap"), (dict(q_out=PTR + (8 << 24)), INV, b"overlap"),
    (dict(q_out=PTR + (6 << 24), dtype=2), INV, b"over q"),
    (dict(q_out=PTR + (6 << 24), o_sb=64, o_st=128, o_sh=1024), INV, b"over q"),
])
def test_append_refusals_of_queries(kw, code, text):
    refused("nkv_paged_append", rotated(**kw), code, text)


def test_append_refuses_queries_over_rows_and_positions():
    rows, at = PTR + (4 << 24), PTR + (6 << 24)
    refused("nkv_paged_append", rotated(q=rows, q_out=rows), INV, b"overlaps the rows")
    refused("nkv_paged_append", rotated(v=at, q_out=at), INV, b"overlaps the rows")
    refused("nkv_paged_append", rotated(positions=PTR + (7 << 24) + 4, pos_sb=4), INV, b"positions")
    refused("nkv_paged_append", rotated(positions=PTR + 4, pos_sb=4), INV, b"positions")


def test_append_refuses_pools_that_overlap():
    c = cache()
    c.v = c.k + 1024
    refused("nkv_paged_append", append_args(cache=c), INV, b"overlap each other")


ATTEND = [
    (dict(G=0), INV, b"G must"), (dict(Q=-1), INV, b"G must"), (dict(Q=1 << 30), UNS, b"too many"),
    (dict(n=-1), INV, b"n must"), (dict(n=65), INV, b"n must"), (dict(n=(1 << 30) + 1, table_w=1 << 30), INV, b"n must"),
    (dict(softmax_scale=0.0), INV, b"softmax_scale"), (dict(softmax_scale=float("nan")), INV, b"softmax_scale"),
    (dict(softmax_scale=float("inf")), INV, b"softmax_scale"), (dict(causal=1, parents=PTR), INV, b"exclude"),
    (dict(parents=PTR, Q=257), UNS, b"256"), (dict(parents=PTR, parents_sb=-1), INV, b"parents_sb"),
    (dict(q=None), INV, b"required"), (dict(out=None), INV, b"required"), (dict(q=PTR + 2), INV, b"aligned"),
    (dict(q_sh=12), INV, b"strides"), (dict(o_st=7), INV, b"strides"), (dict(o_sh=56), INV, b"rows overlap"),
    (dict(out=PTR), INV, b"overlaps"), (dict(lse=PTR + (1 << 24)), INV, b"overlaps"),
    (dict(length=PTR + (5 << 24)), INV, b"overlaps"), (dict(parents=PTR + (5 << 24)), INV, b"overlaps"),
    (dict(table=PTR + (5 << 24)), INV, b"overlaps"), (dict(lse=PTR + (5 << 24) + 16), INV, b"overlaps"),
    (dict(out=PTR + (4 << 24)), INV, b"strides"),
]


@pytest.mark.parametrize("kw,code,text", ATTEND)
def test_attend_refusals(kw, code, text):
    refused("nkv_paged_attend", attend_args(**kw), code, text, None, 0)
    lib = _lib.lib()
    assert lib.nkv_paged_attend_workspace_size(ctypes.byref(attend_args(**kw))) == 0
    assert text in lib.nkv_last_error()


def packed(**kw):
    a = attend_args(**kw)
    a.q_sb, a.q_st, a.q_sh = a.o_sb, a.o_st, a.o_sh
    return a


def test_attend_refuses_what_overlaps_queries_or_workspace():
    q, out = PTR + (4 << 24), PTR + (5 << 24)
    refused("nkv_paged_attend", packed(out=q + 128), INV, b"out overlaps q", None, 0)
    refused("nkv_paged_attend", packed(lse=q + 16), INV, b"lse overlaps q", None, 0)
    a = packed(n=65536, table_w=4096, table_sb=4096, B=1, lse=PTR + (6 << 24), length=PTR + (7 << 24))
    need = _lib.lib().nkv_paged_attend_workspace_size(ctypes.byref(a))
    for at in (q, out - 16, PTR + (6 << 24) - 16):
        refused("nkv_paged_attend", a, INV, b"workspace overlaps q, out or lse", at, need)
    for at in (PTR, PTR + (1 << 24), PTR + (3 << 24), PTR + (7 << 24) - 16):
        refused("nkv_paged_attend", a, INV, b"workspace overlaps the cache", at, need)
    a.q_st = -64
    refused("nkv_paged_attend", a, INV, b"negative", None, 0)
    refused("nkv_paged_attend", attend_args(B=65535, Q=1 << 28, n=64), UNS, b"too many", None, 0)


def test_workspace_sizes_and_alignment():
    lib = _lib.lib()
    a = attend_args(n=65536, table_w=4096, table_sb=4096, B=1)
    need = lib.nkv_paged_attend_workspace_size(ctypes.byref(a))
    # two heads' fp32 partial rows of 64 columns and eight bytes of statistics
    assert need > 0 and need % (2 * (64 * 4 + 8)) == 0
    refused("nkv_paged_attend", a, INV, b"aligned", PTR + 4, need)


@pytest.mark.parametrize("kw,code,text", [
    (dict(n_caches=0), INV, b"a cache"), (dict(M=-1), INV, b"M must"), (dict(M=257), UNS, b"256"),
    (dict(rows=None), INV, b"rows"), (dict(rows_sb=-1), INV, b"rows_sb"), (dict(start=-1), INV, b"start"),
    (dict(start=62), INV, b"start"), (dict(table=PTR), INV, b"overlap"), (dict(out_length=PTR + (4 << 24) + 4), INV, b"overlap"),
    (dict(out_length=PTR), INV, b"overlap"), (dict(counts=PTR + (5 << 24) + 4), INV, b"overlap"),
])
def test_commit_refusals(kw, code, text):
    refused("nkv_paged_commit", commit_args(**kw), code, text)


def test_commit_refuses_caches_that_overlap_or_are_too_many():
    other = PTR + (16 << 24)
    refused("nkv_paged_commit", commit_args([cache(), cache()]), INV, b"overlap")
    refused("nkv_paged_commit", commit_args([cache(), cache(at=other), cache(at=PTR + 512)]), INV, b"overlap")
    refused("nkv_paged_commit", commit_args([cache(), cache(at=other + 8)]), INV, b"aligned")
    many = [cache(at=other + (i << 26)) for i in range(65)]
    refused("nkv_paged_commit", commit_args(many), UNS, b"64 caches")
    refused("nkv_paged_commit", commit_args(pools=None), INV, b"a cache")


CALLS = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # before the library: its symbols come first
sys.path.insert(0, ".")
from nanokv_amd import _lib
from tests import test_paged as t
lib = _lib.lib()

def attend(B, H, n, Q, G, D=128, dtype=0, work=True, page=16, **kw):
    c = t.cache(pages=1, H=H, D=D, dtype=dtype, page=page)
    a = t.attend_args(cache=c, B=B, table_w=n // page + 1, n=n, Q=Q, G=G, **kw)
    a.q, a.out = 1 << 40, 1 << 41
    a.table = 1 << 42
    need = lib.nkv_paged_attend_workspace_size(ctypes.byref(a))
    return lib.nkv_paged_attend(None, ctypes.byref(a), (1 << 43) if work else None, need if work else 0)

# (call, launches: with a workspace one, or two with a merge of splits)
calls = [(lambda: attend(1, 8, 4096, 1, 4), (2,)), (lambda: attend(32, 8, 4096, 1, 4), (1, 2)),
         (lambda: attend(64, 8, 512, 1, 4), (1, 2)), (lambda: attend(32, 8, 4096, 1, 4, D=64), (1, 2)),
         (lambda: attend(1, 8, 4096, 20, 4, D=96), (1, 2)), (lambda: attend(16, 8, 8192, 10, 2, dtype=1), (1, 2)),
         (lambda: attend(1, 8, 4096, 1, 4, work=False), (1,)),
         (lambda: attend(1, 24, 12480, 1560, 1, work=False), (1,)),
         (lambda: attend(2, 4, 5000, 1023, 4, D=64, work=False), (1,)),
         (lambda: attend(2, 4, 5000, 1023, 4, D=80, work=False, dtype=1), (1,)),
         (lambda: attend(16, 8, 8192, 64, 4, work=False, parents=1 << 44), (1,)),
         (lambda: lib.nkv_paged_append(None, ctypes.byref(t.rotated())), (1,)),
         (lambda: lib.nkv_paged_append(None, ctypes.byref(t.append_args(T=0))), (0,)),
         (lambda: lib.nkv_paged_commit(None, ctypes.byref(t.commit_args())), (1,)),
         (lambda: lib.nkv_paged_commit(None, ctypes.byref(t.commit_args(M=0))), (1,)),
         (lambda: lib.nkv_paged_commit(None, ctypes.byref(t.commit_args(M=0, out_length=None))), (0,))]
for i, (call, n) in enumerate(calls):
    for dev in (0, 1, 0):
        shim.shim_device(dev)
        rc = call()
        assert rc == 0, (i, dev, rc, lib.nkv_last_error())
        assert shim.shim_launches() in n, (i, dev, shim.shim_launches())
        assert shim.shim_missing() == 0, (i, dev, shim.shim_missing())
print("ok")
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_launches_with_and_without_workspace_and_lds_on_every_device(tmp_path):
    """Over stand-ins for the HIP calls (nothing is launched): without a workspace one
    launch instead of splits and their merge, and every launch above 64 KB of dynamic
    LDS has its attribute on the device in use."""
    src, so = tmp_path / "shim.c", tmp_path / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(src), "-o", str(so)], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(so)], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def test_ctypes_structs_match_the_header_layout(tmp_path):
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    structs = {"nkv_paged_cache": _lib.NkvPagedCache, "nkv_paged_append_args": _lib.NkvPagedAppendArgs,
               "nkv_paged_attend_args": _lib.NkvPagedAttendArgs, "nkv_paged_commit_args": _lib.NkvPagedCommitArgs}
    header = Path(__file__).resolve().parent.parent / "include" / "nanokv.h"
    lines, want = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"',
                   "int main(void){"], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    (tmp_path / "layout.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run([gcc, "-std=c99", str(tmp_path / "layout.c"), "-o", str(tmp_path / "layout")],
                   check=True)
    got = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True)
    assert [int(x) for x in got.stdout.split()] == want


def test_wrappers_refuse_what_is_not_on_a_gpu_and_bad_caches():
    c = ops.PagedCache.empty(4, 16, 2, 80, torch.device("cpu"))
    assert c.page == 16 and c.k.shape == (4, 2, 16, 80) and c.k.dtype == torch.bfloat16
    table = torch.zeros((1, 4), dtype=torch.int32)
    x = torch.zeros((1, 3, 2, 80), dtype=torch.bfloat16)
    for call in (lambda: ops.paged_append(c, table, x, x, 0), lambda: ops.paged_attend(x, c, table, 3),
                 lambda: ops.paged_commit(c, table, 0, table)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    cpu = torch.device("cpu")
    for bad in (dict(page=8), dict(page=48), dict(head_dim=12), dict(head_dim=136), dict(pages=0), dict(H=0)):
        with pytest.raises(ValueError):
            ops.PagedCache.empty(**{**dict(pages=1, page=16, H=1, head_dim=64, device=cpu), **bad})
    with pytest.raises(TypeError):
        ops.PagedCache.empty(1, 16, 1, 64, cpu, torch.float32)
    with pytest.raises(TypeError):
        ops.PagedCache(c.k, c.v.half()).struct()
    with pytest.raises(ValueError):
        ops.PagedCache(c.k, c.v[:2]).struct()
    with pytest.raises(ValueError):
        ops.PagedCache(c.k[..., :64], c.v[..., :64]).struct()


def test_wrappers_refuse_arguments_that_do_not_fit(monkeypatch):
    """Before anything is launched (device checks aside, which need a GPU)."""
    def launch(*_):
        raise AssertionError("launched")
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(ops, "_device_call", launch)
    i32, bf = torch.int32, torch.bfloat16
    c = ops.PagedCache.empty(8, 16, 2, 64, torch.device("cpu"))
    table, x, q = torch.zeros((2, 4), dtype=i32), torch.zeros((2, 3, 2, 64), dtype=bf), torch.zeros((2, 3, 4, 64), dtype=bf)
    freqs, ints = torch.zeros(32), torch.zeros(2, dtype=i32)
    append = lambda **kw: ops.paged_append(**{**dict(cache=c, table=table, k=x, v=x, start=0), **kw})
    for kw in (dict(table=table[0]), dict(table=table.long()), dict(table=table.t()), dict(k=x[:1], v=x[:1]),
               dict(k=x[:, :, :1], v=x[:, :, :1]), dict(v=x[:, :2]), dict(k=x[..., :56], v=x[..., :56]),
               dict(start=ints[:1]), dict(start=ints.long()), dict(counts=ints[:1]), dict(q=q), dict(q_out=q),
               dict(positions=ints), dict(q=q[:, :2], freqs=freqs), dict(q=q, freqs=freqs[:12]),
               dict(q=q, freqs=torch.zeros(33)), dict(q=q, freqs=torch.zeros(2), interleaved=True),
               dict(q=q, freqs=freqs, q_out=q.half()), dict(q=q, freqs=freqs, q_out=q[:, :2]),
               dict(q=q, freqs=freqs, positions=table), dict(q=q, freqs=freqs, positions=torch.zeros(2, 3)),
               dict(q=q, freqs=freqs, positions=torch.zeros((3, 3), dtype=i32)), dict(q=q[:, :, :0], freqs=freqs),
               dict(k=x[..., 1:], v=x[..., 1:])):
        with pytest.raises(ValueError):
            append(**kw)
    for kw in (dict(k=x.half(), v=x.half()), dict(v=x.float()), dict(freqs=freqs.double()), dict(q=q.float(), freqs=freqs)):
        with pytest.raises(TypeError):
            append(**kw)
    attend = lambda **kw: ops.paged_attend(**{**dict(q=q, cache=c, table=table, length=5), **kw})
    for kw in (dict(q=q[:1]), dict(q=q[:, :, :3]), dict(q=q[:, :, :0]), dict(q=q[..., :56]), dict(length=65),
               dict(length=-1), dict(length=6, max_length=5), dict(length=ints, max_length=65), dict(length=ints[:1]),
               dict(causal=True, parents=torch.zeros(3, dtype=i32)), dict(parents=torch.zeros((2, 4), dtype=i32)),
               dict(parents=torch.zeros((3, 3), dtype=i32)), dict(parents=torch.zeros((2, 3))), dict(counts=ints[:1]),
               dict(out=q[:, :2]), dict(out=q.half())):
        with pytest.raises(ValueError):
            attend(**kw)
    with pytest.raises(TypeError):
        attend(q=q.half())
    commit = lambda **kw: ops.paged_commit(**{**dict(caches=c, table=table, start=0, rows=torch.zeros((2, 3), dtype=i32)), **kw})
    wide = ops.PagedCache.empty(9, 16, 2, 64, torch.device("cpu"))
    for kw in (dict(caches=[]), dict(caches=[c, wide]), dict(rows=ints), dict(rows=torch.zeros((1, 3), dtype=i32)),
               dict(rows=torch.zeros((2, 257), dtype=i32)), dict(rows=torch.zeros((2, 3))), dict(counts=ints[:1]),
               dict(start=ints[:1])):
        with pytest.raises(ValueError):
            commit(**kw)


def test_the_plain_forms_rules():
    see = ref.visible(4, 6, 3, causal=True)
    assert see.sum(1).tolist() == [4, 5, 6, 0]
    see = ref.visible(4, 3, 4, parents=[-1, 0, 0, 2])
    assert see.astype(int).tolist() == [[0, 0, 0], [1, 0, 0], [0, 1, 0], [0, 1, 1]]
    see = ref.visible(3, 5, 3, parents=[5, 1, 0])
    assert see.astype(int).tolist() == [[1, 1, 1, 0, 0], [1, 1, 0, 1, 0], [1, 1, 1, 0, 1]]
    x = np.arange(8.0).reshape(1, 1, 8)
    y, _ = ref.rotate(x, [np.pi / 2], np.ones(2), False)
    assert np.allclose(y[0, 0], [-2, -3, 0, 1, 4, 5, 6, 7])
    y, _ = ref.rotate(x, [np.pi / 2], np.ones(2), True)
    assert np.allclose(y[0, 0], [-1, 0, -3, 2, 4, 5, 6, 7])
    pool = np.arange(32.0).reshape(2, 1, 16, 1)
    new = ref.commit(pool, [[1, 0]], [14], [[2, 1, 0]], [3])
    assert new[1, 0, 14, 0] == 0 and new[1, 0, 15, 0] == 31 and new[0, 0, 0, 0] == 30
