"""Refusals of the 8-bit cache's entry points, without a GPU: the C ABI checks
every shape on the host and launches nothing, and the torch wrappers refuse
what cannot be on a GPU."""
import ctypes
import shutil
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from tests import _cache8_ref as ref
from nanokv_amd import _lib, ops
from tests.test_device_attributes import SHIM

PTR = 1 << 20      # stands for device memory; never read


def cache(B=2, H=2, cap=128, D=64, fmt=0, at=PTR):
    return _lib.NkvCache8(at, at + (1 << 24), at + (2 << 24), at + (3 << 24), cap, B, H, D, fmt)


def write_args(**kw):
    a = _lib.NkvCache8WriteArgs()
    a.cache = kw.pop("cache", cache())
    a.k = a.v = PTR
    a.k_sb = a.k_st = a.k_sh = a.v_sb = a.v_st = a.v_sh = 64
    a.T = 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attend_args(cls=_lib.NkvCache8AttendArgs, **kw):
    a = cls()
    a.cache = kw.pop("cache", cache())
    a.G, a.Q, a.n, a.q, a.out, a.softmax_scale = 1, 1, 128, PTR, PTR + (8 << 24), 1.0
    if cls is _lib.NkvCache8MassArgs:
        a.lse, a.mass = PTR, PTR + (8 << 24)
    for k, v in kw.items():
        setattr(a, k, v)
    if cls is _lib.NkvCache8AttendArgs:        # contiguous, where not given
        c, heads = a.cache, a.cache.H * a.G
        given = {k: kw[k] for k in ("o_sb", "o_st", "o_sh") if k in kw}
        for k, v in {**dict(o_sb=a.Q * heads * c.D, o_st=heads * c.D, o_sh=c.D), **given}.items():
            setattr(a, k, v)
    return a


def evict_args(**kw):
    a = _lib.NkvCache8EvictArgs()
    a.cache, a.out = kw.pop("cache", cache()), kw.pop("out", cache(at=PTR + (4 << 24)))
    a.mass, a.out_mass, a.rows = PTR + (8 << 24), PTR + (9 << 24), PTR + (10 << 24)
    a.out_length, a.n, a.keep = PTR - 1024, 128, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(name, args, code, text, *more):
    lib = _lib.lib()
    assert getattr(lib, name)(None, ctypes.byref(args), *more) == code
    assert text in lib.nkv_last_error(), lib.nkv_last_error()


BAD_CACHES = [
    (dict(D=60), _lib.NKV_ERR_UNSUPPORTED, b"multiple of 8"),
    (dict(D=136), _lib.NKV_ERR_UNSUPPORTED, b"multiple of 8"),
    (dict(D=0), _lib.NKV_ERR_INVALID, b"D >= 1"),
    (dict(B=-1), _lib.NKV_ERR_INVALID, b"B >= 0"),
    (dict(H=0), _lib.NKV_ERR_INVALID, b"H >= 1"),
    (dict(fmt=2), _lib.NKV_ERR_INVALID, b"format"),
    (dict(cap=0), _lib.NKV_ERR_INVALID, b"multiple of 64"),
    (dict(cap=100), _lib.NKV_ERR_INVALID, b"multiple of 64"),
    (dict(cap=1 << 31), _lib.NKV_ERR_INVALID, b"at most 2^29"),
    (dict(at=PTR + 8), _lib.NKV_ERR_INVALID, b"aligned"),
    (dict(B=1 << 16, H=1 << 16), _lib.NKV_ERR_UNSUPPORTED, b"too many heads"),
]


@pytest.mark.parametrize("kw,code,text", BAD_CACHES)
def test_bad_caches(kw, code, text):
    c = cache(**kw)
    refused("nkv_cache8_write", write_args(cache=c), code, text)
    refused("nkv_cache8_attend", attend_args(cache=c), code, text, None, 0)
    refused("nkv_cache8_mass", attend_args(_lib.NkvCache8MassArgs, cache=c), code, text, None, 0)
    refused("nkv_cache8_evict", evict_args(cache=c), code, text, None, 0)


@pytest.mark.parametrize("kw,code,text", [
    (dict(T=-1), _lib.NKV_ERR_INVALID, b"T must"),
    (dict(dtype=3), _lib.NKV_ERR_INVALID, b"dtype"),
    (dict(start=125), _lib.NKV_ERR_INVALID, b"start + T"),
    (dict(start=-1), _lib.NKV_ERR_INVALID, b"start + T"),
    (dict(T=1 << 31), _lib.NKV_ERR_INVALID, b"T must"),
    (dict(k=None), _lib.NKV_ERR_INVALID, b"required"),
    (dict(v=PTR + 4), _lib.NKV_ERR_INVALID, b"aligned"),
    (dict(v_st=100), _lib.NKV_ERR_INVALID, b"strides"),
    (dict(cache=cache(H=70000, B=1)), _lib.NKV_ERR_UNSUPPORTED, b"too many heads"),
    (dict(cache=_lib.NkvCache8(PTR, PTR, PTR + (2 << 24), PTR + (3 << 24), 128, 2, 2, 64, 0)),
     _lib.NKV_ERR_INVALID, b"overlap each other"),
    (dict(cache=_lib.NkvCache8(PTR, PTR + (1 << 24), PTR + (2 << 24), PTR + (2 << 24) + 28, 128, 2, 2,
                               64, 0)), _lib.NKV_ERR_INVALID, b"overlap each other"),
])
def test_write_refusals(kw, code, text):
    refused("nkv_cache8_write", write_args(**kw), code, text)


QUERY = [
    (dict(G=0), _lib.NKV_ERR_INVALID, b"G must"),
    (dict(Q=-1), _lib.NKV_ERR_INVALID, b"Q not"),
    (dict(Q=1 << 31), _lib.NKV_ERR_UNSUPPORTED, b"too many query rows"),
    (dict(dtype=2), _lib.NKV_ERR_INVALID, b"bf16 or fp16"),
    (dict(n=129), _lib.NKV_ERR_INVALID, b"n must"),
    (dict(n=-1), _lib.NKV_ERR_INVALID, b"n must"),
    (dict(softmax_scale=0.0), _lib.NKV_ERR_INVALID, b"softmax_scale"),
    (dict(softmax_scale=-1.0), _lib.NKV_ERR_INVALID, b"softmax_scale"),
    (dict(softmax_scale=float("nan")), _lib.NKV_ERR_INVALID, b"softmax_scale"),
    (dict(softmax_scale=float("inf")), _lib.NKV_ERR_INVALID, b"softmax_scale"),
    (dict(q=None), _lib.NKV_ERR_INVALID, b"q is required"),
    (dict(q=PTR + 2), _lib.NKV_ERR_INVALID, b"aligned"),
    (dict(q_sh=12), _lib.NKV_ERR_INVALID, b"strides"),
]


@pytest.mark.parametrize("kw,code,text", QUERY + [
    (dict(out=None), _lib.NKV_ERR_INVALID, b"out is required"),
    (dict(out=PTR + 8), _lib.NKV_ERR_INVALID, b"aligned"),
    (dict(o_st=7), _lib.NKV_ERR_INVALID, b"strides"),
])
def test_attend_refusals(kw, code, text):
    refused("nkv_cache8_attend", attend_args(**kw), code, text, None, 0)
    lib = _lib.lib()
    assert lib.nkv_cache8_attend_workspace_size(ctypes.byref(attend_args(**kw))) == 0
    assert text in lib.nkv_last_error()


@pytest.mark.parametrize("strides,fits", [
    ((64 * 6, 128, 64), True),               # [B, Q, H, D]
    ((64 * 6, 64, 64 * 3), True),            # [B, H, Q, D]
    ((64, 128, 64 * 6), True),               # [H, Q, B, D]
    ((64 * 18, 64 * 6, 72), True),           # rows with columns between them
    ((64 * 6, 0, 64), False), ((0, 128, 64), False), ((64 * 6, 128, 0), False),
    ((64 * 6, 128, 56), False),              # a head's last columns are the next one's first
    ((64 * 5, 128, 64), False),              # the last token is the next item's first
    ((-64 * 6, 128, 64), False),
])
def test_attend_refuses_an_out_whose_rows_overlap(strides, fits):
    """Several workgroups would write one row."""
    kw = dict(zip(("o_sb", "o_st", "o_sh"), strides))
    a = attend_args(Q=3, **kw)
    lib = _lib.lib()
    lib.nkv_cache8_attend_workspace_size(ctypes.byref(a))
    assert (lib.nkv_last_error() == b"") == fits
    if not fits:
        refused("nkv_cache8_attend", a, _lib.NKV_ERR_INVALID, b"overlap", None, 0)
    one = attend_args(cache=cache(B=1, H=1), Q=1, o_sb=0, o_st=0, o_sh=0)   # strides of one row
    lib.nkv_cache8_attend_workspace_size(ctypes.byref(one))
    assert lib.nkv_last_error() == b""


def test_workspace_sizes_and_alignment():
    lib = _lib.lib()
    a = attend_args(cache=cache(B=1, H=1, cap=65536), n=65536)
    need = lib.nkv_cache8_attend_workspace_size(ctypes.byref(a))
    # 64 fp16-wide partial rows of 64 columns and 16 bytes of statistics each
    assert need > 0 and need % (64 * 2 + 16) == 0
    refused("nkv_cache8_attend", a, _lib.NKV_ERR_INVALID, b"aligned", PTR + 4, need)
    a.dtype = _lib.NKV_ROWS_FP16
    assert lib.nkv_cache8_attend_workspace_size(ctypes.byref(a)) == need // 144 * (64 * 4 + 16)
    m = attend_args(_lib.NkvCache8MassArgs, cache=cache(B=1, H=1, cap=1024), n=1000, Q=4096)
    need = lib.nkv_cache8_mass_workspace_size(ctypes.byref(m))
    assert need > 0 and need % (1024 * 4) == 0
    refused("nkv_cache8_mass", m, _lib.NKV_ERR_INVALID, b"aligned", PTR + 2, need)
    for n, parts in ((32768, 0), (32832, 5), (1 << 20, 64), (1 << 29, 64)):
        e = evict_args(cache=cache(B=1, H=1, cap=n, at=1 << 44), n=n, keep=64)
        e.cache.v, e.cache.k_scale, e.cache.v_scale, e.mass = 2 << 44, 3 << 44, 4 << 44, 5 << 44
        e.out, e.out_mass = cache(B=1, H=1, cap=64), PTR + (9 << 24)
        need = lib.nkv_cache8_evict_workspace_size(ctypes.byref(e))
        assert need == parts * (2 * 2048 * 4 + 16), lib.nkv_last_error()
        if need:
            refused("nkv_cache8_evict", e, _lib.NKV_ERR_INVALID, b"aligned", PTR + 8, need)
            refused("nkv_cache8_evict", e, _lib.NKV_ERR_WORKSPACE, b"smaller", PTR, need - 1)
            refused("nkv_cache8_evict", e, _lib.NKV_ERR_WORKSPACE, b"smaller", None, need)


CALLS = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # before the library: its symbols come first
sys.path.insert(0, ".")
from nanokv_amd import _lib
from tests import test_cache8 as t
lib = _lib.lib()

def attend(H, cap, Q, G, D=128, dtype=0, work=True):
    a = t.attend_args(cache=t.cache(B=1, H=H, cap=cap, D=D), n=cap, Q=Q, G=G, dtype=dtype)
    need = lib.nkv_cache8_attend_workspace_size(ctypes.byref(a))
    return lib.nkv_cache8_attend(None, ctypes.byref(a), t.PTR if work else None, need if work else 0)

def evict(cap, keep):
    big = 1 << 40
    a = t.evict_args(cache=t.cache(cap=cap, at=t.PTR), n=cap, keep=keep)
    a.out = _lib.NkvCache8(big, 2 * big, 3 * big, 4 * big, cap, 2, 2, 64, 0)
    a.cache.v, a.cache.k_scale, a.cache.v_scale = 5 * big, 6 * big, 7 * big
    a.mass, a.out_mass, a.rows, a.out_length = 8 * big, 9 * big, 10 * big, 11 * big
    need = lib.nkv_cache8_evict_workspace_size(ctypes.byref(a))
    return lib.nkv_cache8_evict(None, ctypes.byref(a), t.PTR, need)

# (call, launches, whether some take more than 64 KB)
calls = [(lambda: attend(8, 4096, 1, 4), 2, False), (lambda: attend(512, 1024, 1, 4), 1, True),
         (lambda: attend(8, 4096, 1, 4, work=False), 1, False),
         (lambda: attend(8, 4096, 40, 1), 2, False), (lambda: attend(64, 8192, 40, 1), 2, True),
         (lambda: attend(24, 12480, 1560, 1), 2, True), (lambda: attend(24, 12480, 1560, 1, work=False), 1, True),
         (lambda: evict(32768, 100), 2, True), (lambda: evict(40000 // 64 * 64, 100), 5, False)]
for i, (call, n, large) in enumerate(calls):
    for dev in (0, 1, 0):
        shim.shim_device(dev)
        rc = call()
        assert rc == 0, (i, dev, rc, lib.nkv_last_error())
        assert shim.shim_launches() == n and (shim.shim_large() > 0) == large, (i, dev, shim.shim_launches(), shim.shim_large())
        assert shim.shim_missing() == 0, (i, dev, shim.shim_missing())
print("ok")
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_launches_with_and_without_workspace_and_lds_on_every_device(tmp_path):
    """Over stand-ins for the HIP calls (nothing is launched): without a workspace
    one launch instead of splits and their merge, and every launch above 64 KB
    of dynamic LDS has its attribute on the device in use."""
    src, so = tmp_path / "shim.c", tmp_path / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(src), "-o", str(so)], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(so)], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


@pytest.mark.parametrize("kw,code,text", QUERY + [
    (dict(lse=None), _lib.NKV_ERR_INVALID, b"lse"),
    (dict(mass=None), _lib.NKV_ERR_INVALID, b"required"),
    (dict(out=PTR + (8 << 24) + 4), _lib.NKV_ERR_INVALID, b"overlap"),
    (dict(cache=cache(B=300, H=300)), _lib.NKV_ERR_UNSUPPORTED, b"too many heads"),
])
def test_mass_refusals(kw, code, text):
    refused("nkv_cache8_mass", attend_args(_lib.NkvCache8MassArgs, **kw), code, text, None, 0)


@pytest.mark.parametrize("kw,code,text", [
    (dict(out=cache(D=128, at=PTR + (4 << 24))), _lib.NKV_ERR_INVALID, b"same items"),
    (dict(out=cache(fmt=1, at=PTR + (4 << 24))), _lib.NKV_ERR_INVALID, b"same items"),
    (dict(out=cache()), _lib.NKV_ERR_INVALID, b"overlap"),
    (dict(out_mass=PTR + (8 << 24)), _lib.NKV_ERR_INVALID, b"overlap"),
    (dict(rows=PTR + (9 << 24)), _lib.NKV_ERR_INVALID, b"overlap"),
    (dict(length=PTR - 64, out_length=PTR - 60), _lib.NKV_ERR_INVALID, b"overlap"),
    (dict(out_length=PTR + (9 << 24)), _lib.NKV_ERR_INVALID, b"overlap"),
    (dict(keep=0), _lib.NKV_ERR_INVALID, b"keep"),
    (dict(keep=129), _lib.NKV_ERR_INVALID, b"keep"),
    (dict(sink=40, recent=30), _lib.NKV_ERR_INVALID, b"sink"),
    (dict(sink=-1), _lib.NKV_ERR_INVALID, b"sink"),
    (dict(recent=-1), _lib.NKV_ERR_INVALID, b"sink"),
    (dict(n=129), _lib.NKV_ERR_INVALID, b"n must"),
    (dict(mass=None), _lib.NKV_ERR_INVALID, b"required"),
    (dict(mass=PTR + (8 << 24) + 4), _lib.NKV_ERR_INVALID, b"mass must be 16"),
])
def test_evict_refusals(kw, code, text):
    refused("nkv_cache8_evict", evict_args(**kw), code, text, None, 0)


def test_ctypes_structs_match_the_header_layout(tmp_path):
    gcc = shutil.which("gcc") or shutil.which("cc")
    if gcc is None:
        pytest.skip("no C compiler")
    structs = {"nkv_cache8": _lib.NkvCache8, "nkv_cache8_write_args": _lib.NkvCache8WriteArgs,
               "nkv_cache8_attend_args": _lib.NkvCache8AttendArgs,
               "nkv_cache8_mass_args": _lib.NkvCache8MassArgs,
               "nkv_cache8_evict_args": _lib.NkvCache8EvictArgs}
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


def test_empty_calls_need_no_memory():
    lib = _lib.lib()
    none = _lib.NkvCache8(None, None, None, None, 64, 0, 1, 64, 0)
    assert lib.nkv_cache8_write(None, ctypes.byref(write_args(cache=none, k=None))) == 0
    assert lib.nkv_cache8_write(None, ctypes.byref(write_args(T=0, k=None))) == 0
    a = attend_args(cache=none, n=0, q=None, out=None)
    assert lib.nkv_cache8_attend(None, ctypes.byref(a), None, 0) == 0
    a = attend_args(Q=0, q=None, out=None)
    assert lib.nkv_cache8_attend(None, ctypes.byref(a), None, 0) == 0
    assert lib.nkv_last_error() == b""


def test_wrappers_refuse_what_is_not_on_a_gpu_and_bad_caches():
    c = ops.Cache8.empty(1, 2, 100, 80, torch.device("cpu"), "e4m3")
    assert c.cap == 128 and c.k.shape == (1, 2, 128, 128) and c.k_scale.shape == (1, 2, 2)
    x = torch.zeros((1, 3, 2, 80), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.cache8_write(c, x, x, 0)
    with pytest.raises(ValueError, match="GPU"):
        ops.cache8_attend(x, c, 3)
    with pytest.raises(ValueError, match="format"):
        ops.Cache8.empty(1, 1, 64, 64, torch.device("cpu"), "int4")
    for bad in (0, 12, 136):
        with pytest.raises(ValueError, match="head_dim"):
            ops.Cache8.empty(1, 1, 64, bad, torch.device("cpu"))
    with pytest.raises(ValueError, match="cap"):
        ops.Cache8.empty(1, 1, 0, 64, torch.device("cpu"))
    for broken, error in ((dict(v=c.v.view(torch.int8)), TypeError),
                          (dict(k=c.k[..., :64], v=c.v[..., :64]), ValueError),
                          (dict(k_scale=c.k_scale[:, :, :1]), ValueError),
                          (dict(k_scale=c.k_scale.double()), TypeError),
                          (dict(head_dim=64), ValueError)):
        fields = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale, head_dim=80)
        with pytest.raises(error):
            ops.Cache8(**{**fields, **broken}).struct()


def test_the_plain_form_of_the_codes():
    """The oracle's own rules: ties to even, the clamp, NaN, and the scale of a
    block that grows."""
    x = np.array([0.5, 1.5, -2.5, 200.0, np.nan, np.inf, -np.inf], np.float32)
    assert ref.to_codes(x, "int8").tolist() == [0, 2, -2, 127, 0, 127, -127]
    # 200 lies between 192 and 208, both 8 away: the even mantissa is 192's
    assert ref.values(ref.to_codes(x, "e4m3"), "e4m3").tolist() == \
        [0.5, 1.5, -2.5, 192.0, 0.0, 448.0, -448.0]
    c, s = np.zeros((1, 1, 64, 64), np.int8), np.ones((1, 1, 1), np.float32)
    one = np.zeros((1, 1, 1, 64), np.float32)
    one[..., 0] = 127.0
    c, s = ref.write(c, s, one, [0], [1], "int8")
    assert s.item() == 1.0 and c[0, 0, 0, 0] == 127
    c, s = ref.write(c, s, 2 * one, [1], [1], "int8")
    assert s.item() == 2.0 and c[0, 0, 0, 0] == 64 and c[0, 0, 1, 0] == 127
