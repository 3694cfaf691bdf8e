"""Calls of the 8-bit cache at the edges of what is allowed, without a GPU: the
library runs over stand-ins for the HIP calls, which count its launches."""
import ctypes
import shutil
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from nanokv_amd import _lib, build, ops
from tests import test_cache8 as t
from tests.test_device_attributes import SHIM

ROOT = Path(__file__).resolve().parent.parent

HEAD = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # before the library: its symbols come first
sys.path.insert(0, ".")
from nanokv_amd import _lib
from tests import test_cache8 as t
lib = _lib.lib()

def launches(name, args, *more):
    shim.shim_device(0)
    rc = getattr(lib, name)(None, ctypes.byref(args), *more)
    assert rc == 0, (rc, lib.nkv_last_error())
    return shim.shim_launches()
"""


def over_stand_ins(tmp_path, code):
    if shutil.which("gcc") is None:
        pytest.skip("needs a C compiler")
    src, so = tmp_path / "shim.c", tmp_path / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(src), "-o", str(so)], check=True)
    run = subprocess.run([sys.executable, "-c", HEAD + code + "\nprint('ok')", str(so)],
                         capture_output=True, text=True, cwd=ROOT, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr


def test_no_query_rows_launch_no_attention(tmp_path):
    """The weight of no queries: nothing in place, one copy into another array."""
    over_stand_ins(tmp_path, r"""
for causal in (0, 1):
    a = t.attend_args(_lib.NkvCache8MassArgs, Q=0, q=None, lse=None, causal=causal)
    assert lib.nkv_cache8_mass_workspace_size(ctypes.byref(a)) == 0
    a.out = a.mass
    assert launches("nkv_cache8_mass", a, None, 0) == 0
    a.out = t.PTR + (12 << 24)
    assert launches("nkv_cache8_mass", a, None, 0) == 1
    assert launches("nkv_cache8_attend", t.attend_args(Q=0, q=None, out=None, causal=causal),
                    None, 0) == 0
""")


def test_the_attention_is_compiled_with_nans():
    """What a NaN query does to its own row is documented, so no flag may let the
    compiler take NaN for impossible there."""
    assert not [f for f in build.SOURCES["nkv_cache8_attend.hip"] if "nan" in f or "fast" in f]


def test_the_wrappers_refuse_counts_of_another_kind():
    ints = torch.zeros(2, dtype=torch.int32)
    for bad in (ints.long(), ints[:1], torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="counts"):
            ops._cache8_ints(bad, 2, "counts")


@pytest.mark.parametrize("what", ["k", "v", "k_scale", "v_scale", "length", "counts", "lse"])
def test_attend_refuses_outputs_over_what_it_reads(what):
    """Workgroups would read what others have written."""
    base = t.PTR + (16 << 24)
    a = t.attend_args(Q=3, length=base, counts=base + 4096, lse=base + 8192)
    lib = _lib.lib()
    lib.nkv_cache8_attend_workspace_size(ctypes.byref(a))
    assert lib.nkv_last_error() == b""
    at = getattr(a.cache, what) if hasattr(a.cache, what) else getattr(a, what)
    a.out = at
    t.refused("nkv_cache8_attend", a, _lib.NKV_ERR_INVALID, b"overlap", None, 0)
    a.o_st *= 2                               # gaps, which may hold anything
    a.o_sb *= 2
    lib.nkv_cache8_attend_workspace_size(ctypes.byref(a))
    assert lib.nkv_last_error() == b""
    if what != "lse":
        a = t.attend_args(Q=3, length=base, counts=base + 4096, lse=at)
        t.refused("nkv_cache8_attend", a, _lib.NKV_ERR_INVALID, b"overlap", None, 0)


@pytest.mark.parametrize("what", ["k", "k_scale", "length", "counts", "lse"])
def test_mass_refuses_outputs_over_what_it_reads(what):
    base = t.PTR + (16 << 24)
    a = t.attend_args(_lib.NkvCache8MassArgs, Q=3, length=base, counts=base + 4096, lse=base + 8192)
    lib = _lib.lib()
    lib.nkv_cache8_mass_workspace_size(ctypes.byref(a))
    assert lib.nkv_last_error() == b""
    a.out = getattr(a.cache, what) if hasattr(a.cache, what) else getattr(a, what)
    t.refused("nkv_cache8_mass", a, _lib.NKV_ERR_INVALID, b"overlap", None, 0)
    a.mass = a.out                            # in place no less
    t.refused("nkv_cache8_mass", a, _lib.NKV_ERR_INVALID, b"overlap", None, 0)


@pytest.mark.parametrize("name", ["start_dev", "counts"])
def test_write_refuses_a_cache_over_its_starts_or_counts(name):
    c = t.cache()
    for at in (c.k + 64, c.v, c.k_scale + 4, c.v_scale):
        t.refused("nkv_cache8_write", t.write_args(**{name: at}), _lib.NKV_ERR_INVALID, b"overlaps")
