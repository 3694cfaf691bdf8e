"""How many launches a call of the paged attention takes, on either side of each edge of
its rules for key splits: one, or two where the splits are merged.  Over stand-ins for the
HIP calls; no GPU is needed."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

from tests.test_device_attributes import SHIM

CALLS = r"""
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # before the library: its symbols come first
sys.path.insert(0, ".")
from nanokv_amd import _lib
from tests import test_paged as t
lib = _lib.lib()
FAR = 1 << 44

def call(B, H, n, Q=1, G=4, D=128, length=False, less=None, **kw):
    '''(launches, bytes of workspace wanted); less: those that it is given'''
    c = t.cache(pages=1, H=H, D=D, dtype=kw.pop("dtype", 0))
    a = t.attend_args(cache=c, B=B, table_w=n // 16 + 1, n=n, Q=Q, G=G, length=FAR if length else None, **kw)
    a.q, a.out, a.table = 1 << 40, 1 << 41, 1 << 42
    need = lib.nkv_paged_attend_workspace_size(ctypes.byref(a))
    given = need if less is None else less
    shim.shim_device(0)
    rc = lib.nkv_paged_attend(None, ctypes.byref(a), (1 << 43) if given else None, given)
    assert rc == 0, (rc, lib.nkv_last_error())
    assert shim.shim_missing() == 0
    return shim.shim_launches(), need

def splits(launches, need, B, H, rows, D=128, length=False):
    '''... and that is the partial rows of this many splits, and the shares of 2 to 64
    sequences with lengths of their own'''
    if launches == 1:
        assert need == 0, need
        return 1
    shares = 8 * B if length and 1 < B <= 64 else 0
    assert (need - shares) % (B * H * rows * (4 * D + 8)) == 0, (need, shares)
    return (need - shares) // (B * H * rows * (4 * D + 8))

def want(n_splits, B, H, n, Q=1, G=4, D=128, length=False, **kw):
    got = splits(*call(B, H, n, Q, G, D, length, **kw), B, H, Q * G, D, length)
    assert got == n_splits, (got, n_splits, B, H, n, Q, G, D, length, kw)

# few rows: none up to 32 tiles of 32 keys; then a workgroup a CU, of four tiles at least
want(1, 1, 8, 1024)
want(8, 1, 8, 1025)
want(32, 1, 8, 4096)
assert call(1, 8, 4096, 0) == (0, 0)
for B, n_splits in ((31, 2), (32, 1), (33, 1)):
    want(n_splits, B, 8, 4096)
    want(n_splits, B, 8, 4096, D=64)
    want(n_splits, B, 4, 4096, 10, 2, dtype=1)
want(1, 64, 8, 512)
# two workgroups a CU in long calls of unlike lengths, shared out by length up to 64
# sequences and fewer than 512 workgroups
want(2, 32, 8, 4096, length=True)
want(1, 32, 8, 4064, length=True)
want(2, 32, 8, 16384, length=True)
want(2, 63, 8, 131072, length=True)
want(1, 64, 8, 131072, length=True)
want(1, 32, 16, 131072, length=True)
want(2, 64, 4, 131072, length=True)
want(2, 65, 4, 131072, length=True)
want(1, 32, 8, 16384)
# two groups of 16 rows to a wave: one workgroup a CU at most
want(10, 1, 8, 4096, 20, 4, D=96)
want(2, 8, 8, 4096, 16, 4)
want(1, 9, 8, 4096, 16, 4)
# many rows: by the cost of rounds, with 256 keys a split at least
want(3, 1, 24, 12480, 1560, 1)
want(1, 1, 24, 255, 1560, 1)
want(1, 16, 8, 131072, 128, 4, length=True)
want(1, 2, 128, 8192, 128, 2)

# a workspace that is too small takes fewer splits, to one
launches, need = call(4, 8, 4096, length=True)
each = 4 * 8 * 4 * (4 * 128 + 8)
assert launches == 2 and need == 8 * each + 32, need
for less, n in ((need - 1, 2), (2 * each + 32, 2), (2 * each + 31, 1), (each + 32, 1), (31, 1), (1, 1), (0, 1)):
    assert call(4, 8, 4096, length=True, less=less)[0] == n, (less, n)
print("ok")
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_launches_at_the_edges_of_the_rules(tmp_path):
    src, so = tmp_path / "shim.c", tmp_path / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", str(src), "-o", str(so)], check=True)
    run = subprocess.run([sys.executable, "-c", CALLS, str(so)], capture_output=True, text=True,
                         cwd=Path(__file__).resolve().parent.parent, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "ok", run.stdout + run.stderr
