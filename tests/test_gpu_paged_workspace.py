"""The paged attention's workspace: a call writes no byte outside what it was given, and
reads none of it that it has not written, whatever was there."""
import numpy as np
import pytest
import torch

from nanokv_amd import _lib, ops
from tests.test_gpu_paged import check_large, make_pool, queries, random_tree

pytestmark = pytest.mark.gpu

GUARD = 4096


@pytest.fixture
def need(monkeypatch):
    """What the size query wanted for the last call."""
    wanted = []
    lib = _lib.lib()

    class Asked:
        def __getattr__(self, name):
            fn = getattr(lib, name)
            if name != "nkv_paged_attend_workspace_size":
                return fn

            def ask(args):
                wanted.append(fn(args))
                return wanted[-1]
            return ask
    monkeypatch.setattr(ops, "lib", lambda: Asked())
    return wanted


def guarded(dev, size):
    """A workspace of that many bytes between guards, all of it 0xff: NaN as fp32."""
    whole = torch.full((GUARD + (size + 15) // 16 * 16 + GUARD,), 0xff, dtype=torch.uint8, device=dev)
    assert whole.data_ptr() % 16 == 0
    return whole, whole[GUARD:GUARD + size]


def run(dev, need, q, cache, table, lengths, length, **kw):
    """The call in workspaces of the size wanted, smaller ones, and a larger one."""
    counts, parents, causal = kw.pop("counts", None), kw.pop("parents", None), kw.get("causal", False)
    if counts is not None:
        kw["counts"] = torch.tensor(counts, dtype=torch.int32, device=dev)
    if parents is not None:
        kw["parents"] = torch.tensor(parents, dtype=torch.int32, device=dev)
    ops.paged_attend(q, cache, table, length, **kw)
    wanted = need[-1]
    assert wanted > 0 or len(lengths) == 64            # (as many sequences as fill the chip)
    for size in (wanted, wanted - 1, wanted // 2 + 8, wanted // 3, wanted + 1000) if wanted else (1000,):
        whole, work = guarded(dev, size)
        for _ in range(2):
            out, lse = ops.paged_attend(q, cache, table, length, workspace=work, **kw)
            check_large(q, cache, table, lengths, out, lse, causal, parents, counts)
            work.fill_(0xff)
        whole[GUARD:GUARD + size] = 0xff
        assert (whole == 0xff).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Q,G,D", [(1, 4, 128), (20, 2, 64), (5, 5, 80), (150, 4, 128), (90, 8, 64)])
def test_one_length_for_all(dev, need, Q, G, D, dtype):
    n, H = 9000, 2
    cache, table = make_pool(dev, [n] * 2, H, D, 64, dtype, 51)
    q = queries(dev, 2, Q, H * G, D, dtype, 52)
    run(dev, need, q, cache, table, [n] * 2, n, causal=Q > 1)


@pytest.mark.parametrize("Q,G,D", [(1, 4, 128), (20, 2, 64), (150, 4, 128)])
@pytest.mark.parametrize("lengths", [
    [9000] + [17] * 9, [0, 5000, 0, 1, 129, 4999], [2500] * 4, [1] * 63 + [6000], [0, 0, 4000], [0] * 4,
])
def test_lengths_on_the_device(dev, need, lengths, Q, G, D):
    """Slots that the sharing by length leaves over are not written, and must not be
    read; the shares lie at the workspace's end."""
    B, H = len(lengths), 2
    cache, table = make_pool(dev, lengths, H, D, 64, torch.bfloat16, 53, width=160)
    q = queries(dev, B, Q, H * G, D, torch.bfloat16, 54)
    length = torch.tensor(lengths, dtype=torch.int32, device=dev)
    run(dev, need, q, cache, table, lengths, length)
    run(dev, need, q, cache, table, lengths, length, causal=True,
        counts=[Q if b % 3 else b % 2 * (Q // 2) for b in range(B)])


@pytest.mark.parametrize("Q", [16, 64])
def test_trees(dev, need, Q):
    rng = np.random.default_rng(55)
    lengths = [4000, 300, 2100]
    cache, table = make_pool(dev, lengths, 2, 128, 16, torch.bfloat16, 56)
    q = queries(dev, 3, Q, 8, 128, torch.bfloat16, 57)
    length = torch.tensor(lengths, dtype=torch.int32, device=dev)
    run(dev, need, q, cache, table, lengths, length, parents=[random_tree(rng, Q) for _ in range(3)])
