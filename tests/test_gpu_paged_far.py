"""The paged cache at the end of what its lengths can say."""
import pytest
import torch

from nanokv_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("device_start", [False, True])
def test_committed_lengths_stay_in_their_type(dev, device_start):
    """A table of more rows than an int32 counts (no pages behind it): lengths past the
    type's end stop there, and do not turn negative."""
    top = 2 ** 31 - 1
    cache = ops.PagedCache.empty(1, 1024, 1, 8, dev)
    table = torch.full((3, 2 ** 21 + 4), -1, dtype=torch.int32, device=dev)
    rows = torch.zeros((3, 4), dtype=torch.int32, device=dev)
    counts = torch.tensor([0, 1, 4], dtype=torch.int32, device=dev)
    for start in (top, top - 1, top - 2, top - 4):
        at = torch.full((3,), start, dtype=torch.int32, device=dev) if device_start else start
        got = ops.paged_commit(cache, table, at, rows, counts)
        assert got.tolist() == [min(top, start + n) for n in (0, 1, 4)]
    assert not cache.k.any() and not cache.v.any()
