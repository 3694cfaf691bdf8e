"""The 8-bit cache on the GPU at the edges of what its calls allow."""
import numpy as np
import pytest
import torch

from tests import _cache8_ref as ref
from tests.test_gpu_cache8 import FORMATS, cache_values, check_attend, make_cache, raw
from nanokv_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("fmt", FORMATS)
def test_mass_of_no_queries_is_the_mass(dev, fmt, causal):
    """To the last bit, in place and into another array, below and past the length."""
    cache = make_cache(dev, 2, 3, 192, 64, fmt, 100, [192, 70])
    m = torch.rand((2, 3, cache.cap), generator=torch.Generator().manual_seed(101)).to(dev)
    m[:, :, ::5] = -0.0
    m[0, 1, 3] = float("nan")
    was = m.cpu().numpy().view(np.uint32).copy()
    n = torch.tensor([192, 70], dtype=torch.int32, device=dev)
    q = torch.empty((2, 0, 6, 64), dtype=torch.bfloat16, device=dev)
    out, lse = ops.cache8_attend(q, cache, n, causal=causal)
    assert out.shape == q.shape and lse.shape == (2, 6, 0)
    other = torch.full_like(m, 7.0)
    assert ops.cache8_mass(q, cache, lse, m, n, out=other, causal=causal) is other
    assert ops.cache8_mass(q, cache, lse, m, n, causal=causal) is m
    for t in (m, other):
        assert np.array_equal(t.cpu().numpy().view(np.uint32), was)
