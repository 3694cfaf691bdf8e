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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Q,N", [(1, 700), (9, 700), (100, 700), (1, 8000), (100, 8000)])
@pytest.mark.parametrize("loud", [2.0 ** 40, 2.0 ** 76, 2.0 ** 100, 1e38])
def test_log_sums_do_not_depend_on_the_values(dev, dtype, loud, Q, N):
    """Values of any finite size beside blocks of zeros, as the write takes them:
    the log sums are those of the keys, the outputs finite numbers."""
    g = torch.Generator().manual_seed(102)
    k, v = torch.randn((2, 1, N, 2, 64), generator=g).to(dev)
    v[:, :64] *= loud / v[:, :64].abs().max()
    v[:, 128:192] = 0
    v[:, 256:320] = 0                         # (the first block's wave, where it has two)
    v[:, -65:] = 0
    cache = ops.Cache8.empty(1, 2, N, 64, dev, "int8")
    ops.cache8_write(cache, k, v, 0)
    q = torch.randn((1, Q, 4, 64), generator=g).to(dtype).to(dev)
    out, lse = ops.cache8_attend(q, cache, N)
    if dtype == torch.bfloat16:
        check_attend(q, cache, "int8", [N], False, out, lse)
    else:                                     # (outputs beyond the type's range are infinite)
        assert not torch.isnan(out).any()
    cv = cache_values(cache, "int8")
    _, rl, _, ltol = ref.attend(q.double().cpu().numpy(), cv[0], cv[1] / loud, [N], False, 0.125, 2.0 ** -8)
    assert (np.abs(lse.double().cpu().numpy() - rl) <= ltol).all()
    # as those beside even values are
    quiet = ops.Cache8(cache.k, cache.v, cache.k_scale, torch.ones_like(cache.v_scale), 64)
    _, l2 = ops.cache8_attend(q, quiet, N)
    assert (np.abs(l2.double().cpu().numpy() - rl) <= ltol).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("fmt,D,Q,N,H", [("int8", 128, 1, 700, 2), ("e4m3", 64, 7, 20_000, 1),
                                         ("e4m3", 128, 5, 4096, 40), ("int8", 64, 20, 16_384, 8),
                                         ("e4m3", 64, 90, 300, 1), ("int8", 128, 90, 9000, 1)])
def test_queries_that_are_not_finite_stay_in_their_rows(dev, fmt, D, Q, N, H, value):
    """In every kernel, with key splits and without: the row is NaN, and no other."""
    cache = make_cache(dev, 1, H, N, D, fmt, 105, [N])
    q = torch.randn((1, Q, 2 * H, D), generator=torch.Generator().manual_seed(106)).bfloat16().to(dev)
    bad = q.clone()
    bad[0, Q // 2, 1, 5] = value
    keep = torch.ones((Q, 2 * H), dtype=torch.bool, device=dev)
    keep[Q // 2, 1] = False
    for work in (None, torch.zeros(16, dtype=torch.uint8, device=dev)):
        clean, lse = ops.cache8_attend(q, cache, N, workspace=work)
        out, l2 = ops.cache8_attend(bad, cache, N, workspace=work)
        assert torch.isnan(out[0, Q // 2, 1]).all() and torch.isnan(l2[0, 1, Q // 2])
        assert torch.equal(out[0][keep], clean[0][keep]) and torch.equal(l2[0].T[keep], lse[0].T[keep])
