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
def check_rows(q, cache, fmt, lengths, causal, out, lse):
    """check_attend with a bound of the row's own: what a weight below fp16's normal
    range is off by (2^-25, where the row's largest is at least 2^12) counts against
    the largest weight that the row gives, not against the loudest value there is."""
    D, B, Q = q.shape[3], q.shape[0], q.shape[1]
    k, v = cache_values(cache, fmt)
    half = 2.0 ** -8 if q.dtype == torch.bfloat16 else 2.0 ** -11
    qd = q.double().cpu().numpy()
    ro, rl, otol, ltol = ref.attend(qd, k, v, lengths, causal, D ** -0.5, half)
    end = ref.visible(B, Q, lengths, causal)
    top = np.repeat(np.nan_to_num(cache.v_scale.double().cpu().numpy()), 64, 2) * float(ref.TOP[fmt])
    G = q.shape[2] // k.shape[1]
    for b in range(B):
        for h in range(q.shape[2]):
            n = int(end[b].max())
            hidden = np.arange(n)[None] >= end[b][:, None]
            z = np.where(hidden, -np.inf, qd[b, :, h] @ k[b, h // G, :n].T * D ** -0.5)
            w = np.exp(z - rl[b, h][:, None]) * top[b, h // G, :n]
            mag = np.where(hidden, 0, np.abs(qd[b, :, h]) @ np.abs(k[b, h // G, :n]).T * D ** -0.5)
            ez = (D + 4) * 2.0 ** -24 * mag + 2.0 ** -21
            a = (w / top[b, h // G, :n])[:, :, None] * np.abs(v[b, h // G, :n])[None]
            # the weight's two roundings, the score's, the output's, and a partial result's
            # below fp16's normal range
            otol[b, :, h] = (a * (2.0 ** -10 + 4 * ez)[:, :, None]).sum(1) * 1.01 \
                + half * np.abs(ro[b, :, h]) + (n * 2.0 ** -37 * w.max(1) + 2.0 ** -25 * w.sum(1))[:, None] \
                + (2.0 ** -25 if half == 2.0 ** -11 else 1e-30)
            ltol[b, h] = 2 * (np.exp(z - rl[b, h][:, None]) * ez).sum(1) \
                + 2.0 ** -22 * (np.abs(rl[b, h]) + 16)
    got = out.double().cpu().numpy()
    assert (np.abs(got - ro) <= otol).all(), np.max(np.abs(got - ro) / otol)
    assert (np.abs(lse.double().cpu().numpy() - rl) <= ltol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Q,N", [(1, 700), (9, 700), (100, 700), (1, 8000), (9, 8000), (100, 8000)])
@pytest.mark.parametrize("loud", [2.0 ** 20, 2.0 ** 28, 2.0 ** 40, 2.0 ** 90])
def test_loud_values_without_weight_cost_nothing(dev, dtype, loud, Q, N):
    """Blocks of very large values whose keys have next to no weight: outputs as
    near as the values that count allow, with key splits and without."""
    g = torch.Generator().manual_seed(103)
    k, v = torch.randn((2, 1, N, 2, 64), generator=g).to(dev)
    for first in (0, 256, N - 65):
        v[:, first:first + 64] *= loud
        k[:, first:first + 64] = 0
        k[:, first:first + 64, :, 0] = -200.0              # a score of -200 below
    cache = ops.Cache8.empty(1, 2, N, 64, dev, "int8")
    ops.cache8_write(cache, k, v, 0)
    q = torch.randn((1, Q, 4, 64), generator=g)
    q[..., 0] = 8.0
    q[..., 1:] *= 3                                        # weight on few keys
    q = q.to(dtype).to(dev)
    # (the last block holds loud and other values: its own scale is what it is)
    cache.v_scale[:, :, (N - 65) // 64] = cache.v_scale[:, :, 1]
    out, lse = ops.cache8_attend(q, cache, N)
    check_rows(q, cache, "int8", [N], False, out, lse)
    none = torch.zeros(16, dtype=torch.uint8, device=dev)  # no room for splits
    out, lse = ops.cache8_attend(q, cache, N, workspace=none)
    check_rows(q, cache, "int8", [N], False, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("Q,G", [(60, 1), (150, 1), (150, 4)])
def test_causal_rows_do_not_depend_on_later_values(dev, dtype, fmt, Q, G):
    """Queries before a run of very large values: as near as if it were not there."""
    g = torch.Generator().manual_seed(104)
    N = 2018 + Q
    k, v = torch.randn((2, 2, N, 1, 128), generator=g).to(dev)
    k *= 3
    v[:, N - Q // 2:] *= 2.0 ** 45
    cache = ops.Cache8.empty(2, 1, N, 128, dev, fmt)
    at = torch.tensor([0, 0], dtype=torch.int32, device=dev)
    for first in range(0, N, 64):                          # (a block's scale is its own)
        ops.cache8_write(cache, k[:, first:first + 64], v[:, first:first + 64], at)
        at += 64
    q = torch.randn((2, Q, G, 128), generator=g).to(dtype).to(dev)
    out, lse = ops.cache8_attend(q, cache, N, causal=True)
    seen = 2048 - 2018                                     # queries that see whole quiet blocks only
    few = ops.cache8_attend(q[:, :seen], cache, N - Q + seen, causal=True)
    check_rows(q[:, :seen], cache, fmt, [N - Q + seen] * 2, True, out[:, :seen], lse[:, :, :seen])
    check_rows(q[:, :seen], cache, fmt, [N - Q + seen] * 2, True, *few)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("fmt,dtype,H,G,D,T,start", [
    ("int8", torch.bfloat16, 2, 1, 64, 5, [0, 7, 100, 3, 0]),
    ("e4m3", torch.float16, 1, 4, 128, 9, [0, 7, 100, 3, 0]),
    ("e4m3", torch.bfloat16, 2, 2, 80, 70, [0, 64, 100, 3, 1]),
    ("int8", torch.float16, 1, 2, 64, 300, [0, 64, 1000, 3, 1]),
    ("e4m3", torch.bfloat16, 1, 3, 128, 100, [0, 64, 9000, 3, 1]),      # key splits
])
def test_a_batch_padded_on_the_right(dev, fmt, dtype, H, G, D, T, start, causal):
    """Write, attention and weight with one tensor of counts: each sequence as if it
    were alone, whatever the padding holds."""
    B, counts = len(start), [T, T - 2, 1, 0, T // 2]
    g = torch.Generator().manual_seed(107)
    cache = make_cache(dev, B, H, max(start) + T, D, fmt, 108, start)
    kv = torch.randn((2, B, T, H, D), generator=g)
    q = torch.randn((B, T, H * G, D), generator=g)
    for b, c in enumerate(counts):
        kv[:, b, c:] = float("nan")
        q[b, c:] = float("nan")
    kv, q = kv.to(dtype).to(dev), q.to(dtype).to(dev)
    ints = dict(dtype=torch.int32, device=dev)
    dc, ds = torch.tensor(counts, **ints), torch.tensor(start, **ints)
    ops.cache8_write(cache, kv[0], kv[1], ds, dc)
    lengths = [a + b for a, b in zip(start, counts)]
    n = torch.tensor(lengths, **ints)
    m0 = torch.rand((B, H, cache.cap), generator=g)
    m, other = m0.to(dev), torch.full((B, H, cache.cap), float("nan"), device=dev)
    for work in (None, torch.zeros(16, dtype=torch.uint8, device=dev)):
        out, lse = ops.cache8_attend(q, cache, n, causal=causal, counts=dc, workspace=work)
        bad = lse.clone()                     # (nor is the padding's lse read)
        for b, c in enumerate(counts):
            assert (out[b, c:] == 0).all() and torch.isneginf(lse[b, :, c:]).all()
            bad[b, :, c:] = 0.0
            if c:
                one = ops.Cache8(*(t[b:b + 1].contiguous() for t in (cache.k, cache.v, cache.k_scale,
                                                                     cache.v_scale)), D)
                check_rows(q[b:b + 1, :c], one, fmt, lengths[b:b + 1], causal, out[b:b + 1, :c],
                           lse[b:b + 1, :, :c])
        m.copy_(m0)
        ops.cache8_mass(q, cache, bad, m, n, out=other, causal=causal, counts=dc, workspace=work)
        ops.cache8_mass(q, cache, bad, m, n, causal=causal, counts=dc, workspace=work)
        assert torch.equal(m, other)
        k, _ = cache_values(cache, fmt)
        for b, c in enumerate(counts):
            if c:
                rm, tol = ref.mass(q[b:b + 1, :c].double().cpu().numpy(), k[b:b + 1],
                                   lse[b:b + 1, :, :c].double().cpu().numpy(), m0[b:b + 1].numpy(),
                                   lengths[b:b + 1], causal, D ** -0.5)
                assert (np.abs(m[b:b + 1].double().cpu().numpy() - rm) <= tol).all()
            else:
                assert torch.equal(m[b].cpu(), m0[b])
    # counts outside [0, Q] are those
    wide = torch.tensor([T + 5 if c == T else -3 if c == 0 else c for c in counts], **ints)
    again, l2 = ops.cache8_attend(q, cache, n, causal=causal, counts=wide, workspace=work)
    assert torch.equal(again, out) and torch.equal(l2, lse)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("fmt,dtype,Q,G,N,causal", [
    ("int8", torch.bfloat16, 1, 4, 700, False), ("e4m3", torch.float16, 9, 2, 130, True),
    ("e4m3", torch.bfloat16, 40, 2, 1000, True), ("int8", torch.bfloat16, 600, 2, 900, False),
])
def test_queries_that_are_not_finite_add_no_weight(dev, fmt, dtype, Q, G, N, causal, value):
    """The masses equal those of the other rows alone, to the last bit."""
    cache = make_cache(dev, 2, 1, N, 64, fmt, 109, [N, N - 64])
    n = torch.tensor([N, N - 64], dtype=torch.int32, device=dev)
    q = torch.randn((2, Q, G, 64), generator=torch.Generator().manual_seed(110)).to(dtype).to(dev)
    _, lse = ops.cache8_attend(q, cache, n, causal=causal)
    bad = q.clone()
    bad[0, Q // 2, 1, 5] = value
    _, l2 = ops.cache8_attend(bad, cache, n, causal=causal)
    assert torch.isnan(l2[0, 1, Q // 2])
    lse[0, 1, Q // 2] = float("-inf")
    m0 = torch.rand((2, 1, cache.cap), generator=torch.Generator().manual_seed(111)).to(dev)
    for work in (None, torch.zeros(16, dtype=torch.uint8, device=dev)):
        want = ops.cache8_mass(q, cache, lse, m0.clone(), n, causal=causal, workspace=work)
        got = ops.cache8_mass(bad, cache, l2, m0.clone(), n, causal=causal, workspace=work)
        assert torch.equal(got, want) and torch.isfinite(got).all()
        for other in (float("inf"), float("nan")):
            l2[0, 1, Q // 2] = other
            got = ops.cache8_mass(q, cache, l2, m0.clone(), n, causal=causal, workspace=work)
            assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fmt", FORMATS)
def test_zeros_keep_their_sign(dev, fmt, dtype):
    """-0 and quotients that round to it, in finite blocks and beside infinities and
    NaN, and under a scale that grows: the codes of the division, to the last bit."""
    cache = ops.Cache8.empty(1, 1, 192, 64, dev, fmt)
    x = torch.randn((1, 150, 1, 64), generator=torch.Generator().manual_seed(112))
    x[:, :, :, ::3] = -0.0
    x[:, :, :, 1::6] *= -1e-6
    x[0, 70, 0, 5], x[0, 71, 0, 8] = float("inf"), float("nan")
    x[0, 135:] *= 3
    x = x.to(dtype).to(dev)
    want = raw(cache.k).copy(), cache.k_scale.cpu().numpy()
    for first, last in ((0, 130), (130, 135), (135, 150)):
        part = x[:, first:last].contiguous()
        ops.cache8_write(cache, part, part, first)
        want = ref.write(*want, part.float().cpu().numpy(), [first], [last - first], fmt)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert np.array_equal(scale.cpu().numpy(), want[1])
        assert np.array_equal(raw(codes).view(np.uint8), want[0].view(np.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
def test_a_write_over_old_rows(dev, fmt):
    """Rows behind those written keep their codes; a write that starts on a block's
    first row sets its scale anew, also below the old one, one that starts inside
    the block does not lower it."""
    cache = make_cache(dev, 1, 2, 192, 64, fmt, 113)
    x = torch.randn((1, 20, 2, 64), generator=torch.Generator().manual_seed(114)).to(dev) * 2.0 ** -20
    for start in (64, 130):
        before = raw(cache.k).copy(), cache.k_scale.cpu().numpy()
        ops.cache8_write(cache, x, x, start)
        rc, rs = ref.write(*before, x.cpu().numpy(), [start], [20], fmt)
        assert np.array_equal(raw(cache.k), rc) and np.array_equal(cache.k_scale.cpu().numpy(), rs)
        assert np.array_equal(rc[:, :, start + 20:], before[0][:, :, start + 20:])
        lower = rs[:, :, start // 64] < before[1][:, :, start // 64]
        assert lower.all() if start % 64 == 0 else not lower.any()


def test_mass_over_a_cache_written_in_the_same_graph(dev):
    """A captured write and the weight over what it wrote: every replay with new
    tokens against the plain form and against eager calls between."""
    B, H, G, D, T = 2, 2, 2, 64, 70
    start, lengths = [130, 7], [200, 77]
    ints = dict(dtype=torch.int32, device=dev)
    ds, n = torch.tensor(start, **ints), torch.tensor(lengths, **ints)
    cache = ops.Cache8.empty(B, H, 256, D, dev, "int8")
    q = torch.zeros((B, 40, H * G, D), dtype=torch.bfloat16, device=dev)
    kv = torch.zeros((2, B, T, H, D), dtype=torch.bfloat16, device=dev)
    m0 = torch.rand((B, H, cache.cap), generator=torch.Generator().manual_seed(115)).to(dev)

    def calls(c):
        ops.cache8_write(c, kv[0], kv[1], ds)
        _, lse = ops.cache8_attend(q, c, n, causal=True)
        out = torch.empty_like(m0)
        return lse, ops.cache8_mass(q, c, lse, m0, n, out=out, causal=True)

    def empty(c):
        for t in (c.k, c.v):
            t.zero_()
        for t in (c.k_scale, c.v_scale):
            t.fill_(1.0)

    calls(ops.Cache8.empty(B, H, 256, D, dev, "int8"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lse, got = calls(cache)
    for i in range(3):
        g = torch.Generator().manual_seed(116 + i)
        q.copy_(torch.randn(q.shape, generator=g))
        kv.copy_(torch.randn(kv.shape, generator=g))
        empty(cache)
        graph.replay()
        torch.cuda.synchronize()
        k, _ = cache_values(cache, "int8")
        rm, tol = ref.mass(q.double().cpu().numpy(), k, lse.double().cpu().numpy(), m0.cpu().numpy(),
                           lengths, True, D ** -0.5)
        assert (np.abs(got.double().cpu().numpy() - rm) <= tol).all()
        other = ops.Cache8.empty(B, H, 256, D, dev, "int8")
        l2, want = calls(other)
        assert torch.equal(got, want) and torch.equal(lse, l2) and torch.equal(cache.k, other.k)


@pytest.mark.parametrize("softmax_scale", [1e-40, 1e-25, 1e30, 3e38])
@pytest.mark.parametrize("Q,G,causal", [(1, 2, False), (9, 2, True), (100, 1, True)])
def test_softmax_scales_of_any_size(dev, Q, G, causal, softmax_scale):
    """Beside keys of zeros, whose scale is the least there is: hidden keys stay
    hidden, and where every visible score is zero the weights are equal."""
    cache = make_cache(dev, 1, 1, 192, 64, "int8", 120, [170])
    for first, s in ((0, float(ref.TINY) / 127), (64, float(ref.TINY) / 127), (128, 1e12)):
        cache.k_scale[:, :, first // 64] = s
    cache.k.zero_()
    q = torch.randn((1, Q, G, 64), generator=torch.Generator().manual_seed(121)).bfloat16().to(dev)
    n = torch.tensor([170], dtype=torch.int32, device=dev)
    out, lse = ops.cache8_attend(q, cache, n, causal=causal, softmax_scale=softmax_scale)
    check_attend(q, cache, "int8", [170], causal, out, lse, softmax_scale)
    m = torch.zeros((1, 1, cache.cap), device=dev)
    ops.cache8_mass(q, cache, lse, m, n, causal=causal, softmax_scale=softmax_scale)
    rm, tol = ref.mass(q.double().cpu().numpy(), cache_values(cache, "int8")[0],
                       lse.double().cpu().numpy(), np.zeros((1, 1, 192)), [170], causal, softmax_scale)
    assert (np.abs(m.double().cpu().numpy() - rm) <= tol).all()


@pytest.mark.parametrize("T,N", [(3, 5000), (90, 5000)])
def test_counts_of_a_captured_call_may_change(dev, T, N):
    """One graph of a write, attention and weight, replayed with other counts and
    lengths, equals eager calls between the replays; so it does on a stream of its own."""
    B, H, G, D = 3, 2, 2, 128
    ints = dict(dtype=torch.int32, device=dev)
    base = make_cache(dev, B, H, N + T, D, "e4m3", 122)
    x = torch.randn((3, B, T, H * G, D), generator=torch.Generator().manual_seed(123)).half().to(dev)
    start, counts = torch.zeros(B, **ints), torch.zeros(B, **ints)
    m0 = torch.zeros((B, H, base.cap), device=dev)

    def calls():
        c = ops.Cache8(*(t.clone() for t in (base.k, base.v, base.k_scale, base.v_scale)), D)
        ops.cache8_write(c, x[0, :, :, :H], x[1, :, :, :H], start, counts)
        n = start + counts
        out, lse = ops.cache8_attend(x[2], c, n, causal=True, counts=counts)
        return out, lse, ops.cache8_mass(x[2], c, lse, m0, n, out=torch.empty_like(m0), causal=True,
                                         counts=counts), c.k, c.v_scale

    calls()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        got = calls()
    for st, ct in (([0, 70, N], [T, 1, T]), ([N, 0, 5], [T - 1, 0, T]), ([1, 2, 3], [0, 0, 0]),
                   ([N, N, N], [T, T, T])):
        start.copy_(torch.tensor(st))
        counts.copy_(torch.tensor(ct))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = calls()
        torch.cuda.current_stream().wait_stream(side)
        for a, b, c in zip(got, calls(), other):
            assert torch.equal(a, b) and torch.equal(a, c)
