"""The paged cache at its edges on the GPU: fused projections rotated in place, nothing to
do, views and shared pages, several streams, and a draft's step captured into a graph."""
import numpy as np
import pytest
import torch

from nanokv_amd import ops
from tests.test_gpu_paged import TYPES, check_large, freqs_of, make_pool, queries, random_tree

pytestmark = pytest.mark.gpu


def clone(cache):
    return ops.PagedCache(cache.k.clone(), cache.v.clone())


def same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [1, 37])
def test_append_from_a_fused_projection_in_place(dev, T, interleaved):
    B, H, Hq, D = 2, 2, 6, 96
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn((B, T, Hq + 2 * H, D), generator=g).bfloat16().to(dev)
    q, k, v = qkv.split([Hq, H, H], 2)
    cache, table = make_pool(dev, [T + 9] * B, H, D, 16, torch.bfloat16, 2)
    other = clone(cache)
    kept = k.clone(), v.clone()
    kw = dict(freqs=freqs_of(64, dev), interleaved=interleaved)
    want = ops.paged_append(other, table, k.contiguous(), v.contiguous(), 9, q=q.contiguous(), **kw)
    assert ops.paged_append(cache, table, k, v, 9, q=q, q_out=q, **kw) is q
    assert torch.equal(q, want) and torch.equal(k, kept[0]) and torch.equal(v, kept[1])
    assert same_bits(cache.k, other.k) and same_bits(cache.v, other.v)
    # queries and keys in one place cannot both be kept
    with pytest.raises(RuntimeError, match="overlaps the rows"):
        ops.paged_append(cache, table, k, v, 9, q=k, q_out=k, **kw)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_nothing_to_do(dev, name):
    H, D = 2, 64
    cache, table = make_pool(dev, [40, 33], H, D, 16, TYPES[name], 3)
    before = clone(cache)
    row = lambda B, T, h: torch.zeros((B, T, h, D), dtype=TYPES[name], device=dev)
    none = torch.empty((0, 3), dtype=torch.int32, device=dev)
    freqs = freqs_of(64, dev)
    assert ops.paged_append(cache, table, row(2, 0, H), row(2, 0, H), 5, q=row(2, 0, 4), freqs=freqs).shape == (2, 0, 4, D)
    assert ops.paged_append(cache, none, row(0, 5, H), row(0, 5, H), 5) is None
    out, lse = ops.paged_attend(row(2, 0, 4), cache, table, 40)
    assert out.shape == (2, 0, 4, D) and lse.shape == (2, 4, 0)
    out, lse = ops.paged_attend(row(0, 7, 4), cache, none, 40)
    assert out.shape == (0, 7, 4, D) and lse.shape == (0, 4, 7)
    assert ops.paged_commit(cache, none, 0, none).shape == (0,)
    # no keys at all: an empty table, or lengths of zero
    zero = torch.zeros(2, dtype=torch.int32, device=dev)
    for Q in (1, 50, 700):
        for t, n in ((torch.empty((2, 0), dtype=torch.int32, device=dev), 0), (table, 0), (table, zero)):
            for kw in (dict(), dict(causal=True)):
                out, lse = ops.paged_attend(queries(dev, 2, Q, 4, D, TYPES[name], 4), cache, t, n, **kw)
                assert (out == 0).all() and torch.isneginf(lse).all()
    out, lse = ops.paged_attend(queries(dev, 2, 3, 4, D, TYPES[name], 4), cache, table, 40, counts=zero)
    assert (out == 0).all() and torch.isneginf(lse).all()
    assert ops.paged_append(cache, table, row(2, 3, H), row(2, 3, H), 5, counts=zero) is None
    assert same_bits(cache.k, before.k) and same_bits(cache.v, before.v)


@pytest.mark.parametrize("Q,n", [(1, 900), (1, 9000), (20, 900), (200, 3000)])
def test_views_and_shared_pages(dev, Q, n):
    """A table that is a slice of a larger one or one row for all, queries and outputs in
    another layout, sequences that share pages: the same bits as plain tensors give."""
    H, Hq, D, page, B = 8, 16, 128, 32, 3
    cache, one = make_pool(dev, [n], H, D, page, torch.bfloat16, 5)
    plain = one.expand(B, -1).contiguous()
    q = queries(dev, B, Q, Hq, D, torch.bfloat16, 6)
    lengths = [n, n - 77, 5]
    length = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = ops.paged_attend(q, cache, plain, length)
    check_large(q, cache, plain, lengths, *want)
    wide = torch.full((B, plain.shape[1] + 7), -5, dtype=torch.int32, device=dev)
    wide[:, 3:-4] = plain
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    place = torch.empty((B, Hq, Q, D), dtype=q.dtype, device=dev).transpose(1, 2)
    holes = torch.full((B, Q, Hq, D + 8), 7.0, dtype=q.dtype, device=dev)
    for t in (one.expand(B, -1), wide[:, 3:-4]):
        for out in (None, place, holes[..., :D]):
            got = ops.paged_attend(turned, cache, t, length, out=out)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (holes[..., D:] == 7).all()
    got = ops.paged_attend(q, cache, plain, length, return_lse=False)
    assert torch.equal(got[0], want[0]) and got[1] is None


@pytest.mark.parametrize("Q,Hq", [(1, 8), (3, 16), (24, 8), (150, 16)])
@pytest.mark.parametrize("lengths", [
    [9000] + [17] * 9, [0, 5000, 0, 1, 129, 4999], [3000 + 128 * i for i in range(5)], [2500] * 4, [0, 0, 4000],
    [1] * 63 + [6000], [40 * i for i in range(65)],
])
def test_sequences_of_unlike_lengths(dev, Q, Hq, lengths):
    """Splits by length: one long among short ones, empty ones, as many as a wave's lanes
    and one more; some without queries; in a smaller workspace too."""
    B, H, D = len(lengths), 2, 64
    cache, table = make_pool(dev, lengths, H, D, 64, torch.bfloat16, 11)
    q = queries(dev, B, Q, Hq, D, torch.bfloat16, 12)
    length = torch.tensor(lengths, dtype=torch.int32, device=dev)
    check_large(q, cache, table, lengths, *ops.paged_attend(q, cache, table, length))
    counts = [Q if b % 3 else b % 2 * (Q // 2) for b in range(B)]
    ct = torch.tensor(counts, dtype=torch.int32, device=dev)
    for size in (None, 100, 8 * B + 3 * B * Hq * Q * (4 * D + 8)):
        work = None if size is None else torch.empty(size, dtype=torch.uint8, device=dev)
        out, lse = ops.paged_attend(q, cache, table, length, causal=True, counts=ct, workspace=work)
        check_large(q, cache, table, lengths, out, lse, True, None, counts)


def test_calls_on_several_streams_with_splits(dev):
    """Calls of both kernels with key splits, several at once: each has a workspace of its
    own."""
    streams = [torch.cuda.Stream() for _ in range(3)]
    cache, table = make_pool(dev, [20000], 2, 128, 64, torch.bfloat16, 7)
    calls = []
    for i, Q in enumerate((1, 40, 500)):
        q = queries(dev, 1, Q, 4, 128, torch.bfloat16, 8 + i)
        calls.append((q, ops.paged_attend(q, cache, table, 20000)))
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                for q, want in calls[i:] + calls[:i]:
                    got.append((ops.paged_attend(q, cache, table, 20000), want))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("T,n,Hq", [(6, 3000, 8), (70, 2500, 16)])
def test_graph_of_a_drafts_step(dev, T, n, Hq):
    """A tree's tokens appended, attended over key splits and committed in two layers, in
    one graph replayed with other rows, trees and accepted paths, eager work between."""
    rng = np.random.default_rng(9)
    B, H, D, page, M = 2, 2, 128, 16, 5
    lengths = [n, n - 700]
    first, table = make_pool(dev, [x + 6 * M + T for x in lengths], H, D, page, torch.bfloat16, 10)
    layers = [first, clone(first)]
    mirror = [clone(c) for c in layers]
    freqs = freqs_of(D, dev)
    ints = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)
    length, depth, parents, path, accepted = ints(B), ints(B, T), ints(B, T), ints(B, M), ints(B)
    length.copy_(torch.tensor(lengths))
    k, v, q = (torch.zeros((B, T, h, D), device=dev, dtype=torch.bfloat16) for h in (H, H, Hq))
    most = n + 6 * M + T

    def step(caches):
        results = []
        for c in caches:
            turned = ops.paged_append(c, table, k, v, length, q=q, freqs=freqs,
                                      positions=length[:, None] + depth)
            results += ops.paged_attend(turned, c, table, length + T, parents=parents, max_length=most)
        return results + [ops.paged_commit(caches, table, length, path, accepted)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([clone(c) for c in layers])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(layers)
    for i in range(5):
        trees = [random_tree(rng, T, b == 1) for b in range(B)]
        parents.copy_(torch.tensor(trees))
        depth.copy_(torch.tensor(rng.integers(0, 9, (B, T))))
        path.copy_(torch.tensor(np.stack([np.sort(rng.choice(T, M, replace=False)) for _ in range(B)])))
        accepted.copy_(torch.tensor(rng.integers(0, M + 1, B)))
        for x, s in ((k, 20), (v, 30), (q, 40)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(s + i)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        want = step(mirror)
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        for a, b in zip(layers, mirror):
            assert same_bits(a.k, b.k) and same_bits(a.v, b.v)
        length.copy_(want[-1])
    assert length.tolist() == held[-1].tolist()
