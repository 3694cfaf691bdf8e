"""The paged cache on the GPU: appended and moved rows against 64-bit rotation and to
the last bit, attention of tokens, chunks and trees against 64 bits with derived
bounds, and a run of them together."""
import numpy as np
import pytest
import torch

from tests import _paged_ref as ref
from nanokv_amd import ops

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# few query rows: bf16 weights in two parts, what the first leaves is rounded again
FINE = {"bf16": 2.0 ** -16, "fp16": 2.0 ** -11}


def f64(t):
    return t.detach().double().cpu().numpy()


def bits(t):
    return t.detach().view(torch.int16).cpu().numpy()


def make_pool(dev, lengths, H, D, page, dtype, seed, extra=2, width=None):
    """Pools whose rows below the lengths are random and all others NaN, and a table of
    pages in random order, -1 behind them."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + extra
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lengths), width or max(1, max(need))), -1, dtype=torch.int32)
    k, v = (torch.full((pages, H, page, D), float("nan"), dtype=dtype) for _ in range(2))
    at = 0
    for b, n in enumerate(lengths):
        for i in range(need[b]):
            p = order[at]
            at += 1
            table[b, i] = p
            rows = min(page, n - i * page)
            for x in (k, v):
                x[p, :, :rows] = torch.randn((H, rows, D), generator=g).to(dtype)
    return ops.PagedCache(k.to(dev), v.to(dev)), table.to(dev)


def queries(dev, B, Q, Hq, D, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn((B, Q, Hq, D), generator=g)).to(dtype).to(dev)


def check(q, cache, table, lengths, out, lse, causal=False, parents=None, counts=None, scale=None,
          W=None):
    B, Q, Hq, D = q.shape
    name = "bf16" if q.dtype == torch.bfloat16 else "fp16"
    u = ref.HALF[name]
    tab, pk, pv = table.cpu().numpy(), f64(cache.k), f64(cache.v)
    got, gl, qq = f64(out), f64(lse), f64(q)
    for b in range(B):
        n = lengths[b]
        c = Q if counts is None else min(max(counts[b], 0), Q)
        tree = None if parents is None else (parents if np.ndim(parents) == 1 else parents[b])
        see = ref.visible(Q, n, c, causal, tree)
        (k, there), (v, _) = ref.gather(pk, tab[b], n), ref.gather(pv, tab[b], n)
        see &= there[None]
        unseen = ~see.any(0)
        k[:, unseen], v[:, unseen] = 0, 0
        ro, rl, ot, lt = ref.attend(qq[b], k, v, see, scale or D ** -0.5, u, u if W is None else W)
        assert np.isfinite(got[b][see.any(1)]).all()
        err = np.abs(got[b] - ro) - ot
        assert (err <= 0).all(), (b, err.max(), np.unravel_index(err.argmax(), err.shape))
        empty = np.isneginf(rl)
        assert np.array_equal(np.isneginf(gl[b]), empty)
        assert (np.moveaxis(got[b], 1, 0)[empty] == 0).all()
        assert (np.abs(gl[b][~empty] - rl[~empty]) <= lt[~empty]).all()


def random_tree(rng, n, loose=False):
    """Parents of n tokens: each any lower one, the first none; loose: some others none
    too, by any number outside [0, t)."""
    parents = [-1] + [int(rng.integers(0, t)) for t in range(1, n)]
    if loose:
        for t in range(n):
            if rng.random() < 0.2:
                parents[t] = int(rng.choice([-1, -7, t, t + 5, 2 ** 31 - 1, -2 ** 31]))
    return parents


# ---------------------------------------------------------------- append
def check_append(dev, cache, table, k, v, starts, got, before, counts=None, q=None, freqs=None,
                 positions=None, interleaved=False):
    """The pools' rows and the rotated queries; rows that are not written keep their
    bits."""
    name = "bf16" if cache.k.dtype == torch.bfloat16 else "fp16"
    u, f16 = ref.HALF[name], name == "fp16"
    B, T = k.shape[:2]
    page, tab = cache.page, table.cpu().numpy()
    pages = cache.k.shape[0]
    pk, after = f64(cache.k), [bits(cache.k), bits(cache.v)]
    vv = bits(v.to(cache.v.dtype))
    fr = None if freqs is None else freqs.cpu().numpy()
    written = np.zeros((pages, page), bool)
    for b in range(B):
        n = T if counts is None else min(max(counts[b], 0), T)
        at = np.arange(starts[b], starts[b] + T) if positions is None else np.asarray(positions[b])
        kk, mag = f64(k[b]), np.zeros(tuple(k[b].shape))
        if fr is not None:
            kk, mag = ref.rotate(kk, at, fr, interleaved)
        tol = ref.rotate_bound(kk, mag, u, f16)
        for t in range(n):
            s = ref.slots(tab[b], page, starts[b] + t)
            if s is None or not 0 <= s[0] < pages:
                continue
            written[s] = True
            assert (np.abs(pk[s[0], :, s[1]] - kk[t]) <= tol[t]).all(), (b, t)
            assert np.array_equal(after[1][s[0], :, s[1]], vv[b, t])
        if q is not None:
            qq, mag = ref.rotate(f64(q[b]), at, fr, interleaved)
            tol = ref.rotate_bound(qq, mag, u, f16)
            assert (np.abs(f64(got[b]) - qq) <= tol)[:n].all()
    for a, c in zip(after, before):
        assert np.array_equal(np.moveaxis(a, 1, 2)[~written], np.moveaxis(c, 1, 2)[~written])
    return written


def freqs_of(rot, dev, theta=10000.0):
    return (theta ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))).float().to(dev)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("src", ["same", "fp32"])
@pytest.mark.parametrize("D,rot,interleaved,page,T,start", [
    (128, 128, False, 16, 1, 0), (128, 128, True, 16, 1, 15), (128, 64, False, 64, 40, 60),
    (64, 64, True, 32, 33, 1), (80, 80, False, 16, 65, 100), (96, 48, False, 128, 20, 3),
    (72, 72, True, 16, 17, 31), (8, 8, True, 16, 50, 2), (120, 24, True, 32, 9, 0), (40, 16, False, 16, 5, 14),
])
def test_append_rotates_and_writes(dev, name, src, D, rot, interleaved, page, T, start):
    B, H, G = 2, 2, 3
    dtype = TYPES[name]
    cache, table = make_pool(dev, [start + T] * B, H, D, page, dtype, 1)
    before = [bits(cache.k), bits(cache.v)]
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn((B, T, (G + 2) * H, D), generator=g).to(dtype if src == "same" else torch.float32).to(dev)
    q, k, v = qkv.split([G * H, H, H], 2)
    freqs = freqs_of(rot, dev)
    got = ops.paged_append(cache, table, k, v, start, q=q, freqs=freqs, interleaved=interleaved)
    assert got.dtype == dtype and got.shape == q.shape
    written = check_append(dev, cache, table, k, v, [start] * B, got, before, q=q, freqs=freqs,
                           interleaved=interleaved)
    assert written.sum() == B * T


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_append_without_rotation_keeps_every_bit(dev, name):
    """NaN, infinities and signs among them; D odd in 16-column units."""
    dtype, D = TYPES[name], 88
    cache, table = make_pool(dev, [70], 3, D, 16, dtype, 3)
    before = [bits(cache.k), bits(cache.v)]
    k, v = (torch.randint(-32768, 32767, (1, 30, 3, D), generator=torch.Generator().manual_seed(s),
                          dtype=torch.int16).to(dev) for s in (4, 5))
    quiet = lambda x: torch.where(x.view(dtype).isnan(), torch.full_like(x, 0x7FC0 if name == "bf16" else 0x7E00), x).view(dtype)
    k, v = quiet(k), quiet(v)
    assert ops.paged_append(cache, table, k, v, 40) is None
    for pool, x, old in ((cache.k, k, before[0]), (cache.v, v, before[1])):
        new = bits(pool)
        for t in range(30):
            p, r = ref.slots(table[0].tolist(), 16, 40 + t)
            assert np.array_equal(new[p, :, r], bits(x)[0, t])
            old[p, :, r] = new[p, :, r]
        assert np.array_equal(new, old)


def test_append_ragged_starts_counts_bad_pages_and_the_tables_end(dev):
    B, H, D, page, T = 7, 2, 64, 16, 40
    lengths = [48] * B
    cache, table = make_pool(dev, lengths, H, D, page, torch.bfloat16, 6)
    table[3, 1] = -1
    table[4, 1] = cache.k.shape[0]
    table[4, 2] = 2 ** 31 - 1
    starts, counts = [0, 5, 30, 2, 0, 48, -9], [40, 0, 40, 41, 40, 3, 7]
    before = [bits(cache.k), bits(cache.v)]
    g = torch.Generator().manual_seed(7)
    k, v, q = (torch.randn((B, T, h, D), generator=g).bfloat16().to(dev) for h in (H, H, 4))
    freqs = freqs_of(64, dev)
    st, ct = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (starts, counts))
    got = ops.paged_append(cache, table, k, v, st, counts=ct, q=q, freqs=freqs)
    clamped = [min(max(s, 0), 48) for s in starts]
    check_append(dev, cache, table, k, v, clamped, got, before, counts, q, freqs)
    for b, n in enumerate(counts):
        assert (got[b, min(n, T):] == 0).all()
    # in place, rows past counts are left as they were
    mine = q.clone()
    assert ops.paged_append(cache, table, k, v, st, counts=ct, q=mine, q_out=mine, freqs=freqs) is mine
    for b, n in enumerate(counts):
        n = min(n, T)
        assert torch.equal(mine[b, :n], got[b, :n]) and torch.equal(mine[b, n:], q[b, n:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_far_positions(dev, interleaved):
    """Angles of positions up to 2^31 are those of 64 bits."""
    B, T, H, D = 2, 6, 1, 128
    cache, table = make_pool(dev, [T] * B, H, D, 16, torch.float16, 8)
    before = [bits(cache.k), bits(cache.v)]
    positions = [[0, -1, 1000003, 2 ** 31 - 1, -2 ** 31, 131071], [7, 7, 7, 8, 8, 9]]
    k, v, q = (torch.randn((B, T, H, D), generator=torch.Generator().manual_seed(s)).half().to(dev)
               for s in (9, 10, 11))
    freqs = freqs_of(128, dev, 500000.0)
    pos = torch.tensor(positions, dtype=torch.int32, device=dev)
    got = ops.paged_append(cache, table, k, v, 0, q=q, freqs=freqs, positions=pos, interleaved=interleaved)
    check_append(dev, cache, table, k, v, [0] * B, got, before, q=q, freqs=freqs, positions=positions,
                 interleaved=interleaved)
    one = ops.paged_append(cache, table, k, v, 0, q=q, freqs=freqs, positions=pos[0].contiguous(),
                           interleaved=interleaved)
    assert torch.equal(one[0], got[0]) and not torch.equal(one[1], got[1])


def test_append_many_rows(dev):
    """Where a thread takes several heads of a token."""
    B, T, H, Hq, D, page = 3, 1333, 4, 16, 128, 32
    cache, table = make_pool(dev, [T + 5] * B, H, D, page, torch.bfloat16, 12)
    before = [bits(cache.k), bits(cache.v)]
    g = torch.Generator().manual_seed(13)
    k, v, q = (torch.randn((B, T, h, D), generator=g).bfloat16().to(dev) for h in (H, H, Hq))
    freqs = freqs_of(128, dev)
    got = ops.paged_append(cache, table, k, v, 5, q=q, freqs=freqs)
    check_append(dev, cache, table, k, v, [5] * B, got, before, q=q, freqs=freqs)


# ---------------------------------------------------------------- attend
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Hq,H,D,page,lengths", [
    (1, 4, 1, 128, 16, [1]), (3, 8, 2, 128, 16, [31, 0, 33]), (2, 7, 1, 64, 32, [500, 64]),
    (2, 16, 1, 80, 16, [333, 17]), (1, 24, 3, 96, 64, [129]), (2, 2, 2, 40, 128, [100, 257]),
    (1, 32, 1, 128, 16, [2000]), (1, 8, 8, 8, 1024, [1500]), (4, 4, 4, 120, 16, [16, 15, 48, 1]),
])
def test_attend_token(dev, name, B, Hq, H, D, page, lengths):
    cache, table = make_pool(dev, lengths, H, D, page, TYPES[name], 20)
    q = queries(dev, B, 1, Hq, D, TYPES[name], 21)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = ops.paged_attend(q, cache, table, n)
    check(q, cache, table, lengths, out, lse, W=FINE[name])
    if len(set(lengths)) == 1:
        o2, l2 = ops.paged_attend(q, cache, table, lengths[0], return_lse=False)
        assert l2 is None
        check(q, cache, table, lengths, o2, lse, W=FINE[name])


CHUNKS = [
    # B, Hq, H, D, page, Q, lengths, counts
    (1, 2, 2, 128, 16, 33, [33], None), (2, 4, 2, 128, 16, 50, [77, 20], None),
    (2, 4, 1, 64, 32, 70, [200, 70], [70, 3]), (1, 3, 3, 96, 64, 130, [300], None),
    (3, 2, 1, 80, 16, 100, [100, 0, 260], [64, 0, 100]), (1, 1, 1, 128, 128, 257, [700], None),
    (2, 8, 2, 128, 16, 129, [513, 129], [1, 129]), (1, 2, 1, 104, 32, 31, [95], None),
    (1, 5, 1, 64, 16, 300, [290], None), (1, 16, 2, 72, 16, 20, [1111], None),
]


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Hq,H,D,page,Q,lengths,counts", CHUNKS)
def test_attend_chunks(dev, name, causal, B, Hq, H, D, page, Q, lengths, counts):
    """Causal and whole, ragged, padded (rows past counts hold NaN), with rows that see
    nothing."""
    cache, table = make_pool(dev, lengths, H, D, page, TYPES[name], 22)
    q = queries(dev, B, Q, Hq, D, TYPES[name], 23)
    ct = None
    if counts:
        for b, c in enumerate(counts):
            q[b, c:] = float("nan")
        ct = torch.tensor(counts, dtype=torch.int32, device=dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = ops.paged_attend(q, cache, table, n, causal=causal, counts=ct)
    if counts:
        for b, c in enumerate(counts):
            q[b, c:] = 0
    check(q, cache, table, lengths, out, lse, causal=causal, counts=counts)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("B,Hq,H,D,page,Q,lengths,counts", [
    (1, 4, 1, 128, 16, 16, [40], None), (2, 8, 2, 128, 16, 7, [7, 100], None),
    (3, 4, 4, 64, 32, 33, [64, 33, 700], [33, 0, 20]), (1, 2, 1, 96, 16, 256, [300], None),
    (2, 4, 1, 80, 64, 64, [64, 191], [64, 63]), (1, 8, 1, 128, 16, 64, [1000], None),
    (1, 1, 1, 128, 16, 1, [1], None), (1, 4, 2, 72, 16, 100, [60], None),
    (2, 8, 1, 128, 128, 200, [900, 200], None),
])
def test_attend_tree(dev, name, B, Hq, H, D, page, Q, lengths, counts):
    rng = np.random.default_rng(24)
    cache, table = make_pool(dev, lengths, H, D, page, TYPES[name], 25)
    q = queries(dev, B, Q, Hq, D, TYPES[name], 26)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    ct = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=dev)
    for loose in (False, True):
        parents = [random_tree(rng, Q, loose) for _ in range(B)]
        out, lse = ops.paged_attend(q, cache, table, n, counts=ct,
                                    parents=torch.tensor(parents, dtype=torch.int32, device=dev))
        check(q, cache, table, lengths, out, lse, parents=np.array(parents), counts=counts)
    # one tree for all sequences
    shared = torch.tensor(parents[0], dtype=torch.int32, device=dev)
    out, lse = ops.paged_attend(q, cache, table, n, counts=ct, parents=shared)
    check(q, cache, table, lengths, out, lse, parents=np.array(parents[0]), counts=counts)


def check_large(q, cache, table, lengths, out, lse, causal=False, parents=None, counts=None):
    """check on the GPU, sequence by sequence."""
    B, Q, Hq, D = q.shape
    u = ref.HALF["bf16" if q.dtype == torch.bfloat16 else "fp16"]
    pages, H, page, _ = cache.k.shape
    for b in range(B):
        n, c = lengths[b], Q if counts is None else counts[b]
        see = torch.tensor(ref.visible(Q, n, c, causal, None if parents is None else parents[b]),
                           device=q.device)
        at = table[b, :-(-n // page)].long()
        there = ((at >= 0) & (at < pages)).repeat_interleave(page)[:n]
        see &= there
        k, v = (x[at.clamp(0, pages - 1)].transpose(0, 1).reshape(H, -1, D)[:, :n].double().clone()
                for x in (cache.k, cache.v))
        unseen = ~see.any(0)
        k[:, unseen] = 0
        v[:, unseen] = 0
        qq = q[b].double()
        qq[c:] = 0
        ro, rl, ot, lt = ref.attend_gpu(qq, k, v, see, D ** -0.5, u, u)
        got, gl = out[b].double(), lse[b].double()
        assert torch.isfinite(got).all()
        assert ((got - ro).abs() <= ot).all(), (b, ((got - ro).abs() - ot).max().item())
        empty = torch.isneginf(rl)
        assert torch.equal(torch.isneginf(gl), empty)
        assert (got.transpose(0, 1)[empty] == 0).all()
        assert ((gl - rl).abs()[~empty] <= lt[~empty]).all()


# more than 2^24 (row, key) pairs in all heads, and more than 64 rows of a key head
LARGE = [
    # B, Hq, H, D, page, Q, lengths, counts
    (2, 16, 8, 128, 16, 256, [2300, 2111], None), (3, 12, 12, 64, 32, 333, [1800, 0, 2049], [333, 5, 100]),
    (1, 32, 8, 96, 128, 130, [4097], None), (2, 16, 4, 80, 16, 111, [5000, 111], [111, 60]),
    (1, 7, 1, 40, 64, 300, [9000], [300]), (4, 8, 8, 128, 64, 257, [3000, 257, 1, 2500], None),
    (1, 24, 24, 120, 16, 100, [8200], None),
]


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["whole", "causal", "tree"])
@pytest.mark.parametrize("B,Hq,H,D,page,Q,lengths,counts", LARGE)
def test_attend_many_rows(dev, name, what, B, Hq, H, D, page, Q, lengths, counts):
    if what == "tree":
        Q = min(Q, 256)
        counts = None if counts is None else [min(c, Q) for c in counts]
    rng = np.random.default_rng(100)
    cache, table = make_pool(dev, lengths, H, D, page, TYPES[name], 101)
    q = queries(dev, B, Q, Hq, D, TYPES[name], 102)
    ct = None
    if counts:
        for b, c in enumerate(counts):
            q[b, c:] = float("nan")
        ct = torch.tensor(counts, dtype=torch.int32, device=dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    parents = [random_tree(rng, Q, b % 2 == 1) for b in range(B)] if what == "tree" else None
    tree = None if parents is None else torch.tensor(parents, dtype=torch.int32, device=dev)
    out, lse = ops.paged_attend(q, cache, table, n, causal=what == "causal", parents=tree, counts=ct)
    check_large(q, cache, table, lengths, out, lse, what == "causal", parents, counts)
    # some pages are none
    for b, m in enumerate(lengths):
        if m > 4 * page:
            table[b, 1], table[b, m // page // 2], table[b, m // page - 1] = -1, 2 ** 31 - 1, cache.k.shape[0]
    out, lse = ops.paged_attend(q, cache, table, n, causal=what == "causal", parents=tree, counts=ct)
    check_large(q, cache, table, lengths, out, lse, what == "causal", parents, counts)


# more than 512 times 32 rows, more than 64 of a key head, over few keys
FEW_KEYS = [
    (40, 64, 8, 128, 16, 11, [5, 0, 1, 16] * 10, None), (3, 24, 24, 96, 64, 300, [16, 0, 37], [300, 0, 5]),
    (13, 16, 16, 72, 16, 96, [96, 130, 1, 0, 500, 97, 95, 17, 16, 15, 33, 129, 128], None),
    (1, 16, 8, 64, 32, 1100, [64], None), (33, 32, 16, 40, 1024, 40, [1] * 33, [40, 1, 0] * 11),
]


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["whole", "causal", "tree"])
@pytest.mark.parametrize("B,Hq,H,D,page,Q,lengths,counts", FEW_KEYS)
def test_attend_many_rows_over_few_keys(dev, name, what, B, Hq, H, D, page, Q, lengths, counts):
    test_attend_many_rows(dev, name, what, B, Hq, H, D, page, Q, lengths, counts)


@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["causal", "tree"])
def test_many_rows_that_are_not_seen_may_hold_anything(dev, what, name):
    rng = np.random.default_rng(103)
    dtype, n, Q, H = TYPES[name], 2200, 200, 40
    cache, table = make_pool(dev, [n], H, 128, 16, dtype, 104)
    q = queries(dev, 1, Q, H, 128, dtype, 105)
    parents = random_tree(rng, Q)
    kw = dict(causal=True) if what == "causal" else dict(
        parents=torch.tensor(parents, dtype=torch.int32, device=dev))
    clean = ops.paged_attend(q, cache, table, n, **kw)
    see = ref.visible(Q, n, Q, what == "causal", None if what == "causal" else parents)
    for x, row, value in ((cache.k, n - 2, "nan"), (cache.v, n - Q + 3, "nan"), (cache.v, n - 1, "inf"),
                          (cache.v, n - 77, "-inf")):
        p, r = ref.slots(table[0].tolist(), 16, row)
        held = x[p, :, r, 21].clone()
        x[p, :, r, 21] = float(value)
        out, lse = ops.paged_attend(q, cache, table, n, **kw)
        x[p, :, r, 21] = held
        hit = torch.tensor(see[:, row], device=dev)
        assert hit.any() and not hit.all()
        assert torch.equal(out[0, ~hit], clean[0][0, ~hit])
        assert torch.equal(lse[0][:, ~hit], clean[1][0][:, ~hit])
        if x is cache.v:
            got = out[0, hit][..., 21]
            assert (got.isnan() if value == "nan" else got == float(value)).all()
            others = torch.arange(128, device=dev) != 21
            assert torch.equal(out[0, hit][..., others], clean[0][0, hit][..., others])
            assert torch.equal(lse, clean[1])
        else:
            assert out[0, hit].isnan().all() and lse[0][:, hit].isnan().all()


@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_many_rows_of_large_scores(dev, name):
    dtype = TYPES[name]
    cache, table = make_pool(dev, [4200], 16, 128, 32, dtype, 106)
    q = queries(dev, 1, 300, 16, 128, dtype, 107, scale=30.0)
    out, lse = ops.paged_attend(q, cache, table, 4200)
    check_large(q, cache, table, [4200], out, lse)
    cache.k[..., 0] = -1.0
    q[..., 0] = 3e4
    out, lse = ops.paged_attend(q, cache, table, 4200, softmax_scale=1e5)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    for size in (16, 1 << 20):
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        fewer = ops.paged_attend(q, cache, table, 4200, softmax_scale=1e5, workspace=work)
        assert torch.isfinite(fewer[0]).all()


@pytest.mark.parametrize("Q,G", [(5, 1), (48, 2), (200, 2)])
def test_a_chain_is_the_causal_mask(dev, Q, G):
    cache, table = make_pool(dev, [333], 2, 128, 16, torch.bfloat16, 27)
    q = queries(dev, 1, Q, 2 * G, 128, torch.bfloat16, 28)
    chain = torch.arange(-1, Q - 1, dtype=torch.int32, device=dev)
    # (the sums' order may differ: key ranges are divided by what a group of rows sees)
    for kw in (dict(causal=True), dict(parents=chain)):
        out, lse = ops.paged_attend(q, cache, table, 333, **kw)
        check(q, cache, table, [333], out, lse, causal=True)


@pytest.mark.parametrize("Q,Hq", [(9, 2), (64, 4)])
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("what", ["causal", "tree"])
def test_rows_that_are_not_seen_may_hold_anything(dev, what, name, Q, Hq):
    """NaN and infinities in keys and values reach the rows that see them and no
    other."""
    rng = np.random.default_rng(29)
    dtype, n = TYPES[name], 150
    cache, table = make_pool(dev, [n], 1, 128, 16, dtype, 30)
    q = queries(dev, 1, Q, Hq, 128, dtype, 31)
    parents = random_tree(rng, Q)
    kw = dict(causal=True) if what == "causal" else dict(
        parents=torch.tensor(parents, dtype=torch.int32, device=dev))
    clean = ops.paged_attend(q, cache, table, n, **kw)
    see = ref.visible(Q, n, Q, what == "causal", None if what == "causal" else parents)
    for x, row, value in ((cache.k, n - 2, "nan"), (cache.v, n - Q + 3, "nan"), (cache.v, n - 1, "inf"),
                          (cache.v, n - Q // 2, "-inf")):
        p, r = ref.slots(table[0].tolist(), 16, row)
        held = x[p, 0, r, 5].clone()
        x[p, 0, r, 5] = float(value)
        out, lse = ops.paged_attend(q, cache, table, n, **kw)
        x[p, 0, r, 5] = held
        hit = torch.tensor(see[:, row], device=dev)
        assert hit.any() and not hit.all()
        assert torch.equal(out[0, ~hit], clean[0][0, ~hit])
        assert torch.equal(lse[0][:, ~hit], clean[1][0][:, ~hit])
        if x is cache.v:
            got = out[0, hit][..., 5]
            assert (got.isnan() if value == "nan" else got == float(value)).all()
            others = torch.arange(128, device=dev) != 5
            assert torch.equal(out[0, hit][..., others], clean[0][0, hit][..., others])
            assert torch.equal(lse, clean[1])
        else:
            assert out[0, hit].isnan().all() and lse[0][:, hit].isnan().all()


@pytest.mark.parametrize("Q", [1, 100])
def test_attend_pages_that_are_none(dev, Q):
    """Rows of table entries outside the pool are seen by no query."""
    lengths = [200, 64]
    cache, table = make_pool(dev, lengths, 2, 64, 16, torch.bfloat16, 32)
    table[0, 0], table[0, 5], table[0, 12], table[1, 1] = -1, cache.k.shape[0], 2 ** 31 - 1, -2 ** 31
    q = queries(dev, 2, Q, 4, 64, torch.bfloat16, 33)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = ops.paged_attend(q, cache, table, n)
    check(q, cache, table, lengths, out, lse)
    table[:] = -1
    out, lse = ops.paged_attend(q, cache, table, n)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_attend_lengths_are_clamped(dev):
    cache, table = make_pool(dev, [100, 100, 100], 1, 128, 16, torch.bfloat16, 34)
    q = queries(dev, 3, 1, 2, 128, torch.bfloat16, 35)
    n = torch.tensor([-5, 2 ** 31 - 1, 50], dtype=torch.int32, device=dev)
    out, lse = ops.paged_attend(q, cache, table, n, max_length=70)
    check(q, cache, table, [0, 70, 50], out, lse)
    out, lse = ops.paged_attend(q, cache, table, 0)
    assert (out == 0).all() and torch.isneginf(lse).all()


@pytest.mark.parametrize("Q", [1, 40, 300])
@pytest.mark.parametrize("name", ["bf16", "fp16"])
def test_attend_large_scores(dev, name, Q):
    """Peaked softmax: maxima that move late, weights that vanish; and scores near the
    type's ends."""
    dtype = TYPES[name]
    cache, table = make_pool(dev, [700], 1, 128, 32, dtype, 36)
    q = queries(dev, 1, Q, 2, 128, dtype, 37, scale=30.0)
    out, lse = ops.paged_attend(q, cache, table, 700)
    check(q, cache, table, [700], out, lse)
    out, lse = ops.paged_attend(q, cache, table, 700, softmax_scale=1e-30)
    check(q, cache, table, [700], out, lse, scale=1e-30)
    # all scores far below zero: the first maximum is any number
    low = cache.k.clone()
    low[..., 0] = -1.0
    far = ops.PagedCache(low, cache.v)
    q[..., 0] = 3e4
    out, lse = ops.paged_attend(q, far, table, 700, softmax_scale=1e5)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("Q,lengths", [(1, [3000, 2500]), (150, [900, 800])])
def test_attend_with_less_workspace_and_over_q(dev, Q, lengths):
    cache, table = make_pool(dev, lengths, 1, 128, 16, torch.bfloat16, 38)
    q = queries(dev, 2, Q, 2, 128, torch.bfloat16, 39)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    for size in (16, 5000, 40000, 1 << 22):
        work = torch.empty(size, dtype=torch.uint8, device=dev)
        out, lse = ops.paged_attend(q, cache, table, n, workspace=work)
        check(q, cache, table, lengths, out, lse)
    whole = ops.paged_attend(q, cache, table, n)[0]
    # rows with gaps between them, in another order, and over q itself
    wide = torch.full((2, 2, Q, 144), 7.0, device=dev, dtype=torch.bfloat16)
    view = wide[..., :128].transpose(1, 2)
    ops.paged_attend(q, cache, table, n, out=view)
    assert torch.equal(view, whole) and (wide[..., 128:] == 7).all()
    mine = q.clone()
    assert ops.paged_attend(mine, cache, table, n, out=mine)[0] is mine
    assert torch.equal(mine, whole)
    strided = torch.empty((2, Q, 4, 136), device=dev, dtype=torch.bfloat16)[:, :, ::2, :128]
    strided.copy_(q)
    assert torch.equal(ops.paged_attend(strided, cache, table, n)[0], whole)


def test_offsets_past_32_bits(dev):
    """Pages whose elements lie past 2^32 of the pool."""
    pages, H, page, D = 34000, 8, 128, 128
    k, v = (torch.empty((pages, H, page, D), device=dev, dtype=torch.bfloat16) for _ in range(2))
    cache = ops.PagedCache(k, v)
    table = torch.tensor([[33999, 0, 16500], [1, 33001, 2]], dtype=torch.int32, device=dev)
    small, near = make_pool(dev, [300, 300], H, D, page, torch.bfloat16, 40)
    for b in range(2):
        for i in range(3):
            for x, y in ((k, small.k), (v, small.v)):
                x[table[b, i]] = y[near[b, i]]
    for Q in (1, 80):
        q = queries(dev, 2, Q, 16, D, torch.bfloat16, 41)
        a = ops.paged_attend(q, cache, table, 300, causal=True)
        b = ops.paged_attend(q, small, near, 300, causal=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    new = queries(dev, 2, 4, H, D, torch.bfloat16, 42)
    ops.paged_append(cache, table, new, new, 298)
    assert torch.equal(k[16500, :, 42:46], new[0].transpose(0, 1))
    rows = torch.tensor([[3, 1], [2, 2]], dtype=torch.int32, device=dev)
    ops.paged_commit(cache, table, 298, rows)
    assert torch.equal(k[16500, :, 42], new[0, 3]) and torch.equal(v[2, :, 43], new[1, 2])


# ---------------------------------------------------------------- commit
@pytest.mark.parametrize("name", ["bf16", "fp16"])
@pytest.mark.parametrize("M,D,page,layers", [(1, 128, 16, 1), (5, 64, 16, 2), (16, 80, 32, 3), (17, 128, 16, 1),
                                             (64, 8, 16, 1), (65, 96, 16, 1), (256, 128, 64, 2), (3, 128, 16, 70)])
def test_commit_moves_rows(dev, name, M, D, page, layers):
    """Any order, the same row twice, rows past the table, counts of their own."""
    rng = np.random.default_rng(43)
    B, H, T = 4, 3, 2 * M + 3
    starts = [0, 5, page, 40]
    caches, table = [], None
    for i in range(layers):
        cache, table = make_pool(dev, [s + T for s in starts], H, D, page, TYPES[name], 44)
        for x in (cache.k, cache.v):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(45 + i)))
        caches.append(cache)
    rows = rng.integers(0, T, (B, M)).astype(np.int32)
    rows[1] = np.sort(rng.choice(T, M, replace=False))          # as a draft's path
    if M > 1:
        rows[2, 1], rows[3, 0] = -1, 2 ** 31 - 1
    table[3, -1] = -1
    counts = [M, max(0, M - 1), M + 7, M // 2]
    tab = table.cpu().numpy()
    want = [[ref.commit(bits(x), tab, starts, rows.astype(np.int64), [min(c, M) for c in counts])
             for x in (c.k, c.v)] for c in caches]
    st, ct, rw = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (starts, counts, rows))
    length = ops.paged_commit(caches, table, st, rw, ct)
    assert length.tolist() == [s + min(c, M) for s, c in zip(starts, counts)]
    for c, (k, v) in zip(caches, want):
        assert np.array_equal(bits(c.k), k) and np.array_equal(bits(c.v), v)


def test_commit_of_one_cache_and_of_nothing(dev):
    cache, table = make_pool(dev, [40], 1, 64, 16, torch.bfloat16, 46)
    before = bits(cache.k)
    none = torch.empty((1, 0), dtype=torch.int32, device=dev)
    assert ops.paged_commit(cache, table, 30, none).tolist() == [30]
    same = torch.arange(4, dtype=torch.int32, device=dev)[None]
    assert ops.paged_commit(cache, table, 30, same).tolist() == [34]
    assert np.array_equal(bits(cache.k), before)


# ---------------------------------------------------------------- together
def test_a_run_of_drafts(dev):
    """Prompts, then steps of: draft a tree, append it at its depths' positions, attend
    it, commit a path; the cache is what a token-by-token run leaves, and each
    token's attention that of the run."""
    B, H, Hq, D, page, T = 2, 2, 4, 128, 16, 12
    rng = np.random.default_rng(50)
    freqs = freqs_of(D, dev)
    prompts = [37, 20]
    pages = 16
    order = torch.randperm(2 * pages, generator=torch.Generator().manual_seed(51)).to(torch.int32)
    table = order.view(B, pages).to(dev)
    nan = lambda: torch.full((2 * pages, H, page, D), float("nan"), device=dev, dtype=torch.bfloat16)
    cache, plain = ops.PagedCache(nan(), nan()), ops.PagedCache(nan(), nan())
    g = torch.Generator().manual_seed(52)
    make = lambda n, h: torch.randn((B, n, h, D), generator=g).bfloat16().to(dev)
    k, v, q = make(37, H), make(37, H), make(37, Hq)
    counts = torch.tensor(prompts, dtype=torch.int32, device=dev)
    zero = torch.zeros(B, dtype=torch.int32, device=dev)
    for c in (cache, plain):
        turned = ops.paged_append(c, table, k, v, zero, counts=counts, q=q, freqs=freqs)
        out, lse = ops.paged_attend(turned, c, table, counts, causal=True, counts=counts)
        check(turned, c, table, prompts, out, lse, causal=True, counts=prompts)
    length = counts
    for step in range(4):
        parents = [random_tree(rng, T) for _ in range(B)]
        depth = [[0] * T for _ in range(B)]
        paths = []
        for b in range(B):
            for t in range(1, T):
                depth[b][t] = depth[b][parents[b][t]] + 1
            path = [int(rng.integers(0, T))]
            while parents[b][path[0]] >= 0:
                path.insert(0, parents[b][path[0]])
            paths.append(path)
        k, v, q = make(T, H), make(T, H), make(T, Hq)
        tree = torch.tensor(parents, dtype=torch.int32, device=dev)
        at = length[:, None] + torch.tensor(depth, dtype=torch.int32, device=dev)
        turned = ops.paged_append(cache, table, k, v, length, q=q, freqs=freqs, positions=at)
        out, lse = ops.paged_attend(turned, cache, table, length + T, parents=tree, max_length=256)
        check(turned, cache, table, (length + T).tolist(), out, lse, parents=np.array(parents))
        rows = torch.zeros((B, T), dtype=torch.int32, device=dev)
        kept = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=dev)
        for b, p in enumerate(paths):
            rows[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
        # the accepted tokens one after the other, without drafts
        for j in range(max(map(len, paths))):
            pick = [p[min(j, len(p) - 1)] for p in paths]
            one = lambda x: torch.stack([x[b, pick[b]] for b in range(B)])[:, None]
            n = torch.tensor([1 if j < len(p) else 0 for p in paths], dtype=torch.int32, device=dev)
            tq = ops.paged_append(plain, table, one(k), one(v), length + j, counts=n, q=one(q), freqs=freqs)
            o, z = ops.paged_attend(tq, plain, table, length + j + 1, counts=n)
            check(tq, plain, table, (length + j + 1).tolist(), o, z, counts=n.tolist())
            for b in range(B):
                if j < len(paths[b]):
                    assert torch.equal(tq[b, 0], turned[b, pick[b]])
                    # two sums of the same weights, each within its bound
                    assert (o[b, 0].float() - out[b, pick[b]].float()).abs().max() <= 2.0 ** -6
        length = ops.paged_commit(cache, table, length, rows, kept)
        for b, n in enumerate(length.tolist()):
            for r in range(n):
                p, i = ref.slots(table[b].tolist(), page, r)
                assert torch.equal(cache.k[p, :, i], plain.k[p, :, i])
                assert torch.equal(cache.v[p, :, i], plain.v[p, :, i])


def test_graph_of_a_decoding_step(dev):
    """Append and attention captured once and replayed with other rows, positions and
    lengths, eager work between the replays."""
    B, H, Hq, D, page = 3, 2, 8, 128, 16
    lengths = [40, 7, 200]
    cache, table = make_pool(dev, [n + 8 for n in lengths], H, D, page, torch.bfloat16, 60)
    freqs = freqs_of(D, dev)
    length = torch.tensor(lengths, dtype=torch.int32, device=dev)
    k, v, q = (torch.zeros((B, 1, h, D), device=dev, dtype=torch.bfloat16) for h in (H, H, Hq))
    turned, out = torch.empty_like(q), torch.empty_like(q)

    def step():
        ops.paged_append(cache, table, k, v, length, q=q, q_out=turned, freqs=freqs)
        return ops.paged_attend(turned, cache, table, length + 1, out=out)[1]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lse = step()
    for i in range(5):
        for x, s in ((k, 61), (v, 71), (q, 81)):
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(s + i)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        check(turned, cache, table, [n + 1 for n in lengths], *got)
        eager = ops.paged_attend(turned, cache, table, length + 1)
        assert torch.equal(eager[0], got[0]) and torch.equal(eager[1], got[1])
        length += 1
        lengths = [n + 1 for n in lengths]


def test_calls_on_a_stream_of_their_own(dev):
    lengths = [500, 100]
    cache, table = make_pool(dev, lengths, 2, 128, 16, torch.bfloat16, 90)
    q = queries(dev, 2, 3, 4, 128, torch.bfloat16, 91)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    want = ops.paged_attend(q, cache, table, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.paged_attend(q, cache, table, n))
    torch.cuda.synchronize()
    for o, z in got:
        assert torch.equal(o, want[0]) and torch.equal(z, want[1])
