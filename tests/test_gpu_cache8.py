"""The 8-bit cache on the GPU: codes, scales and evicted rows to the last bit,
attention and received weight against 64 bits with derived bounds."""
import numpy as np
import pytest
import torch

from tests import _cache8_ref as ref
from nanokv_amd import ops

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
FORMATS = ["int8", "e4m3"]


def raw(t):
    """Codes as numpy: int8, or the bytes of e4m3."""
    return (t if t.dtype == torch.int8 else t.view(torch.uint8)).cpu().numpy()


def make_cache(dev, B, H, cap, D, fmt, seed, lengths=None):
    """A cache whose written rows are random and whose rows past the lengths,
    and scales of blocks past them, are hostile: NaN codes, NaN scales."""
    g = torch.Generator().manual_seed(seed)
    cache = ops.Cache8.empty(B, H, cap, D, dev, fmt)
    cap = cache.cap
    x = torch.randn((2, B, H, cap, D), generator=g)
    x *= torch.exp(0.5 * torch.randn((2, B, H, cap // 64, 1, 1), generator=g)).expand(
        2, B, H, cap // 64, 64, 1).reshape(2, B, H, cap, 1)
    for i, (codes, scale) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        s = x[i].view(B, H, cap // 64, -1).abs().amax(-1) / float(ref.TOP[fmt])
        y = ref.to_codes((x[i] / s.repeat_interleave(64, 2)[..., None]).numpy(), fmt)
        w = np.zeros((B, H, cap, ref.pitch(D)), y.dtype)
        w[..., :D] = y
        for b, n in enumerate(lengths or [cap] * B):
            w[b, :, n:] = 0x7F if fmt == "e4m3" else 127
            s[b, :, -(-n // 64):] = float("nan")
        view = codes if fmt == "int8" else codes.view(torch.uint8)
        view.copy_(torch.from_numpy(w))
        scale.copy_(s)
    return cache


def cache_values(cache, fmt):
    return [np.nan_to_num(ref.dequant(raw(c), s.cpu().numpy(), fmt, cache.head_dim))
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


def check_attend(q, cache, fmt, lengths, causal, out, lse, scale=None):
    D = q.shape[3]
    k, v = cache_values(cache, fmt)
    scale = D ** -0.5 if scale is None else scale
    ro, rl, otol, ltol = ref.attend(q.double().cpu().numpy(), k, v, lengths, causal, scale,
                                    HALF[q.dtype])
    got, gl = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.isfinite(got).all()
    assert (np.abs(got - ro) <= otol).all(), np.max(np.abs(got - ro) - otol)
    empty = np.isneginf(rl)
    assert np.array_equal(np.isneginf(gl), empty)
    assert (got.transpose(0, 2, 1, 3)[empty] == 0).all()
    assert (np.abs(gl[~empty] - rl[~empty]) <= ltol[~empty]).all()
    return gl


# ---------------------------------------------------------------- write
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,start,D", [(1, 0, 128), (1, 63, 64), (1, 64, 128), (65, 100, 80),
                                       (64, 64, 8), (200, 1, 128), (2, 63, 40)])
def test_write_codes_and_scales(dev, fmt, dtype, T, start, D):
    B, H, cap = 2, 3, 320
    cache = make_cache(dev, B, H, cap, D, fmt, 1)
    g = torch.Generator().manual_seed(2)
    kv = (torch.randn((B, T, 2, H, D), generator=g)
          * torch.exp(torch.randn((B, T, 2, 1, 1), generator=g))).to(dtype).to(dev)
    k, v = kv.unbind(2)
    before = [raw(cache.k).copy(), raw(cache.v).copy(), cache.k_scale.cpu().numpy(),
              cache.v_scale.cpu().numpy()]
    ops.cache8_write(cache, k, v, start)
    for codes, scale, c0, s0, x in ((cache.k, cache.k_scale, before[0], before[2], k),
                                    (cache.v, cache.v_scale, before[1], before[3], v)):
        rc, rs = ref.write(c0, s0, x.float().cpu().numpy(), [start] * B, [T] * B, fmt)
        assert np.array_equal(scale.cpu().numpy(), rs)
        assert np.array_equal(raw(codes), rc)


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_ragged_starts_counts_and_the_end_of_the_cache(dev, fmt):
    B, H, cap, D, T = 6, 2, 192, 64, 100
    cache = make_cache(dev, B, H, cap, D, fmt, 3)
    x = torch.randn((2, B, T, H, D), generator=torch.Generator().manual_seed(4)).to(dev)
    start, counts = [0, 5, 150, 191, 192, -7], [100, 0, 100, 3, 100, 101]
    before = [raw(cache.k).copy(), cache.k_scale.cpu().numpy()]
    st = torch.tensor(start, dtype=torch.int32, device=dev)
    ct = torch.tensor(counts, dtype=torch.int32, device=dev)
    ops.cache8_write(cache, x[0], x[1], st, ct)
    rc, rs = ref.write(*before, x[0].cpu().numpy(), start, counts, fmt)
    assert np.array_equal(cache.k_scale.cpu().numpy(), rs)
    assert np.array_equal(raw(cache.k), rc)


@pytest.mark.parametrize("fmt", FORMATS)
def test_write_special_values(dev, fmt):
    """Infinities, NaN, zeros, the type's extremes: codes and scales stay finite
    and the finite values set the scale."""
    cache = ops.Cache8.empty(1, 1, 256, 64, dev, fmt)
    x = torch.randn((1, 256, 1, 64), generator=torch.Generator().manual_seed(5))
    x[0, 0:64] = 0
    x[0, 64, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 3.0])
    x[0, 130, 0, 0] = torch.finfo(torch.float32).max
    x[0, 192:] = float("nan")
    x = x.to(dev)
    before = raw(cache.k).copy(), cache.k_scale.cpu().numpy()
    ops.cache8_write(cache, x, x, 0)
    rc, rs = ref.write(*before, x.cpu().numpy(), [0], [256], fmt)
    assert np.isfinite(rs).all() and np.array_equal(cache.k_scale.cpu().numpy(), rs)
    assert np.array_equal(raw(cache.k), rc) and np.array_equal(raw(cache.v), rc)
    assert np.isfinite(ref.values(rc, fmt)).all()


def test_write_token_by_token_equals_its_plain_form(dev):
    """A block filled a token at a time: every growth of its scale."""
    B, H, D, n = 2, 2, 128, 130
    cache = ops.Cache8.empty(B, H, n, D, dev, "int8")
    x = torch.randn((B, n, H, D), generator=torch.Generator().manual_seed(6))
    x *= torch.linspace(0.1, 3, n)[None, :, None, None]
    x = x.bfloat16().to(dev)
    rc, rs = raw(cache.k).copy(), cache.k_scale.cpu().numpy()
    at = torch.zeros(B, dtype=torch.int32, device=dev)
    for t in range(n):
        ops.cache8_write(cache, x[:, t:t + 1], x[:, t:t + 1], at)
        at += 1
        rc, rs = ref.write(rc, rs, x[:, t:t + 1].float().cpu().numpy(), [t] * B, [1] * B, "int8")
    assert np.array_equal(cache.k_scale.cpu().numpy(), rs)
    assert np.array_equal(raw(cache.k), rc)


# ---------------------------------------------------------------- attend
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G,D,Q,lengths,causal", [
    (2, 1, 128, 1, [0, 1, 63, 64, 65, 200], False),
    (1, 8, 128, 1, [1000, 129], False),
    (2, 3, 64, 1, [511, 0, 64], False),
    (1, 4, 80, 5, [77, 3], True),        # the second: two queries see nothing
    (2, 1, 8, 17, [130], True),
    (1, 2, 40, 33, [65, 64, 1], False),
    (3, 1, 128, 70, [150], True),
    (1, 1, 64, 130, [40, 200], True),
    (2, 4, 128, 100, [700, 90], True),
    (1, 1, 128, 300, [1900], False),
    (1, 5, 96, 33, [64, 63, 0], False),
    (2, 1, 24, 257, [300, 512], True),
    (1, 1, 64, 1000, [3000], True),
])
def test_attend(dev, fmt, dtype, H, G, D, Q, lengths, causal):
    B = len(lengths)
    cache = make_cache(dev, B, H, max(max(lengths), 1), D, fmt, 7, lengths)
    q = torch.randn((B, Q, H * G, D), generator=torch.Generator().manual_seed(8)) * 2
    q = q.to(dtype).to(dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = ops.cache8_attend(q, cache, n, max_length=max(lengths), causal=causal)
    gl = check_attend(q, cache, fmt, lengths, causal, out, lse)
    # the weight each key received, on the kernel's own lse
    k, _ = cache_values(cache, fmt)
    m0 = torch.rand((B, H, cache.cap), generator=torch.Generator().manual_seed(9))
    rm, tol = ref.mass(q.double().cpu().numpy(), k, gl, m0.numpy(), lengths, causal, D ** -0.5)
    m = m0.to(dev)
    other = torch.full_like(m, float("nan"))
    ops.cache8_mass(q, cache, lse, m, n, out=other, max_length=max(lengths), causal=causal)
    got = ops.cache8_mass(q, cache, lse, m, n, max_length=max(lengths), causal=causal)
    assert got is m and torch.equal(m, other)
    assert (np.abs(m.double().cpu().numpy() - rm) <= tol).all()


@pytest.mark.parametrize("H,G,Q,N", [(1, 1, 1, 20000), (1, 16, 1, 8191), (2, 2, 3, 5000),
                                     (1, 1, 40, 4097), (1, 2, 90, 9001),
                                     (8, 1, 33, 16500), (2, 4, 16, 65537)])
def test_attend_long(dev, H, G, Q, N):
    """Key splits and their merge."""
    cache = make_cache(dev, 1, H, N, 128, "int8", 10, [N])
    q = torch.randn((1, Q, H * G, 128), generator=torch.Generator().manual_seed(11)) * 1.5
    q = q.bfloat16().to(dev)
    out, lse = ops.cache8_attend(q, cache, N)
    check_attend(q, cache, "int8", [N], False, out, lse)


def test_attend_strides_scale_and_preallocated(dev):
    B, Q, Hq, D, N = 2, 9, 4, 64, 100
    cache = make_cache(dev, B, 2, 128, D, "e4m3", 12, [N, N])
    big = torch.randn((B, Hq, Q, 3 * D), generator=torch.Generator().manual_seed(13))
    big = big.bfloat16().to(dev)
    q = big[..., D:2 * D].transpose(1, 2)
    out = torch.full((B, Hq, Q, D), 7.0, dtype=torch.bfloat16, device=dev).transpose(1, 2)
    got, lse = ops.cache8_attend(q, cache, N, softmax_scale=0.25, out=out)
    assert got is out
    check_attend(q, cache, "e4m3", [N, N], False, out, lse, 0.25)
    again, none = ops.cache8_attend(q, cache, N, softmax_scale=0.25, return_lse=False)
    assert none is None and torch.equal(again, out)


def test_attend_uneven_scales(dev):
    """Blocks whose scales differ by many powers of two, zero blocks among them."""
    for dtype in (torch.bfloat16, torch.float16):
        cache = make_cache(dev, 1, 1, 512, 64, "int8", 14)
        f = torch.tensor([1.0, 2.0 ** -12, 2.0 ** 10, 1e-3, 1.0, 2.0 ** 5, 3.0, 1.0], device=dev)
        cache.v_scale.mul_(f)
        cache.v[:, :, 64:128] = 0
        cache.v_scale[:, :, 1] = float(ref.TINY) / 127
        cache.k[:, :, 256:320] = 0
        cache.k_scale[:, :, 4] = float(ref.TINY) / 127
        q = torch.randn((1, 20, 1, 64), generator=torch.Generator().manual_seed(15)).to(dtype)
        out, lse = ops.cache8_attend(q.to(dev), cache, 512)
        check_attend(q, cache, "int8", [512], False, out, lse)


def test_offsets_past_32_bits(dev):
    """The last head of a cache whose codes take more than 2^32 bytes."""
    H, cap, D, N = 17, 1 << 21, 128, 70
    cache = ops.Cache8.empty(1, H, cap, D, dev, "int8")
    g = torch.Generator().manual_seed(16)
    x = torch.randn((1, N, H, D), generator=g).bfloat16().to(dev)
    start = cap - 2 * N
    ops.cache8_write(cache, x, x.flip(1), start)
    codes, scale = ref.write(np.zeros((1, 1, 192, 128), np.int8), np.ones((1, 1, 3), np.float32),
                             x[:, :, -1:].float().cpu().numpy(), [start % 64], [N], "int8")
    first = start // 64 * 64
    assert np.array_equal(raw(cache.k[:, -1:, first:first + 128]), codes[:, :, :128])
    assert np.array_equal(cache.k_scale[:, -1:, first // 64:first // 64 + 2].cpu().numpy(),
                          scale[:, :, :2])
    # 2,097,012 zero keys and the 70 written ones: zero keys score 0
    q = (torch.randn((1, 1, H, D), generator=g) * 4).bfloat16().to(dev)
    out, lse = ops.cache8_attend(q, cache, start + N)
    k, v = (ref.dequant(raw(c[:, -1:, first:]), s[:, -1:, first // 64:].cpu().numpy(), "int8", D)
            [0, 0, start - first:start - first + N]
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    z = k @ q[0, 0, -1].double().cpu().numpy() * D ** -0.5
    p = np.exp(z)
    tot = p.sum() + start
    assert abs(float(lse[0, -1, 0]) - np.log(tot)) < 1e-4
    want = p @ v / tot
    # the weights are off by half a step of fp16, the output by one of bf16
    tol = 2.0 ** -8 * (p @ np.abs(v) / tot + np.abs(want)) * 1.01 + 1e-9
    assert (np.abs(out[0, 0, -1].double().cpu().numpy() - want) <= tol).all()


# ---------------------------------------------------------------- evict
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lengths,keep,sink,recent,D", [
    ([200, 100, 64, 1, 0], 100, 3, 10, 64), ([2000, 1500], 777, 0, 0, 128),
    ([130], 1, 0, 0, 80), ([130], 1, 1, 0, 8), ([130], 64, 32, 32, 128), ([300, 65], 299, 0, 299, 64),
])
def test_evict(dev, fmt, lengths, keep, sink, recent, D):
    B, H = len(lengths), 3
    cache = make_cache(dev, B, H, max(lengths), D, fmt, 20, lengths)
    g = torch.Generator().manual_seed(21)
    m = torch.randint(0, 40, (B, H, cache.cap), generator=g).float() / 8      # many ties
    m[0, 0, ::7] = 0.0
    m[0, 0, 1::7] = -0.0
    m[0, 1, 5] = float("inf")
    m[0, 1, 6] = float("nan")
    m[0, 2] = 1.0
    m[:, :, -1] = 1e30
    out = make_cache(dev, B, H, keep + 70, D, fmt, 22)
    out_m = torch.full((B, H, out.cap), -1.0, device=dev)
    old = [raw(out.k).copy(), raw(out.v).copy(), out.k_scale.cpu().numpy(),
           out.v_scale.cpu().numpy()]
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    rows, left = ops.cache8_evict(cache, m.to(dev), n, out, out_m, keep=keep, sink=sink,
                                  recent=recent)
    want = ref.evict(m.numpy(), lengths, keep, sink, recent)
    assert left.tolist() == [min(x, keep) for x in lengths]
    full = np.full((B, H, keep), -1)
    wm = np.full((B, H, out.cap), -1.0, np.float32)
    for b in range(B):
        for h in range(H):
            r = want[b][h]
            full[b, h, :len(r)] = r
            wm[b, h, :len(r)] = m.numpy()[b, h, r]
    assert np.array_equal(rows.cpu().numpy(), full)
    assert np.array_equal(out_m.cpu().numpy(), wm, equal_nan=True)
    for codes, scale, oc, os_, got, gs in (
            (cache.k, cache.k_scale, old[0], old[2], out.k, out.k_scale),
            (cache.v, cache.v_scale, old[1], old[3], out.v, out.v_scale)):
        rc, rs = ref.compact(raw(codes), scale.cpu().numpy(), want, oc, os_, fmt)
        assert np.array_equal(gs.cpu().numpy(), rs)
        assert np.array_equal(raw(got), rc)


# ---------------------------------------------------------------- together
def test_decode_loop_with_eviction_and_a_codec_history(dev):
    """A prompt, tokens one by one with the weight their keys receive, an
    eviction, more tokens; each step against the plain form, and the result
    merged with an uncompressed partition as the other partitions are."""
    B, H, G, D, fmt = 2, 2, 4, 64, "e4m3"
    g = torch.Generator().manual_seed(30)
    cache = ops.Cache8.empty(B, H, 256, D, dev, fmt)
    mass = torch.zeros((B, H, cache.cap), device=dev)
    n = [150, 150]
    kv = torch.randn((2, B, 150, H, D), generator=g).bfloat16().to(dev)
    ops.cache8_write(cache, kv[0], kv[1], 0)
    dn = torch.tensor(n, dtype=torch.int32, device=dev)
    for step in range(6):
        kv = torch.randn((2, B, 1, H, D), generator=g).bfloat16().to(dev)
        ops.cache8_write(cache, kv[0], kv[1], dn)
        dn += 1
        n = [x + 1 for x in n]
        q = torch.randn((B, 1, H * G, D), generator=g).bfloat16().to(dev)
        out, lse = ops.cache8_attend(q, cache, dn)
        gl = check_attend(q, cache, fmt, n, False, out, lse)
        k, _ = cache_values(cache, fmt)
        rm, tol = ref.mass(q.double().cpu().numpy(), k, gl, mass.cpu().numpy(), n, False, D ** -0.5)
        ops.cache8_mass(q, cache, lse, mass, dn)
        assert (np.abs(mass.double().cpu().numpy() - rm) <= tol).all()
        if step == 2:
            small = ops.Cache8.empty(B, H, 128, D, dev, fmt)
            kept = torch.zeros((B, H, 128), device=dev)
            want = ref.evict(mass.cpu().numpy(), n, 100, 4, 16)
            rows, dn = ops.cache8_evict(cache, mass, dn, small, kept, keep=100, sink=4, recent=16)
            assert rows.cpu().numpy().tolist() == want
            cache, mass, n = small, kept, [100, 100]
    # merged with an uncompressed partition through the library's own merge
    kc, vc = torch.randn((2, B, 40, H * G, D), generator=g).bfloat16().to(dev)
    o2, l2 = ops.attend(q, kc, vc)
    both, bl = ops.lse_merge(out.permute(0, 2, 1, 3).contiguous(), lse,
                             o2.permute(0, 2, 1, 3).contiguous(), l2)
    want = torch.logaddexp(lse.double(), l2.double())
    wo = (torch.exp(lse.double() - want)[..., None] * out.double().permute(0, 2, 1, 3)
          + torch.exp(l2.double() - want)[..., None] * o2.double().permute(0, 2, 1, 3))
    assert (bl.double() - want).abs().max() < 1e-5
    assert (both.double() - wo).abs().max() < 2.0 ** -8 * float(wo.abs().max()) * 1.1


def test_streams_and_graph(dev):
    """Back-to-back calls on a stream of their own and a captured decoding step,
    replayed with new tokens and eager work between, equal one-at-a-time calls."""
    B, H, G, D = 3, 2, 2, 128
    g = torch.Generator().manual_seed(40)
    new = torch.randn((5, 3, B, 1, H * G, D), generator=g).bfloat16().to(dev)

    def fresh():
        c = ops.Cache8.empty(B, H, 256, D, dev, "int8")
        x = torch.randn((2, B, 100, H, D), generator=torch.Generator().manual_seed(41))
        x = x.bfloat16().to(dev)
        ops.cache8_write(c, x[0], x[1], 0)
        return c, torch.tensor([100, 60, 0], dtype=torch.int32, device=dev), \
            torch.zeros((B, H, c.cap), device=dev)

    def step(c, n, m, q, k, v):
        ops.cache8_write(c, k[:, :, :H], v[:, :, :H], n)
        n += 1
        out, lse = ops.cache8_attend(q, c, n)
        ops.cache8_mass(q, c, lse, m, n)
        return out, lse

    state = fresh()
    want = []
    for i in range(5):
        o, l = step(*state, *new[i])
        torch.cuda.synchronize()
        want.append((o.clone(), l.clone()))
    side = torch.cuda.Stream()
    s2 = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(*s2, *new[i]) for i in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(s2[2], state[2]) and torch.equal(s2[0].k, state[0].k)
    s3 = fresh()
    box = new[0].clone()
    warm = fresh()
    with torch.cuda.stream(side):
        step(*warm, *box)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step(*s3, *box)
    for i in range(5):
        box.copy_(new[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])
        step(*warm, *new[i])                   # eager work between replays
    assert torch.equal(s3[2], state[2]) and torch.equal(s3[0].v, state[0].v)


# ---------------------------------------------------------------- what callers may do
@pytest.mark.parametrize("Q,G", [(1, 2), (20, 2), (100, 2)])
def test_attend_lengths_outside_the_bound(dev, Q, G):
    """Lengths below zero are none, above max_length the bound."""
    cache = make_cache(dev, 3, 2, 192, 64, "e4m3", 50, [100, 100, 100])
    q = torch.randn((3, Q, 2 * G, 64), generator=torch.Generator().manual_seed(51)).bfloat16().to(dev)
    n = torch.tensor([-5, 10_000, 70], dtype=torch.int32, device=dev)
    out, lse = ops.cache8_attend(q, cache, n, max_length=100)
    gl = check_attend(q, cache, "e4m3", [0, 100, 70], False, out, lse)
    assert np.isneginf(gl[0]).all()
    m = torch.zeros((3, 2, cache.cap), device=dev)
    ops.cache8_mass(q, cache, lse, m, n, max_length=100)
    assert (m[0] == 0).all() and (m[:, :, 100:] == 0).all() and (m[2, :, 70:] == 0).all()
    # every query gives a weight of one: the sums of fp32 sums, a few steps off
    want = torch.tensor([0.0, Q * G, Q * G], device=dev)[:, None].expand(3, 2)
    assert ((m.sum(2) - want).abs() <= 1e-4 * Q * G).all()


@pytest.mark.parametrize("Q", [1, 40, 200])
def test_attend_a_nan_query_spoils_its_own_row_alone(dev, Q):
    cache = make_cache(dev, 1, 2, 700, 128, "int8", 52, [700])
    q = torch.randn((1, Q, 4, 128), generator=torch.Generator().manual_seed(53)).bfloat16().to(dev)
    clean, lse = ops.cache8_attend(q, cache, 700)
    bad = q.clone()
    bad[0, Q // 2, 1, 5] = float("nan")
    out, l2 = ops.cache8_attend(bad, cache, 700)
    assert torch.isnan(out[0, Q // 2, 1]).all() and torch.isnan(l2[0, 1, Q // 2])
    keep = torch.ones((Q, 4), dtype=torch.bool, device=dev)
    keep[Q // 2, 1] = False
    assert torch.equal(out[0][keep], clean[0][keep])
    assert torch.equal(l2[0].T[keep], lse[0].T[keep])


@pytest.mark.parametrize("Q", [1, 50, 130])
def test_attend_into_the_queries_and_in_a_given_workspace(dev, Q):
    cache = make_cache(dev, 1, 1, 9000, 128, "int8", 54, [9000])
    q = torch.randn((1, Q, 3, 128), generator=torch.Generator().manual_seed(55)).bfloat16().to(dev)
    want, lse = ops.cache8_attend(q, cache, 9000)
    same = q.clone()
    work = torch.full((1 << 24,), 0xFF, dtype=torch.uint8, device=dev)
    got, l2 = ops.cache8_attend(same, cache, 9000, out=same, workspace=work)
    assert got is same and torch.equal(got, want) and torch.equal(l2, lse)
    # less workspace: fewer splits, the same attention within its bound, and
    # nothing written past its end
    for nbytes in (16, 20_000 * Q // 16 * 16):
        work = torch.full((nbytes + 4096,), 0xAB, dtype=torch.uint8, device=dev)
        less, l3 = ops.cache8_attend(q, cache, 9000, workspace=work[:nbytes])
        check_attend(q, cache, "int8", [9000], False, less, l3)
        assert (work[nbytes:] == 0xAB).all()


def test_mass_row_splits_and_their_join(dev):
    """Few blocks of keys and many rows, a hostile workspace, another output."""
    cache = make_cache(dev, 2, 1, 200, 64, "e4m3", 56, [200, 77])
    q = torch.randn((2, 600, 3, 64), generator=torch.Generator().manual_seed(57)).half().to(dev)
    n = torch.tensor([200, 77], dtype=torch.int32, device=dev)
    _, lse = ops.cache8_attend(q, cache, n, causal=True)
    m0 = torch.rand((2, 1, cache.cap), generator=torch.Generator().manual_seed(58))
    k, _ = cache_values(cache, "e4m3")
    rm, tol = ref.mass(q.double().cpu().numpy(), k, lse.double().cpu().numpy(), m0.numpy(),
                       [200, 77], True, 0.125)
    work = torch.full((1 << 20,), 0xFF, dtype=torch.uint8, device=dev)
    m, out = m0.to(dev), torch.full((2, 1, cache.cap), float("nan"), device=dev)
    ops.cache8_mass(q, cache, lse, m, n, out=out, causal=True, workspace=work)
    assert torch.equal(m.cpu(), m0)
    assert (np.abs(out.double().cpu().numpy() - rm) <= tol).all()
    ops.cache8_mass(q, cache, lse, m, n, causal=True)
    assert torch.equal(m, out)
    # a workspace for two splits, and for none
    for nbytes in (2 * 2 * cache.cap * 4, 16):
        work = torch.full((nbytes + 4096,), 0xAB, dtype=torch.uint8, device=dev)
        ops.cache8_mass(q, cache, lse, m0.to(dev), n, out=out, causal=True, workspace=work[:nbytes])
        assert (np.abs(out.double().cpu().numpy() - rm) <= tol).all()
        assert (work[nbytes:] == 0xAB).all()


@pytest.mark.parametrize("Q,causal", [(1, False), (9, True)])
def test_mass_of_several_blocks_a_wave(dev, Q, causal):
    """Enough blocks that a wave takes more than one, ragged lengths, both outputs."""
    B, H, G, N = 6, 24, 2, 4100
    lengths = [4100, 1, 0, 2049, 64, 3000]
    cache = make_cache(dev, B, H, N, 64, "int8", 63, lengths)
    q = torch.randn((B, Q, H * G, 64), generator=torch.Generator().manual_seed(64)).bfloat16().to(dev)
    n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out, lse = ops.cache8_attend(q, cache, n, max_length=N, causal=causal)
    gl = check_attend(q, cache, "int8", lengths, causal, out, lse)
    k, _ = cache_values(cache, "int8")
    m0 = torch.rand((B, H, cache.cap), generator=torch.Generator().manual_seed(65))
    rm, tol = ref.mass(q.double().cpu().numpy(), k, gl, m0.numpy(), lengths, causal, 0.125)
    m, other = m0.to(dev), torch.full((B, H, cache.cap), float("nan"), device=dev)
    ops.cache8_mass(q, cache, lse, m, n, out=other, max_length=N, causal=causal)
    assert torch.equal(m.cpu(), m0)
    ops.cache8_mass(q, cache, lse, m, n, max_length=N, causal=causal)
    assert torch.equal(m, other)
    assert (np.abs(m.double().cpu().numpy() - rm) <= tol).all()


def test_evict_long_heads(dev):
    """Heads whose keys do not fit the selection's LDS, equal masses among them."""
    n, keep, H = 40_000, 9_001, 3
    cache = make_cache(dev, 1, H, n, 8, "int8", 59, [n])
    m = torch.rand((1, H, cache.cap), generator=torch.Generator().manual_seed(60))
    m[0, 1] = 0.25
    m[0, 2] = (m[0, 2] * 50).floor()
    out = ops.Cache8.empty(1, H, keep, 8, dev, "int8")
    out_m = torch.zeros((1, H, out.cap), device=dev)
    old = raw(out.k).copy(), out.k_scale.cpu().numpy()
    rows, left = ops.cache8_evict(cache, m.to(dev), n, out, out_m, keep=keep, sink=7, recent=100)
    want = ref.evict(m.numpy(), [n], keep, 7, 100)
    assert left.tolist() == [keep] and rows[0].tolist() == want[0]
    rc, rs = ref.compact(raw(cache.k), cache.k_scale.cpu().numpy(), want, *old, "int8")
    assert np.array_equal(out.k_scale.cpu().numpy(), rs) and np.array_equal(raw(out.k), rc)


@pytest.mark.parametrize("n,lengths,keep,sink,recent", [
    (33_000, [33_000, 32_769, 8_193, 100, 0], 100, 3, 20),       # parts that end inside, or never start
    (40_000, [40_000, 24_576, 9_000], 9_000, 8_193, 300),        # the first rows pass a part
    (70_000, [70_000, 65_537], 30_000, 10, 20_000),              # so do the last ones
    (70_000, [70_000], 500, 200, 300),                           # none to choose
    (70_000, [70_000, 69_999], 69_998, 0, 0),                    # one or two go
    (600_001, [600_001], 150_000, 1, 1),                         # parts of more than one step
])
def test_evict_in_parts(dev, n, lengths, keep, sink, recent):
    """Heads longer than one workgroup takes: rows, lengths and masses equal the
    plain form's, nothing behind the workspace is written, and a captured call
    replayed with new masses gives what an eager one gives."""
    B, H = len(lengths), 4
    cache = ops.Cache8.empty(B, H, n, 8, dev, "e4m3")
    g = torch.Generator().manual_seed(81)
    m = torch.rand((B, H, cache.cap), generator=g)
    m[:, 1] = (m[:, 1] * 7).floor() - 3             # equal masses in every part, zero of both signs
    m[:, 1, ::2] = -m[:, 1, ::2]
    m[:, 2] = 0.25
    m[:, 2, 5::4096] = float("nan")
    m[:, 2, 9::1000] = float("-inf")
    m[:, 3, 11::777] = float("inf")
    device_n = torch.tensor(lengths, dtype=torch.int32, device=dev)
    out = ops.Cache8.empty(B, H, keep, 8, dev, "e4m3")
    out_m = torch.full((B, H, out.cap), -7.0, device=dev)
    parts = -(-n // (8192 if n < 64 * 8192 else -(-n // 64 // 4096) * 4096))
    need = B * H * parts * (2 * 2048 * 4 + 16)
    work = torch.full((need + 4096,), 0x5a, dtype=torch.uint8, device=dev)
    md = m.to(dev)

    def call(**kw):
        return ops.cache8_evict(cache, md, device_n, out, out_m, keep=keep, sink=sink,
                                recent=recent, max_length=n, **kw)

    with pytest.raises(RuntimeError, match="workspace"):
        call(workspace=work[:need - 16])
    rows, left = call(workspace=work[:need])
    want = ref.evict(m.numpy(), lengths, keep, sink, recent)
    assert left.tolist() == [min(x, keep) for x in lengths]
    rows, kept = rows.cpu().numpy(), out_m.cpu().numpy()
    for b in range(B):
        for h in range(H):
            w = np.asarray(want[b][h], np.int64)
            assert np.array_equal(rows[b, h, :len(w)], w), (b, h)
            assert (rows[b, h, len(w):] == -1).all()
            assert np.array_equal(kept[b, h, :len(w)], m[b, h].numpy()[w], equal_nan=True)
            assert (kept[b, h, len(w):] == -7.0).all()
    assert (work[need:] == 0x5a).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(3):
        md.copy_(m.roll(1000 * i + 1, 2))
        graph.replay()
        torch.cuda.synchronize()
        eager = call()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def test_calls_of_every_kernel_captured_and_replayed(dev):
    """Many rows, few rows over many blocks, the weight of many rows with a join
    and an eviction in one graph, replayed with new inputs and eager calls
    between, equal the eager calls."""
    B, H, G, D, N = 2, 4, 2, 128, 16_000
    g = torch.Generator().manual_seed(61)
    cache = make_cache(dev, B, H, N, D, "int8", 62, [N, N])
    small = ops.Cache8.empty(B, H, 512, D, dev, "int8")
    q = torch.zeros((B, 150, H * G, D), dtype=torch.bfloat16, device=dev)
    kv = torch.zeros((2, B, 70, H, D), dtype=torch.bfloat16, device=dev)
    start = torch.tensor([130, 7], dtype=torch.int32, device=dev)
    n = torch.tensor([N, 901], dtype=torch.int32, device=dev)

    def calls(small):
        ops.cache8_write(small, kv[0], kv[1], start)
        a, la = ops.cache8_attend(q, cache, n)
        b, lb = ops.cache8_attend(q[:, :1].contiguous(), cache, n)
        c, lc = ops.cache8_attend(q[:, :9].contiguous(), cache, n, causal=True)
        m = torch.zeros((B, H, cache.cap), device=dev)
        ops.cache8_mass(q, cache, la, m, n)
        ops.cache8_mass(q, small, torch.zeros_like(la), m[:, :, :512].contiguous(), 200)
        out = ops.Cache8.empty(B, H, 300, D, dev, "int8")
        om = torch.zeros((B, H, out.cap), device=dev)
        rows, left = ops.cache8_evict(cache, m, n, out, om, keep=300, sink=3, recent=20)
        return [a, la, b, lb, c, lc, m, rows, left, out.k, out.v, out.k_scale, om, small.k,
                small.v_scale]

    def fill(i):
        gi = torch.Generator().manual_seed(70 + i)
        q.copy_(torch.randn(q.shape, generator=gi))
        kv.copy_(torch.randn(kv.shape, generator=gi))

    def fresh():
        return ops.Cache8.empty(B, H, 512, D, dev, "int8")

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls(fresh())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls(small)
    for i in range(4):
        fill(i)
        for t in (small.k, small.v):
            t.zero_()
        for t in (small.k_scale, small.v_scale):
            t.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        want = calls(fresh())                  # eager work between replays
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
