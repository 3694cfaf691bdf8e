"""Plain implementations of the 8-bit cache's operators for its tests: codes and
scales to the last bit (fp32 numpy, torch's e4m3 cast), attention in 64 bits
with a bound on what a kernel may be off by."""
import numpy as np
import torch

BLOCK = 64
TOP = {"int8": np.float32(127), "e4m3": np.float32(448)}
TINY = np.float32(2.0 ** -64)


def pitch(D):
    return 64 if D <= 64 else 128


def to_codes(x, fmt):
    """fp32 array -> codes (int8 array, or the bytes of e4m3)."""
    x = np.where(np.isnan(x), np.float32(0), x.astype(np.float32))
    x = np.clip(x, -TOP[fmt], TOP[fmt])
    if fmt == "int8":
        return np.rint(x).astype(np.int8)
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def values(codes, fmt):
    if fmt == "int8":
        return codes.astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(codes)).view(torch.float8_e4m3fn).float().numpy()


def write(codes, scale, x, start, counts, fmt):
    """codes [B, H, cap, P], scale [B, H, nb], x [B, T, H, D] fp32; start and
    counts lists.  Returns new copies."""
    codes, scale = codes.copy(), scale.copy()
    B, H, cap, P = codes.shape
    D = x.shape[3]
    for b in range(B):
        st = min(max(start[b], 0), cap)
        end = min(st + min(max(counts[b], 0), x.shape[1]), cap)
        for h in range(H):
            for blk in range(st // BLOCK, -(-end // BLOCK)):
                lo, hi = max(st, blk * BLOCK), min(end, (blk + 1) * BLOCK)
                if lo >= hi:
                    continue
                rows = x[b, lo - st:hi - st, h].astype(np.float32)
                a = np.abs(rows)
                top = np.float32(np.max(np.where(np.isfinite(a), a, 0)))
                s = np.float32(max(top, TINY) / TOP[fmt])
                if lo > blk * BLOCK:
                    s0 = scale[b, h, blk]
                    if s0 >= s:
                        s = s0
                    else:
                        old = slice(blk * BLOCK, lo)
                        ratio = np.float32(s0 / s)
                        codes[b, h, old] = to_codes(values(codes[b, h, old], fmt) * ratio, fmt)
                scale[b, h, blk] = s
                with np.errstate(invalid="ignore", over="ignore"):
                    codes[b, h, lo:hi, :D] = to_codes(rows / s, fmt)
                codes[b, h, lo:hi, D:] = 0
    return codes, scale


def dequant(codes, scale, fmt, D):
    """float64 values [B, H, cap, D]."""
    v = values(codes[..., :D], fmt).astype(np.float64)
    return v * np.repeat(scale.astype(np.float64), BLOCK, axis=2)[..., None]


def visible(B, Q, lengths, causal):
    """[B, Q] first hidden key of each query."""
    n = np.asarray(lengths)[:, None] + np.zeros((B, Q), int)
    return np.maximum(n - Q + 1 + np.arange(Q)[None] if causal else n, 0)


def attend(q, k, v, lengths, causal, scale, u):
    """q [B, Q, Hq, D], k/v [B, H, cap, D] float64 -> out, lse, and bounds on
    the error of a kernel whose outputs have half-step u: a weight is rounded to
    fp16 (W, half a step; absolutely below its normal range), the results of key
    splits to fp16 once more, the output by u, a score by the fp32 sum of its D
    products and one fused multiply-add (D + 4 roundings of 2^-24 of the sum of
    their magnitudes, an exponential twice that)."""
    W = 2 * 2.0 ** -11
    B, Q, Hq, D = q.shape
    H = k.shape[1]
    G = Hq // H
    end = visible(B, Q, lengths, causal)
    out, otol = np.zeros((B, Q, Hq, D)), np.zeros((B, Q, Hq, D))
    lse, ltol = np.full((B, Hq, Q), -np.inf), np.zeros((B, Hq, Q))
    for b in range(B):
        for h in range(Hq):
            n = int(end[b].max())
            if n == 0:
                continue
            kk, vv = k[b, h // G, :n], v[b, h // G, :n]
            hidden = np.arange(n)[None] >= end[b][:, None]
            some = end[b] > 0
            z = np.where(hidden, -np.inf, q[b, :, h] @ kk.T * scale)
            mag = np.where(hidden, 0, np.abs(q[b, :, h]) @ np.abs(kk).T * scale).max(1)
            ez = (D + 4) * 2.0 ** -24 * mag + 2.0 ** -21
            m = np.where(some, z.max(1), 0)
            p = np.exp(z - m[:, None])
            tot = np.where(some, p.sum(1), 1)
            out[b, :, h] = p @ vv / tot[:, None]
            a = p @ np.abs(vv) / tot[:, None]
            # weights below fp16's normal range (they are lifted by 2^12), and
            # fp16 outputs below it: a number under 2^-14 is rounded to a
            # multiple of 2^-24, so it is off by up to 2^-25, not by u of itself
            small = n * 2.0 ** -37 * np.abs(vv).max() + (2.0 ** -25 if u == 2.0 ** -11 else 0)
            otol[b, :, h] = ((W + 4 * ez)[:, None] * a * 1.01 + u * np.abs(out[b, :, h])
                             + small + 1e-30)
            lse[b, h] = np.where(some, m + np.log(tot), -np.inf)
            ltol[b, h] = 2 * ez + 2.0 ** -22 * (np.abs(m) + np.abs(np.log(tot)) + 1)
    return out, lse, otol, ltol


def mass(q, k, lse, start, lengths, causal, scale):
    """[B, H, cap] float64 sums and the bound of the kernel's."""
    B, Q, Hq, D = q.shape
    H = k.shape[1]
    end = visible(B, Q, lengths, causal)
    out, tol = start.astype(np.float64).copy(), np.abs(start).astype(np.float64) * 2.0 ** -23
    for b in range(B):
        for h in range(Hq):
            n = int(end[b].max())
            some = (end[b] > 0) & ~np.isneginf(lse[b, h])
            kk, hk = k[b, h // (Hq // H), :n], h // (Hq // H)
            seen = (np.arange(n)[None] < end[b][:, None]) & some[:, None]
            off = np.where(some, lse[b, h], 0.0)[:, None]
            z = q[b, :, h] @ kk.T * scale
            mag = np.abs(q[b, :, h]) @ np.abs(kk).T * scale
            p = np.where(seen, np.exp(np.where(seen, z - off, 0.0)), 0.0)
            ez = (D + 4) * 2.0 ** -24 * mag + 2.0 ** -22 * (np.abs(off) + 2)
            out[b, hk, :n] += p.sum(0)
            tol[b, hk, :n] += (p * (2 * ez + (Q * Hq // H + 2) * 2.0 ** -24)).sum(0)
    return out, tol + 1e-30


def evict(m, lengths, keep, sink, recent):
    """Kept rows [B][H] lists."""
    B, H, _ = m.shape
    got = []
    for b in range(B):
        heads = []
        for h in range(H):
            n = lengths[b]
            if n <= keep:
                heads.append(list(range(n)))
                continue
            w = m[b, h].astype(np.float64)
            w = np.where(np.isnan(w), np.inf, w)
            nan = np.isnan(m[b, h])
            mid = sorted(range(sink, n - recent), key=lambda i: (not nan[i], -w[i], i))
            heads.append(list(range(sink)) + sorted(mid[:keep - sink - recent])
                         + list(range(n - recent, n)))
        got.append(heads)
    return got


def compact(codes, scale, rows, out_codes, out_scale, fmt):
    out_codes, out_scale = out_codes.copy(), out_scale.copy()
    for b, heads in enumerate(rows):
        for h, r in enumerate(heads):
            for blk in range(-(-len(r) // BLOCK)):
                src = np.array(r[blk * BLOCK:(blk + 1) * BLOCK])
                s0 = scale[b, h, src // BLOCK]
                s = s0.max()
                c = codes[b, h, src]
                moved = to_codes(values(c, fmt) * (s0 / s).astype(np.float32)[:, None], fmt)
                at = slice(blk * BLOCK, blk * BLOCK + len(src))
                out_codes[b, h, at] = np.where((s0 == s)[:, None], c, moved)
                out_scale[b, h, blk] = s
    return out_codes, out_scale
