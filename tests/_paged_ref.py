"""Plain 64-bit forms of the paged cache's operators, on numpy arrays, with bounds of
the kernels' errors derived from where they round."""
import numpy as np
import torch

HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}      # half a step, relative


def rotate(x, at, freqs, interleaved):
    """x [T, heads, D] float64 by positions at [T]; and what each column's error is
    relative to (its pair's two magnitudes)."""
    rot = 2 * len(freqs)
    ang = np.asarray(at, np.float64)[:, None] * freqs.astype(np.float64)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y, mag = x.copy(), np.zeros_like(x)
    i = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., i[0]], x[..., i[1]]
    y[..., i[0]], y[..., i[1]] = a * c - b * s, b * c + a * s
    mag[..., i[0]] = mag[..., i[1]] = np.abs(a) + np.abs(b)
    return y, mag


def rotate_bound(y, mag, u, f16):
    """fp32: the sine and cosine within 2^-22 (the turn's own rounding, half of 2^-24 of a
    turn, and the function's), three roundings of 2^-24; then half a step of the
    16-bit type, and fp16's step below its normal range."""
    return u * np.abs(y) + 2.0 ** -20 * mag + (2.0 ** -25 if f16 else 0) + 1e-30


def slots(table, page, row):
    """(page, row in it) of a sequence's row, or None where there is none."""
    if row < 0 or row // page >= len(table):
        return None
    return int(table[row // page]), row % page


def gather(pool, table, n):
    """[H, n, D] rows of a sequence; NaN where no page is."""
    pages, H, page, D = pool.shape
    out = np.full((H, n, D), np.nan)
    there = np.zeros(n, bool)
    for r in range(n):
        p, i = slots(table, page, r)
        if 0 <= p < pages:
            out[:, r] = pool[p, :, i]
            there[r] = True
    return out, there


def visible(Q, n, count, causal=False, parents=None):
    """[Q, n] truth values."""
    see = np.zeros((Q, n), bool)
    for t in range(min(Q, count)):
        if parents is not None:
            see[t, :max(0, n - count)] = True
            a = t
            while True:
                if n - count + a >= 0:
                    see[t, n - count + a] = True
                up = int(parents[a])
                if not 0 <= up < a:
                    break
                a = up
        else:
            see[t, :max(0, n - count + 1 + t) if causal else n] = True
    return see


def attend(q, k, v, see, scale, u, W):
    """One sequence: q [Q, Hq, D], k and v [H, n, D], see [Q, n].  (out [Q, Hq, D], lse
    [Hq, Q], bounds of both); u: half a step of the output's type, W: of the weights'."""
    Q, Hq, D = q.shape
    H, n, _ = k.shape
    out, otol = np.zeros((Q, Hq, D)), np.zeros((Q, Hq, D))
    lse, ltol = np.full((Hq, Q), -np.inf), np.zeros((Hq, Q))
    for h in range(Hq):
        kk, vv = k[h // (Hq // H)], v[h // (Hq // H)]
        for t in range(Q):
            at = see[t]
            if not at.any():
                continue
            z = kk[at] @ q[t, h] * scale
            # scores: D products added in fp32, and the scale's rounding; the exponent's
            # rounding grows with the distance from the maximum
            ez = (D + 4) * 2.0 ** -24 * (np.abs(kk[at]) @ np.abs(q[t, h])).max() * scale + 2.0 ** -21
            m = z.max()
            p = np.exp(z - m)
            tot = p.sum()
            out[t, h] = p @ vv[at] / tot
            a = p @ np.abs(vv[at]) / tot
            adds = (len(z) + 32) * 2.0 ** -24
            # weights below fp16's normal range (lifted by 2^12, the maximum at most 2^3
            # behind) and fp16 outputs below it
            small = len(z) * 2.0 ** -37 * np.abs(vv[at]).max() + (2.0 ** -25 if u == 2.0 ** -11 else 0)
            otol[t, h] = (W + 4 * ez + 2 * adds) * a * 1.01 + u * np.abs(out[t, h]) + small + 1e-30
            lse[h, t] = m + np.log(tot)
            ltol[h, t] = 2 * ez + adds + 2.0 ** -22 * (abs(m) + abs(np.log(tot)) + 1)
    return out, lse, otol, ltol


def attend_gpu(q, k, v, see, scale, u, W):
    """The same in torch on the tensors' device, for large sequences: q [Q, Hq, D], k and
    v [H, n, D] float64, see [Q, n]."""
    Q, Hq, D = q.shape
    H, n, _ = k.shape
    some = see.any(1)
    out, otol = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((Hq, Q), -np.inf, dtype=q.dtype, device=q.device)
    ltol = torch.zeros_like(lse)
    count = see.sum(1).to(q.dtype)
    if n == 0:
        return out, lse, otol, ltol
    for h in range(Hq):
        kk, vv = k[h // (Hq // H)], v[h // (Hq // H)]
        z = (q[:, h] @ kk.T * scale).masked_fill(~see, -np.inf)
        mag = (q[:, h].abs() @ kk.abs().T).masked_fill(~see, 0).amax(1) * scale
        ez = (D + 4) * 2.0 ** -24 * mag + 2.0 ** -21
        m = torch.where(some, z.amax(1), 0)
        p = torch.exp(z - m[:, None])
        tot = torch.where(some, p.sum(1), 1)
        out[:, h] = p @ vv / tot[:, None]
        a = p @ vv.abs() / tot[:, None]
        adds = (count + 32) * 2.0 ** -24
        top = (see[:, :, None] * vv.abs().amax(1)[None, :, None]).amax((1, 2))
        small = count * 2.0 ** -37 * top + (2.0 ** -25 if u == 2.0 ** -11 else 0)
        otol[:, h] = ((W + 4 * ez + 2 * adds)[:, None] * a * 1.01 + u * out[:, h].abs()
                      + small[:, None] + 1e-30)
        lse[h] = torch.where(some, m + torch.log(tot), -np.inf)
        ltol[h] = 2 * ez + adds + 2.0 ** -22 * (m.abs() + torch.log(tot).abs() + 1)
    return out, lse, otol, ltol


def commit(pool, table, start, rows, count):
    """A pool after the move of each sequence's rows, all read before any is written."""
    new = pool.copy()
    pages, _, page, _ = pool.shape
    for b in range(len(table)):
        for j in range(count[b]):
            if rows[b][j] < 0:
                continue
            src, dst = slots(table[b], page, start[b] + rows[b][j]), slots(table[b], page, start[b] + j)
            if src and dst and 0 <= src[0] < pages and 0 <= dst[0] < pages:
                new[dst[0], :, dst[1]] = pool[src[0], :, src[1]]
    return new
