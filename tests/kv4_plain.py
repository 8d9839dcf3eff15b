"""The 4-bit cache operators in fp64 on the CPU, element by element from their definitions."""
import math

import numpy as np

D = 128


def bf16(x):
    """Nearest bf16 value of fp64 numbers, halves to even (normal range)."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 256.0), e - 8)


def quantise(x, group):
    """fp64 [..., 128] -> (values, codes, scale, zero) of the cache's format."""
    y = np.asarray(x, np.float64).reshape(*x.shape[:-1], D // group, group)
    lo, hi = np.minimum(y.min(-1), 0.0), np.maximum(y.max(-1), 0.0)
    with np.errstate(all="ignore"):
        scale = bf16((hi - lo) / 15.0)
        scale = np.where(np.isfinite(y).all(-1), scale, np.nan)
        by = np.where(scale > 0, scale, 1.0)
        zero = np.clip(np.rint(-lo / by), 0, 15)
        codes = np.clip(np.rint(y / by[..., None]) + zero[..., None], 0, 15)
        values = scale[..., None] * (codes - zero[..., None])
    return values.reshape(x.shape), codes.reshape(x.shape), scale, zero


def block_bytes(group):
    return 2 * 16 * (64 + 4 * (D // group))


def code_place(ch, value):
    """(byte in the row, shift) of a channel's code."""
    if value:
        k, g = (ch // 4) // 8, (ch // 4) % 8
        return (g * 4 + k) * 2 + (ch % 4) // 2, 4 * (ch % 2)
    j, c = (ch // 8) // 4, (ch // 8) % 4
    return (c * 4 + j) * 4 + (ch % 8) // 2, 4 * (ch % 2)


def row_offset(slot_in_page, value, group):
    """(offset of a token's codes, of its pairs) in a page of one head."""
    ng = D // group
    base = (slot_in_page // 16) * block_bytes(group) + value * 16 * (64 + 4 * ng)
    t = slot_in_page % 16
    return base + t * 64, base + 16 * 64 + t * 4 * ng


def read_token(page_row, slot_in_page, value, group):
    """fp64 [128] of one token; page_row is the uint8 row of one (page, head)."""
    at, pairs = row_offset(slot_in_page, value, group)
    out = np.empty(D)
    for ch in range(D):
        byte, shift = code_place(ch, value)
        u = (int(page_row[at + byte]) >> shift) & 15
        p = pairs + 4 * (ch // group)
        word = np.frombuffer(page_row[p:p + 4].tobytes(), np.uint16).astype(np.uint32) << 16
        scale, zero = word.view(np.float32).astype(np.float64)
        out[ch] = scale * (u - zero)
    return out


_BYTE = {v: np.array([code_place(c, v)[0] for c in range(D)]) for v in (0, 1)}
_SHIFT = np.array([code_place(c, 0)[1] for c in range(D)])


def read(pages, table, n, page, group, h, value, scales=False):
    """fp64 [n, 128]: the first n slots of a sequence, head h (or each channel's scale). pages is
    uint8 numpy."""
    i = np.arange(n)
    rows = pages[table[i // page], h]
    s = i % page
    ng = D // group
    base = (s // 16) * block_bytes(group) + value * 16 * (64 + 4 * ng)
    code = np.take_along_axis(rows, (base + (s % 16) * 64)[:, None] + _BYTE[value], 1)
    code = (code >> _SHIFT) & 15
    at = (base + 16 * 64 + (s % 16) * 4 * ng)[:, None] + np.arange(4 * ng)
    raw = np.ascontiguousarray(np.take_along_axis(rows, at, 1)).view(np.uint16).astype(np.uint32) << 16
    pair = raw.view(np.float32).astype(np.float64).reshape(n, ng, 2)
    grp = np.arange(D) // group
    if scales:
        return pair[:, grp, 0]
    with np.errstate(invalid="ignore"):
        return pair[:, grp, 0] * (code.astype(np.float64) - pair[:, grp, 1])


def attention(q, pages, table, lengths, counts, *, page, group, heads, causal=True, scale=None):
    """(o, lse, weights, magnitude, step, spread), fp64: o, magnitude, step [B, T, Hq, 128], lse
    [B, Hq, T], weights a list of [n, heads]. magnitude is the sum of w |v|, step that of w *
    value scale, spread the largest sum of |q k| * scale of any row and key: what rounding errors
    are relative to. Rows past a count are NaN."""
    q = q.double().cpu().numpy()
    B, T, Hq, _ = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, mag, step = np.full(q.shape, np.nan), np.zeros(q.shape), np.zeros(q.shape)
    lse, weights, spread = np.full((B, Hq, T), np.nan), [], 0.0
    for b in range(B):
        n, c = int(lengths[b]), int(counts[b])
        got = np.zeros((n, heads))
        for h in range(heads):
            k = read(pages, table[b], n, page, group, h, 0)
            v = read(pages, table[b], n, page, group, h, 1)
            vs = read(pages, table[b], n, page, group, h, 1, scales=True)
            for i in range(c):
                m = max(0, n - (c - 1 - i)) if causal else n
                for hq in range(h * (Hq // heads), (h + 1) * (Hq // heads)):
                    if m == 0:
                        o[b, i, hq], lse[b, hq, i] = 0.0, -np.inf
                        continue
                    with np.errstate(invalid="ignore", over="ignore"):
                        x = (k[:m] @ q[b, i, hq]) * scale
                        top = x.max()
                        e = np.exp(x - top)
                        w = e / e.sum()
                        lse[b, hq, i] = top + np.log(e.sum())
                        o[b, i, hq] = w @ v[:m]
                        mag[b, i, hq] = w @ np.abs(v[:m])
                        step[b, i, hq] = w @ vs[:m]
                        s = (np.abs(k[:m]) @ np.abs(q[b, i, hq])).max() * scale
                    spread = max(spread, s) if np.isfinite(s) else spread
                    got[:m, h] += w
        weights.append(got)
    return o, lse, weights, mag, step, spread


def select(weights, positions, table, n, *, page, keep, recent, seen, h):
    """src of one (sequence, head), and the new length."""
    i = np.arange(n)
    w = weights[table[i // page], h, i % page].astype(np.float64)
    pos = positions[table[i // page], h, i % page].astype(np.int64)
    def rank(t):
        if pos[t] >= seen - recent:
            return (True, 0.0, 0, t)
        return (False, math.inf, 1, t) if math.isnan(w[t]) else (False, w[t], 0, t)

    order = sorted(range(n), key=rank)
    gone = set(order[:max(0, n - keep)])
    movers = [t for t in range(keep, n) if t not in gone]
    src = np.full(keep, -1, np.int32)
    for d in range(min(n, keep)):
        src[d] = movers.pop(0) if d in gone else d
    assert not movers
    return src, min(n, keep)

