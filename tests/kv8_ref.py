"""Plain 64-bit forms of the operators between the projections (numpy), and the
host arrays that their tests build: e4m3 codes, paged caches, batches."""
from __future__ import annotations

import numpy as np

U32, U24 = 2.0 ** -24, 2.0 ** -22  # half a step of fp32; an fp32 exponential or two-term fp16 weight


def e4m3_values() -> np.ndarray:
    """The value of each of the 256 codes."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 0x7f) == 0x7f, np.nan, v)
    return np.where(c >= 128, -v, v)


VALUES = e4m3_values()
_POS = VALUES[:0x7f]  # ascending, 0 .. 448


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest code, ties to the even one; NaN and infinities to 0xff.  |x| <= 448 + half a step."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(_POS, a), 1, 0x7e)
    lo = hi - 1
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(np.signbit(x), c | 0x80, c)
    return np.where(np.isfinite(x), c, 0xff).astype(np.uint8)


def block_scale(peak: float) -> float:
    """Smallest power of two from 2^-100 on that brings peak to at most 448."""
    s = 2.0 ** -100
    if peak > 448 * s:
        s = 2.0 ** np.ceil(np.log2(peak / 448.0))
        while peak / s > 448:
            s *= 2
        while s > 2.0 ** -100 and peak / (s / 2) <= 448:
            s /= 2
    return float(s)


def norm_rope(x, positions, freq, rot, pairs, w=None, eps=1e-6):
    """x [rows, heads, d] in 64 bits."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    y = x.copy()
    if rot:
        ang = np.asarray(positions, np.float64)[:, None] * np.asarray(freq, np.float64)[None]
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        ia = np.arange(0, rot, 2) if pairs else np.arange(rot // 2)
        ib = ia + 1 if pairs else ia + rot // 2
        a, b = x[..., ia], x[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


class Batch:
    """Ragged sequences over a shuffled page pool: lens tokens each, rows of them the call's own."""

    def __init__(self, rng, lens, rows, P, spare=2, behind=0):
        self.lens, self.rows, self.P = list(lens), list(rows), P
        need = [-(-n // P) for n in lens]
        self.pages = sum(need) + spare
        self.stride = max(1, max(need))
        order = rng.permutation(self.pages)
        self.table = np.full((len(lens), self.stride), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.total = int(self.start[-1]) + behind

    def upload(self, ctx, max_rows=None, max_len=None):
        from edgerunner_amd import KV8Batch
        self.bufs = [ctx.upload(a) for a in (self.table, np.array(self.lens, np.int32), self.start)]
        return KV8Batch(*self.bufs, len(self.lens), self.stride, self.total,
                        max(1, max(self.rows)) if max_rows is None else max_rows,
                        max(self.lens) if max_len is None else max_len)


def append(codes, scales, batch, x):
    """Appends x [total rows, heads, d] (64-bit values) to copies of codes [pages, heads, P, d] and scales [pages, heads]."""
    codes, scales, P = codes.copy(), scales.copy(), batch.P
    for s, (n, m) in enumerate(zip(batch.rows, batch.lens)):
        first = max(m - n, 0)
        for p in range(first // P, -(-m // P)) if n else ():
            page = batch.table[s, p]
            if not 0 <= page < codes.shape[0]:
                continue
            a, b = max(first, p * P), min(m, p * P + P)
            r0 = batch.start[s] + n - m
            for h in range(codes.shape[1]):
                new = x[r0 + a:r0 + b, h]
                fin = np.abs(new[np.isfinite(new)])
                need = block_scale(fin.max() if fin.size else 0.0)
                old = float(scales[page, h]) if a > p * P else 0.0
                now = max(old, need)
                if old and now > old:
                    k = slice(0, a - p * P)
                    codes[page, h, k] = to_e4m3(VALUES[codes[page, h, k]] * (old / now))
                codes[page, h, a - p * P:b - p * P] = to_e4m3(new / now)
                scales[page, h] = now
    return codes, scales


def read(codes, scales, batch, s, h, pages=None):
    """Tokens of sequence s and head h as values, and which of them have a page."""
    m, P = batch.lens[s], batch.P
    d = codes.shape[3]
    v, ok = np.zeros((m, d)), np.zeros(m, bool)
    for p in range(-(-m // P)):
        page = batch.table[s, p]
        if 0 <= page < codes.shape[0]:
            b = min(m, p * P + P)
            v[p * P:b] = VALUES[codes[page, h, :b - p * P]] * np.float64(scales[page, h])
            ok[p * P:b] = True
    return v, ok


def attend(kc, ks, vc, vs, batch, q, scale, window=0, half=False):
    """(out, bound) [total rows, query heads, d]; rows without visible tokens are 0, and rows of no sequence NaN with bound 0.

    The bound, elementwise: scores are off by at most (d + 8) half steps of fp32 of sum |q k| scale (products exact, sums of
    d of them, the query split into two fp16 terms: 22 bits, or one: 11), weights and their sums by 2^-22 each (2^-11 for one
    term) and the length of the sums, all of it on sum w |v| / sum w; the stored value by half a step of its type."""
    H, d = kc.shape[1], kc.shape[3]
    G = q.shape[1] // H
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s, (n, m) in enumerate(zip(batch.rows, batch.lens)):
        for h in range(H):
            if not n:
                continue
            K, ok = read(kc, ks, batch, s, h)
            V, _ = read(vc, vs, batch, s, h)
            for i in range(n):
                r, pos = batch.start[s] + i, m - n + i
                lo = max(0, pos - window + 1) if window else 0
                see = np.zeros(m, bool)
                see[lo:max(pos + 1, 0)] = True
                see &= ok
                for g in range(G):
                    if not see.any():
                        out[r, h * G + g] = 0.0
                        continue
                    x = np.asarray(q[r, h * G + g], np.float64)
                    k, v = K[see], V[see]
                    sc = (k @ x) * scale
                    w = np.exp(sc - sc.max())
                    w = w / w.sum()
                    o = w @ v
                    av = w @ np.abs(v)
                    each = (2.0 ** -12 + 2.0 ** -21) if half else 2.0 ** -22
                    ds = ((d + 8) * U32 + each) * (np.abs(k) @ np.abs(x)).max() * abs(scale)
                    term = 2.0 ** -11 if half else U24
                    t = (2 * ds * (1 + ds) + term + 4 * U24 + 2 * (m + 8) * U32) * av
                    out[r, h * G + g] = o
                    tol[r, h * G + g] = t + (2.0 ** -8 * np.abs(o) * (1 + 1e-6) if half else 0.0)
    return out, tol


def bf16_to_f32(u16: np.ndarray) -> np.ndarray:
    return (u16.astype(np.uint32) << 16).view(np.float32)
