"""Plain 64-bit forms of attention under masks, of the acceptance of drafts and
of rules on logits (numpy), and the trees that their tests build."""
from __future__ import annotations

import numpy as np

import kv8_ref as R

U24 = 2.0 ** -24  # half a step of fp32


def tree(rng, n, tokens=1000, chain=False):
    """(parent, token) of n drafts: the first is the root, every other hangs on an earlier one."""
    parent = np.array([-1] + [i - 1 if chain else int(rng.integers(0, i)) for i in range(1, n)], np.int32)
    return parent[:n], rng.integers(0, tokens, n).astype(np.int32)


def lines(parent):
    """seen[i, j]: j is i or one of its ancestors."""
    n = len(parent)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = int(parent[j])
    return seen


def words(bits, n_words=None):
    """Truth values [rows, n] as uint32 words, lowest bit first; bits behind the last are ones, which nothing may read."""
    rows, n = bits.shape
    n_words = -(-n // 32) if n_words is None else n_words
    padded = np.ones((rows, n_words * 32), np.uint64)
    padded[:, :n] = bits
    return (padded.reshape(rows, n_words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def visible(m, n, window, sinks, seen=None, position=None):
    """[n, m]: the tokens of m that each of a sequence's n rows sees (seen: masks of the drafts)."""
    base, t = m - n, np.arange(m)
    out = np.zeros((n, m), bool)
    for i in range(n):
        if base + i < 0:
            continue
        if seen is None:
            p, hi = base + i, base + i + 1
        else:
            hi = max(base, 0)
            p = min(max(int(position[i]), base), m - 1) if window else m
        out[i] = (t < hi) & ((t < sinks) | ((t > p - window) if window else True))
        if seen is not None:
            for j in range(max(0, -base), n):
                out[i, base + j] = seen[i, j]
    return out


def attend(kc, ks, vc, vs, batch, q, scale, see, half=False):
    """(out, bound) [total rows, query heads, d] over the tokens that see[s] [n, m] shows; the bound as kv8_ref.attend's."""
    H, d = kc.shape[1], kc.shape[3]
    G = q.shape[1] // H
    out, tol = np.full(q.shape, np.nan), np.zeros(q.shape)
    for s, (n, m) in enumerate(zip(batch.rows, batch.lens)):
        for h in range(H):
            if not n:
                continue
            K, ok = R.read(kc, ks, batch, s, h)
            V, _ = R.read(vc, vs, batch, s, h)
            for i in range(n):
                r = batch.start[s] + i
                sees = see[s][i] & ok
                if not sees.any():
                    out[r, h * G:h * G + G] = 0.0
                    continue
                k, v = K[sees], V[sees]
                x = np.asarray(q[r, h * G:h * G + G], np.float64)
                sc = (x @ k.T) * scale
                w = np.exp(sc - sc.max(1, keepdims=True))
                w = w / w.sum(1, keepdims=True)
                o, av = w @ v, w @ np.abs(v)
                each = (2.0 ** -12 + 2.0 ** -21) if half else 2.0 ** -22
                ds = ((d + 8) * U24 + each) * (np.abs(x) @ np.abs(k).T).max(1)[:, None] * abs(scale)
                t = (2 * ds * (1 + ds) + (2.0 ** -11 if half else 2.0 ** -22) + 4 * 2.0 ** -22 + 2 * (m + 8) * U24) * av
                out[r, h * G:h * G + G] = o
                tol[r, h * G:h * G + G] = t + (2.0 ** -8 * np.abs(o) * (1 + 1e-6) if half else 0.0)
    return out, tol


def walk(parent, token, chosen):
    path = [0]
    while True:
        cur, t = path[-1], chosen[path[-1]]
        after = [r for r in range(cur + 1, len(parent)) if parent[r] == cur and token[r] == t] if t >= 0 else []
        if not after:
            return path, int(t)
        path.append(after[0])


def accept(codes, scales, batch, paths):
    """Copies of codes [pages, heads, P, d] and scales after each sequence's kept rows have moved."""
    codes, scales, P = codes.copy(), scales.copy(), batch.P
    pages = codes.shape[0]

    def page_of(s, t):
        p = int(batch.table[s, t // P])
        return p if 0 <= p < pages else -1
    for s, path in enumerate(paths):
        base = batch.lens[s] - batch.rows[s]
        moved = [j for j, r in enumerate(path) if r != j]
        if not moved:
            continue
        first, last = max(base + moved[0], 0), base + len(path)
        was = {}  # the values before anything moves
        for t in range(first, last):
            f = base + path[t - base]
            if page_of(s, f) >= 0:
                was[t] = R.VALUES[codes[page_of(s, f), :, f % P]] * scales[page_of(s, f)].astype(np.float64)[:, None]
        for p in range(first // P, (last - 1) // P + 1):
            page, a, b = page_of(s, p * P), max(first, p * P), min(last, p * P + P)
            here = [t for t in range(a, b) if t in was]
            if page < 0 or not here:
                continue
            for h in range(codes.shape[1]):
                new = np.stack([was[t][h] for t in here])
                fin = np.abs(new[np.isfinite(new)])
                old = float(scales[page, h]) if a > p * P else 0.0
                now = max(old, R.block_scale(fin.max() if fin.size else 0.0))
                if old and now > old:
                    k = slice(0, a - p * P)
                    codes[page, h, k] = R.to_e4m3(R.VALUES[codes[page, h, k]] * (old / now))
                for t, x in zip(here, new):
                    codes[page, h, t % P] = R.to_e4m3(x / now)
                scales[page, h] = now
    return codes, scales


def choose(x, context, penalty=None, bias=(), allowed=None):
    """One row: (value in 64 bits of each token, chosen).  context: tokens; bias: (token, value) in order; allowed: truth values."""
    V = len(x)
    y = np.asarray(x, np.float64).copy()
    if penalty is not None:
        c = np.bincount([t for t in context if 0 <= t < V], minlength=V)
        rep, pres, freq = (np.float64(np.float32(v)) for v in penalty)
        with np.errstate(all="ignore"):
            less = np.where(y > 0, y / rep, y * rep) - (pres + freq * c)
        y = np.where(c > 0, less, y)
    for t, b in dict((t, b) for t, b in bias if 0 <= t < V).items():
        y[t] += np.float64(np.float32(b))
    able = np.ones(V, bool) if allowed is None else allowed
    y = np.where(able, y, -np.inf)
    with np.errstate(over="ignore"):
        z = y.astype(np.float32)
    left = able & ~np.isnan(z)
    return y, int(np.flatnonzero(left & (z == z[left].max()))[0]) if left.any() else -1
