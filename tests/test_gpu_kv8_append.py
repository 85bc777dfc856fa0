"""Head norms with the rotation, and appends to the 8-bit cache, against plain
64-bit forms.  Rotated values: an RMS norm over d fp32 terms, one fp32 product
with the weight, angles reduced in 64 bits and rounded to 2^-25 turns, two
products and a sum: (d / 8 + 24) half steps of fp32 of |a| + |b| bound it.
Codes: where nothing is computed before (values; keys without norm and
rotation) every byte is the nearest code; else a code is at most half a step
plus that error away."""
import numpy as np
import pytest

import kv8_ref as R
from edgerunner_amd import HeadRows, KV8AppendKernel, KV8Batch, KV8Cache, QKNormRopeKernel, Rope

pytestmark = pytest.mark.gpu


def freqs(rot, base=10000.0):
    return (base ** (-np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32)


def turn_tol(x, rot, pairs, w, eps=1e-6):
    """Bound of norm_rope's fp32 error: half steps of |a| + |b| of the normed pair."""
    n = np.abs(R.norm_rope(x, None, None, 0, pairs, w, eps))
    s = n.copy()
    if rot:
        ia = np.arange(0, rot, 2) if pairs else np.arange(rot // 2)
        ib = ia + 1 if pairs else ia + rot // 2
        s[..., ia] = s[..., ib] = n[..., ia] + n[..., ib]
    return (x.shape[-1] / 8 + 24) * R.U32 * s + 1e-40


@pytest.mark.parametrize("d,rot,pairs,norm,rows,hq,hk,pad,far", [
    (64, 64, False, True, 1, 14, 2, 0, 4096), (64, 32, True, False, 77, 14, 2, 0, 1 << 20),
    (64, 8, False, True, 5, 1, 1, 3, 100), (128, 128, False, True, 3, 16, 8, 0, 131072),
    (128, 128, True, True, 33, 5, 3, 1, 1 << 24), (128, 64, False, False, 7, 32, 8, 0, 9000),
    (128, 0, False, True, 2, 3, 1, 0, 10), (256, 256, False, True, 9, 8, 4, 0, 2 ** 31 - 1),
    (256, 128, True, True, 1, 1, 1, 5, 40000), (256, 248, False, False, 4, 3, 2, 0, 500),
    (128, 128, False, True, 6000, 5, 3, 0, 8192)])
def test_norm_rope(ctx, d, rot, pairs, norm, rows, hq, hk, pad, far):
    rng = np.random.default_rng(d + rot + rows)
    width = (hq + hk) * d + pad  # q and k as columns of one row; an odd pad leaves rows 4-byte aligned
    x = (rng.standard_normal((rows, width)) * 3).astype(np.float32)
    pos = rng.integers(0, far, rows).astype(np.int32)
    pos[0] = far - 1
    wq, wk = [(rng.random(d) + 0.5).astype(np.float32) for _ in range(2)]
    xb, pb, qb, kb = ctx.upload(x), ctx.upload(pos), ctx.upload(wq), ctx.upload(wk)
    f = freqs(rot)
    fb = ctx.upload(f) if rot else None
    qo, ko = ctx.upload(np.full((rows, hq * d), 7, np.float32)), ctx.upload(np.full((rows, hk * d + 1), 7, np.float32))
    rope = Rope(fb, rot, pairs)
    q, k = HeadRows(xb, hq, width), HeadRows(xb.view(4 * hq * d), hk, width)
    kern = QKNormRopeKernel(ctx)
    args = (pb, rows, d, rope, qb if norm else None, kb if norm else None)
    kern.encode(None, q, k, HeadRows(qo, hq, hq * d), HeadRows(ko, hk, hk * d + 1), *args)
    ctx.synchronize()
    gq = qo.download(np.float32).reshape(rows, hq, d)
    gk = ko.download(np.float32).reshape(rows, hk * d + 1)
    assert np.all(gk[:, -1] == 7)  # between the rows
    gk = gk[:, :-1].reshape(rows, hk, d)
    for got, at, heads, w in ((gq, 0, hq, wq), (gk, hq * d, hk, wk)):
        src = x[:, at:at + heads * d].reshape(rows, heads, d)
        w = w if norm else None
        exp = R.norm_rope(src, pos, f, rot, pairs, w)
        assert np.all(np.abs(got - exp) <= turn_tol(src, rot, pairs, w))
        if not norm:
            assert np.array_equal(got[..., rot:], src[..., rot:])
    # in place, queries and keys where they are: the same bits; then queries alone
    kern.encode(None, q, k, q, k, *args)
    ctx.synchronize()
    both = xb.download(np.float32).reshape(rows, width)
    assert np.array_equal(both[:, :hq * d].reshape(rows, hq, d), gq)
    assert np.array_equal(both[:, hq * d:(hq + hk) * d].reshape(rows, hk, d), gk)
    assert np.array_equal(both[:, (hq + hk) * d:], x[:, (hq + hk) * d:])
    xb.upload(x)
    kern.encode(None, q, None, q, None, *args[:5])
    ctx.synchronize()
    both = xb.download(np.float32).reshape(rows, width)
    assert np.array_equal(both[:, :hq * d].reshape(rows, hq, d), gq)
    assert np.array_equal(both[:, hq * d:], x[:, hq * d:])


def test_norm_rope_zero_and_non_finite_rows(ctx):
    """A zero head stays zero under eps > 0; NaN and infinity touch their own head alone."""
    d, rows, hq = 128, 3, 5
    x = np.random.default_rng(0).standard_normal((rows, hq, d)).astype(np.float32)
    clean = x.copy()
    x[0, 1] = 0
    x[1, 2, 5] = np.nan
    x[2, 3, 7] = np.inf
    w = np.ones(d, np.float32)
    f, pos = freqs(d), np.arange(rows, dtype=np.int32)
    bufs = [ctx.upload(a) for a in (x, pos, w, f)]
    q = HeadRows(bufs[0], hq, hq * d)
    QKNormRopeKernel(ctx).encode(None, q, None, q, None, bufs[1], rows, d, Rope(bufs[3], d), bufs[2])
    ctx.synchronize()
    got = bufs[0].download(np.float32).reshape(rows, hq, d)
    assert np.all(got[0, 1] == 0) and np.all(np.isnan(got[1, 2])) and np.isnan(got[2, 3, 7])
    exp = R.norm_rope(clean, pos, f, d, False, w)
    tol = turn_tol(clean, d, False, w)
    for r, h in ((0, 1), (1, 2), (2, 3)):
        exp[r, h], got[r, h] = 0, 0
    assert np.all(np.abs(got - exp) <= tol)


def garbage(rng, pages, heads, P, d):
    """A pool as earlier users leave it: any code, NaN among them, and any scale."""
    codes = rng.integers(0, 256, (pages, heads, P, d)).astype(np.uint8)
    scales = np.where(rng.random((pages, heads)) < 0.2, np.nan, 2.0 ** rng.integers(-8, 8, (pages, heads))).astype(np.float32)
    return codes, scales


class Case:
    """An append of rows of random keys and values to ragged sequences, run and compared."""

    def __init__(self, ctx, rng, lens, rows, P, d, heads, rot=None, pairs=False, norm=False, vhalf=False, hq=0, behind=0,
                 spread=1.0):
        self.ctx, self.d, self.heads, self.hq, self.vhalf = ctx, d, heads, hq, vhalf
        self.rot, self.pairs = d if rot is None else rot, pairs
        self.b = R.Batch(rng, lens, rows, P, behind=behind)
        n = self.b.total
        self.k = (rng.standard_normal((n, heads, d)) * 2.0 ** (spread * rng.standard_normal((n, heads, 1)))).astype(np.float32)
        v = (rng.standard_normal((n, heads, d)) * 2.0 ** (spread * rng.standard_normal((n, heads, 1)))).astype(np.float32)
        self.v = v.astype(np.float16) if vhalf else v
        self.q = rng.standard_normal((n, max(hq, 1), d)).astype(np.float32)
        self.w = (rng.random(d) + 0.5).astype(np.float32) if norm else None
        self.f = freqs(self.rot)
        self.kc, self.ks = garbage(rng, self.b.pages, heads, P, d)
        self.vc, self.vs = garbage(rng, self.b.pages, heads, P, d)
        for s, (r, m) in enumerate(zip(rows, lens)):  # tokens of earlier calls: finite codes and a positive scale
            for p in range(max(m - r, 0) // P + 1 if m else 0):
                page = self.b.table[s, p]
                for c, sc in ((self.kc, self.ks), (self.vc, self.vs)):
                    c[page][(c[page] & 0x7f) == 0x7f] = 0x30
                    sc[page] = 2.0 ** rng.integers(-9, -4, heads)

    def run(self, **over):
        ctx, d, heads = self.ctx, self.d, self.heads
        up = ctx.upload
        self.bufs = [up(a) for a in (self.kc, self.vc, self.ks, self.vs)]
        P = self.kc.shape[2]
        self.cache = KV8Cache(*self.bufs, self.kc.shape[0], heads, P, d)
        self.batch = over.pop("batch", None) or self.b.upload(ctx)
        self.io = [up(self.k), up(self.v), up(self.q), up(np.full_like(self.q, 7))]
        fb = up(self.f) if self.rot else None
        wb = up(self.w) if self.w is not None else None
        rows = HeadRows(self.io[2], self.hq, self.hq * d) if self.hq else None
        out = HeadRows(self.io[3], self.hq, self.hq * d) if self.hq else None
        self.args = (self.cache, self.batch, HeadRows(self.io[0], heads, heads * d), HeadRows(self.io[1], heads, heads * d),
                     Rope(fb, self.rot, self.pairs))
        self.more = dict(kNorm=wb, q=rows, qOut=out, qNorm=wb if self.hq else None, vHalf=self.vhalf, **over)
        KV8AppendKernel(ctx).encode(None, *self.args, **self.more)
        ctx.synchronize()
        return self.read()

    def read(self):
        kc, vc, ks, vs = (b.download(t).reshape(a.shape) for b, t, a in zip(
            self.bufs, (np.uint8, np.uint8, np.float32, np.float32), (self.kc, self.vc, self.ks, self.vs)))
        return kc, ks, vc, vs

    def positions(self):
        pos = np.full(self.b.total, -1)
        for s, (r, m) in enumerate(zip(self.b.rows, self.b.lens)):
            pos[self.b.start[s]:self.b.start[s + 1]] = np.arange(m - r, m)
        return pos

    def check(self, got):
        kc, ks, vc, vs = got
        pos = self.positions()
        # values: every byte, of new, old, rescaled and untouched slots
        ec, es = R.append(self.vc, self.vs, self.b, self.v.astype(np.float64))
        assert np.array_equal(vs, es, equal_nan=True) and np.array_equal(vc, ec)
        plain = self.rot == 0 and self.w is None
        kx = R.norm_rope(self.k, np.maximum(pos, 0), self.f, self.rot, self.pairs, self.w)
        ec, es = R.append(self.kc, self.ks, self.b, kx)
        assert np.array_equal(ks, es, equal_nan=True)
        if plain:
            assert np.array_equal(kc, ec)
            return
        new = self.new_slots()
        assert np.array_equal(kc[~new], ec[~new])  # old, rescaled and untouched slots
        tol = turn_tol(self.k, self.rot, self.pairs, self.w)
        P = self.b.P
        for s, (r, m) in enumerate(zip(self.b.rows, self.b.lens)):
            for t in range(max(m - r, 0), m if r else 0):
                page, row = self.b.table[s, t // P], self.b.start[s] + r - m + t
                if not 0 <= page < kc.shape[0]:
                    continue
                sc = ks[page].astype(np.float64)[:, None]
                got_v, x = R.VALUES[kc[page, :, t % P]] * sc, kx[row]
                half = np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * sc)
                assert np.all(np.abs(got_v - x) <= half + tol[row] * (1 + 2.0 ** -4))

    def new_slots(self):
        P = self.b.P
        new = np.zeros(self.kc.shape, bool)
        for s, (r, m) in enumerate(zip(self.b.rows, self.b.lens)):
            for t in range(max(m - r, 0), m if r else 0):
                if 0 <= self.b.table[s, t // P] < new.shape[0]:
                    new[self.b.table[s, t // P], :, t % P] = True
        return new


@pytest.mark.parametrize("d,P,heads,lens,rows,rot,pairs,norm,vhalf,hq", [
    (64, 16, 2, [1], [1], 64, False, False, False, 0), (128, 16, 8, [17, 0, 40, 16], [1, 0, 1, 1], 128, False, True, True, 16),
    (128, 32, 3, [31, 32, 33, 100], [31, 1, 2, 0], 64, True, False, False, 6), (256, 64, 2, [65, 130], [65, 7], 256, False, True, True, 4),
    (64, 64, 1, [200, 64, 63], [137, 64, 63], 0, False, False, False, 3), (256, 16, 1, [50], [33], 0, False, False, True, 0),
    (128, 64, 8, [640, 5, 129], [600, 5, 3], 128, False, True, False, 0), (64, 32, 5, [97, 0, 1], [96, 0, 1], 32, True, True, True, 5),
    (256, 32, 4, [300, 17], [299, 17], 8, True, False, False, 8)])
def test_append(ctx, d, P, heads, lens, rows, rot, pairs, norm, vhalf, hq):
    rng = np.random.default_rng(d + P + heads + len(lens))
    c = Case(ctx, rng, lens, rows, P, d, heads, rot, pairs, norm, vhalf, hq, behind=2)
    c.check(c.run())
    if hq:
        got = c.io[3].download(np.float32).reshape(c.q.shape)
        pos = c.positions()
        assert np.all(got[pos < 0] == 7)  # rows behind the last sequence
        # the same bits as the operator of its own
        qb, pb = ctx.upload(c.q), ctx.upload(np.maximum(pos, 0).astype(np.int32))
        h = HeadRows(qb, hq, hq * d)
        QKNormRopeKernel(ctx).encode(None, h, None, h, None, pb, c.b.total, d, c.args[4], c.more["kNorm"])
        ctx.synchronize()
        assert np.array_equal(got[pos >= 0], qb.download(np.float32).reshape(c.q.shape)[pos >= 0])


def test_many_sequences(ctx):
    """More sequences than a wave has lanes, so that a row's sequence is found in several steps."""
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(1, 50, 150)]
    rows = [int(min(n, rng.integers(0, 4))) for n in lens]
    c = Case(ctx, rng, lens, rows, 16, 64, 1, 64, False, False, False, hq=2, behind=1)
    c.check(c.run())
    got = c.io[3].download(np.float32).reshape(c.q.shape)
    pos = c.positions()
    exp = R.norm_rope(c.q, np.maximum(pos, 0), c.f, 64, False)
    assert np.all(got[pos < 0] == 7)
    assert np.all(np.abs(got - exp)[pos >= 0] <= turn_tol(c.q, 64, False, None)[pos >= 0])


@pytest.mark.parametrize("d,P", [(64, 16), (128, 64)])
def test_token_by_token_is_all_at_once(ctx, d, P):
    """A prompt in one call and token by token: the same scales, and the same values but where a code passed through e4m3's
    subnormals, whose steps are 2^-9 of the scale that it had then."""
    rng = np.random.default_rng(d)
    n = 2 * P + 5
    one = Case(ctx, rng, [n], [n], P, d, 2, spread=2.0)
    a = one.run()
    one.check(a)
    for t in range(n):
        step = KV8Batch(one.batch.buffers[0], ctx.upload(np.array([t + 1], np.int32)), ctx.upload(np.array([0, 1], np.int32)),
                        1, one.b.stride, 1, 1, n)
        if t == 0:
            for b, src in zip(one.bufs, (one.kc, one.vc, one.ks, one.vs)):
                b.upload(src)
        row = [HeadRows(b.view(4 * t * 2 * d), 2, 2 * d) for b in one.io[:2]]
        KV8AppendKernel(ctx).encode(None, one.cache, step, *row, one.args[4])
        ctx.synchronize()
    b = one.read()
    assert np.array_equal(a[1], b[1], equal_nan=True) and np.array_equal(a[3], b[3], equal_nan=True)
    for x, y, sc in ((a[0], b[0], a[1]), (a[2], b[2], a[3])):
        new = one.new_slots()
        x, y = R.VALUES[x][new], R.VALUES[y][new]
        assert np.all((np.abs(x - y) <= 2.0 ** -9) & ((x == y) | (np.abs(x) <= 2.0 ** -6)))


def test_scales(ctx):
    """A block's scale by its largest finite magnitude: the border at 448 times a power of two, zeros, tiny and huge values,
    NaN and infinities, which take the NaN code and leave the scale alone."""
    P, d = 16, 64
    peaks = [448.0, np.nextafter(np.float32(448.0), np.float32(1e9)), 449.0, 1.75, 1.7500001, 0.0, 1e-45, 2.0 ** -120, 3e38, 1.0]
    rng = np.random.default_rng(1)
    c = Case(ctx, rng, [1] * len(peaks), [1] * len(peaks), P, d, 1, rot=0)
    for i, p in enumerate(peaks):
        for x in (c.k, c.v):
            x[i] = (np.float32(p) * rng.uniform(-1, 1, (1, d)).astype(np.float32))
            x[i, 0, 3] = p
    c.v[9, 0, 5], c.v[9, 0, 6], c.v[9, 0, 7] = np.nan, np.inf, -np.inf
    got = c.run()
    c.check(got)
    page = c.b.table[:, 0]
    assert list(got[3][page[:7], 0]) == [1.0, 2.0, 2.0, 2.0 ** -8, 2.0 ** -7, 2.0 ** -100, 2.0 ** -100]
    assert got[3][page[9], 0] == 2.0 ** -8
    assert np.all((got[2][page[9], 0, 0, 5:8] & 0x7f) == 0x7f)


def test_non_finite_keys_under_norm_and_rotation(ctx):
    """An infinite element makes its head's root infinite: it becomes NaN, and the pair it turns with, the others zeros; a NaN
    takes the whole head.  Other heads and tokens keep their codes, and the scales ignore what is not finite."""
    P, d = 16, 64
    rng = np.random.default_rng(8)
    c = Case(ctx, rng, [5], [5], P, d, 3, norm=True)
    c.k[1, 0, 7], c.k[2, 1, 9], c.k[3, 2, 3] = np.inf, np.nan, -np.inf
    kc, ks, _, _ = c.run()
    page = c.b.table[0, 0]
    clean = c.k.copy()
    for r, h in ((1, 0), (2, 1), (3, 2)):
        clean[r, h] = 0
    x = R.norm_rope(clean, np.arange(5), c.f, d, False, c.w)
    for h in range(3):
        assert ks[page, h] == R.block_scale(np.abs(x[:, h]).max())
    got = R.VALUES[kc[page, :, :5]].transpose(1, 0, 2)
    for r, h, e in ((1, 0, 7), (3, 2, 3)):
        pair = [e, e + d // 2]
        assert np.all(np.isnan(got[r, h, pair])) and np.all(np.delete(got[r, h], pair) == 0)
    assert np.all(np.isnan(got[2, 1]))
    for r in range(5):
        for h in range(3):
            if (r, h) not in ((1, 0), (2, 1), (3, 2)):
                assert np.array_equal(kc[page, h, r], R.to_e4m3(x[r, h] / ks[page, h]))


def test_growth_keeps_exact_codes(ctx):
    """A block of normal codes grows by 2^6 and keeps its values exactly; NaN codes stay."""
    P, d = 32, 64
    rng = np.random.default_rng(2)
    c = Case(ctx, rng, [20], [1], P, d, 1, rot=0)
    page = c.b.table[0, 0]
    c.vc[page, 0] = (rng.integers(0x40, 0x7f, (P, d)) | (rng.integers(0, 2, (P, d)) << 7)).astype(np.uint8)
    c.vc[page, 0, 4, 9] = 0x7f
    c.vs[page] = 2.0 ** -6
    c.v[0, 0, 0] = 400.0
    before = R.VALUES[c.vc[page, 0, :19]] * 2.0 ** -6
    got = c.run()
    assert got[3][page, 0] == 1.0
    assert np.array_equal(R.VALUES[got[2][page, 0, :19]], before, equal_nan=True)
    assert np.isnan(R.VALUES[got[2][page, 0, 4, 9]])


def test_pages_outside_the_pool_and_rows_without_a_place(ctx):
    """Entries of the table outside the pool, more rows than tokens, lengths beyond the table and the bounds, row starts beyond
    the rows: what has no place is not written, the rest is; the pool around stays."""
    P, d = 16, 128
    rng = np.random.default_rng(3)
    c = Case(ctx, rng, [40, 3, 33], [40, 3, 2], P, d, 2)
    c.b.table[0, 1] = c.b.pages
    c.b.table[2, 2] = -1
    c.check(c.run())
    # five rows of a sequence of three tokens: the first two have no position
    c = Case(ctx, rng, [3], [5], P, d, 2, hq=3)
    c.check(c.run())
    q = c.io[3].download(np.float32).reshape(c.q.shape)
    assert np.all(q[:2] == 7) and not np.any(q[2:] == 7)
    # a length beyond max_kv_len, then beyond the table, counts as the bound; rows beyond max_rows are left alone
    for bound, most in ((20, 4), (1000, 4), (1000, 2)):
        c = Case(ctx, rng, [32], [4], P, d, 2, hq=1)
        c.b.lens = [1 << 30]
        up = c.b.upload(ctx, max_rows=most, max_len=bound)
        got = c.run(batch=up)
        c.b.lens, c.b.rows = [min(32, bound)], [most]
        c.b.start[1] = most
        c.check(got)
        q = c.io[3].download(np.float32).reshape(c.q.shape)
        assert np.all(q[most:] == 7) and not np.any(q[:most] == 7)
    c = Case(ctx, rng, [9, 9], [3, 2], P, d, 1)
    up = c.b.upload(ctx)
    up.buffers[2].upload(np.array([-7, 3, 1 << 30], np.int32))
    c.check(c.run(batch=up))


def test_empty_batches_do_nothing(ctx):
    rng = np.random.default_rng(4)
    c = Case(ctx, rng, [5, 20], [0, 0], 16, 64, 1, behind=3, hq=1)
    got = c.run(batch=c.b.upload(ctx, max_rows=3))
    for g, e in zip(got, (c.kc, c.ks, c.vc, c.vs)):
        assert np.array_equal(g, e, equal_nan=True)
    assert np.all(c.io[3].download(np.float32) == 7)


def test_cache_beyond_32_bits(ctx):
    """The last pages of a pool of more than 2^32 code bytes."""
    P, d, heads = 64, 256, 2
    pages = (1 << 32) // (P * d * heads) + 40
    rng = np.random.default_rng(6)
    c = Case(ctx, rng, [70], [70], P, d, heads, rot=0)
    codes = [ctx.alloc(pages * heads * P * d) for _ in range(2)]
    scales = [ctx.alloc(4 * pages * heads) for _ in range(2)]
    cache = KV8Cache(*codes, *scales, pages, heads, P, d)
    c.b.table[0] = [pages - 1, pages - 3]
    io = [ctx.upload(c.k), ctx.upload(c.v)]
    KV8AppendKernel(ctx).encode(None, cache, c.b.upload(ctx), HeadRows(io[0], heads, heads * d), HeadRows(io[1], heads, heads * d),
                                Rope(None, 0))
    ctx.synchronize()
    for x, cb, sb in ((c.k, codes[0], scales[0]), (c.v, codes[1], scales[1])):
        for page, a, b in ((pages - 1, 0, 64), (pages - 3, 64, 70)):
            got = cb.download(np.uint8, heads * P * d, page * heads * P * d).reshape(heads, P, d)
            sc = sb.download(np.float32, heads, 4 * page * heads)
            for h in range(heads):
                assert sc[h] == R.block_scale(np.abs(x[a:b, h]).max())
                assert np.array_equal(got[h, :b - a], R.to_e4m3(x[a:b, h].astype(np.float64) / sc[h]))
    for b in codes + scales:
        b.free()
