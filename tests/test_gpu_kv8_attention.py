"""Attention over the 8-bit paged cache against a plain 64-bit form, with the
elementwise bound that kv8_ref.attend derives."""
import numpy as np
import pytest

import kv8_ref as R
from edgerunner_amd import Capture, EncodingFailed, HeadRows, KV8AttentionKernel, KV8Cache

pytestmark = pytest.mark.gpu


def pool(rng, pages, heads, P, d, nans=True):
    """Codes of every kind but NaN in both, scales over a few powers of two."""
    c = rng.integers(0, 256, (pages, heads, P, d)).astype(np.uint8)
    c = np.where((c & 0x7f) > 0x68, c & 0xdf, c).astype(np.uint8)  # values up to 32: scores stay moderate
    s = (2.0 ** rng.integers(-6, -3, (pages, heads))).astype(np.float32)
    return c, s


class Case:
    def __init__(self, ctx, seed, lens, rows, P, d, hq, hkv, behind=0, qscale=1.0):
        rng = np.random.default_rng(seed)
        self.ctx, self.d, self.hq, self.rng = ctx, d, hq, rng
        self.b = R.Batch(rng, lens, rows, P, behind=behind)
        self.kc, self.ks = pool(rng, self.b.pages, hkv, P, d)
        self.vc, self.vs = pool(rng, self.b.pages, hkv, P, d)
        self.scale = d ** -0.5
        self.q = (rng.standard_normal((self.b.total, hq, d)) * qscale).astype(np.float32)
        # bytes behind the last token and pages of nobody are NaN codes and NaN scales
        owned = np.zeros(self.b.pages, bool)
        for s, m in enumerate(lens):
            for p in range(-(-m // P)):
                owned[self.b.table[s, p]] = True
                used = min(P, m - p * P)
                for c in (self.kc, self.vc):
                    c[self.b.table[s, p], :, used:] = 0x7f
        self.kc[~owned], self.vc[~owned], self.ks[~owned], self.vs[~owned] = 0xff, 0x7f, np.nan, np.nan

    def upload(self, pad=0):
        ctx, d = self.ctx, self.d
        self.pad = pad
        self.bufs = [ctx.upload(a) for a in (self.kc, self.vc, self.ks, self.vs)]
        self.cache = KV8Cache(*self.bufs, self.kc.shape[0], self.kc.shape[1], self.kc.shape[2], d)
        wide = np.zeros((self.b.total, self.hq * d + pad), np.float32)
        wide[:, :self.hq * d] = self.q.reshape(self.b.total, -1)
        self.qb = ctx.upload(wide)
        self.qr = HeadRows(self.qb, self.hq, self.hq * d + pad)

    def run(self, half=False, window=0, pad=0, batch=None, **over):
        ctx, d = self.ctx, self.d
        self.upload(pad)
        batch = batch or self.b.upload(ctx)
        kern = KV8AttentionKernel(ctx)
        ws = ctx.alloc(max(16, kern.workspaceBytes(self.cache, batch, self.hq)))
        ws.upload(np.full(ws.length // 4, np.nan, np.float32))  # whatever scratch holds must not matter
        t = np.uint16 if half else np.float32
        fill = np.uint16(0x1234) if half else np.float32(7)
        ob = ctx.upload(np.full((self.b.total, self.hq * d + pad), fill, t))
        kern.encode(None, self.cache, batch, self.qr, HeadRows(ob, self.hq, self.hq * d + pad), self.scale, window=window,
                    workspace=ws, outBF16=half, **over)
        ctx.synchronize()
        got = ob.download(t).reshape(self.b.total, self.hq * d + pad)
        assert np.all(got[:, self.hq * d:] == fill)
        self.raw = got[:, :self.hq * d].reshape(self.b.total, self.hq, d)
        self.fill = fill
        return (R.bf16_to_f32(self.raw) if half else self.raw).astype(np.float64)

    def check(self, got, half=False, window=0):
        exp, tol = R.attend(self.kc, self.ks, self.vc, self.vs, self.b, self.q, self.scale, window, half)
        nobody = np.ones(self.b.total, bool)
        for s in range(len(self.b.lens)):
            nobody[self.b.start[s]:self.b.start[s] + self.b.rows[s]] = False
        assert np.all(self.raw[nobody] == self.fill)
        err, tol = np.abs(got - exp)[~nobody], tol[~nobody]
        assert not np.isnan(err).any()
        assert np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())
        empty = (tol == 0).all((1, 2))
        assert np.all(got[~nobody][empty] == 0)


# one row a sequence, lengths about the 16-, 32- and 64-token borders
EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 95, 96, 127, 128, 129, 160, 200]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv", [(64, 16, 14, 2), (64, 64, 3, 3), (128, 16, 8, 2), (128, 32, 16, 1), (128, 64, 5, 5),
                                        (256, 16, 6, 2), (256, 64, 4, 1), (128, 16, 34, 2), (64, 32, 40, 1), (256, 32, 24, 1)])
def test_one_row_each(ctx, d, P, hq, hkv, half):
    c = Case(ctx, d + P + hq, EDGES + [0], [1] * len(EDGES) + [0], P, d, hq, hkv, behind=2)
    c.check(c.run(half), half)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("window", [0, 1, 7, 16, 50, 64, 100])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows", [
    (64, 16, 4, 2, [70, 33, 0, 5, 130], [5, 8, 0, 5, 1]), (128, 32, 2, 1, [140, 8, 64], [8, 8, 2]),
    (256, 64, 3, 3, [67, 128, 1], [3, 16, 1]), (128, 16, 4, 2, [150, 77, 0, 40], [150, 33, 0, 9]),
    (64, 64, 7, 1, [131, 90], [60, 90]), (256, 32, 4, 2, [100, 65, 17], [37, 65, 17]), (64, 32, 1, 1, [300], [290])])
def test_rows_and_windows(ctx, d, P, hq, hkv, lens, rows, window, half):
    c = Case(ctx, d + window, lens, rows, P, d, hq, hkv, behind=1)
    c.check(c.run(half, window), half, window)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window", [
    (128, 64, 4, 1, [5000], [1], 0), (64, 16, 2, 2, [3001, 100, 0, 1500], [1, 1, 0, 1], 0), (256, 32, 2, 1, [2500, 700], [3, 1], 0),
    (128, 16, 4, 2, [4000, 900], [2, 2], 1000), (128, 32, 6, 2, [2100, 1200, 64], [40, 20, 64], 0),
    (64, 64, 8, 1, [3000], [100], 700), (256, 16, 4, 2, [1700, 130], [30, 1], 0)])
def test_split_along_the_cache(ctx, d, P, hq, hkv, lens, rows, window, half):
    """Few workgroups and long caches: pieces and the join, short sequences of the same batch leaving pieces empty."""
    c = Case(ctx, d + P, lens, rows, P, d, hq, hkv)
    kern = KV8AttentionKernel(ctx)
    c.upload()
    assert kern.workspaceBytes(c.cache, c.b.upload(ctx), hq) > 0
    c.check(c.run(half, window), half, window)


@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window", [
    (64, 16, 8, 8, [9000, 30, 0, 7000, 4500, 1, 700], [1, 1, 0, 1, 1, 1, 1], 0),
    (64, 32, 16, 8, [12000, 64, 128, 6000, 2000], [2, 1, 8, 3, 5], 0),
    (128, 64, 16, 8, [20000, 500], [1, 2], 0), (256, 64, 4, 4, [11000, 7000, 100], [1, 1, 4], 0),
    (64, 64, 8, 8, [30000, 20000, 3000], [1, 3, 2], 9000)])
def test_shared_evenly(ctx, d, P, hq, hkv, lens, rows, window):
    """Enough tokens that workgroups' shares begin and end inside sequences and span several heads and sequences."""
    c = Case(ctx, d + len(lens), lens, rows, P, d, hq, hkv, behind=1)
    c.check(c.run(window=window), window=window)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window", [
    (64, 16, 7, 1, [5000, 300, 0, 1800], [9, 2, 0, 5], 0), (128, 64, 8, 2, [6000, 2000], [16, 3], 0),
    (256, 32, 8, 1, [3000, 900], [16, 16], 0), (128, 32, 24, 1, [4000, 40], [2, 2], 1500),
    (64, 64, 3, 3, [9000, 70, 500], [21, 20, 1], 0), (256, 16, 4, 2, [2000], [32], 300), (128, 16, 17, 1, [2600, 17], [1, 3], 0),
    (256, 64, 6, 2, [1100, 1064], [43, 5], 1)])
def test_blocks_of_columns(ctx, d, P, hq, hkv, lens, rows, window, half):
    """Several blocks of 16 columns to a sequence and head, the last one short, in shares that begin and end inside them."""
    c = Case(ctx, d + P + hq, lens, rows, P, d, hq, hkv, behind=1)
    c.check(c.run(half, window), half, window)


def test_blocks_of_many_sequences(ctx):
    """Sequences with one to four blocks of columns among each other, some empty, more of them than a wave has lanes."""
    rng = np.random.default_rng(70)
    for most in (600, 2500):
        lens = [int(x) for x in rng.integers(0, most, 70)]
        lens[3], lens[69] = 0, most
        rows = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 21, 70))]
        c = Case(ctx, 71, lens, rows, 64, 64, 6, 2)
        c.check(c.run())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window", [
    (256, 16, 8, 1, [1700, 130], [30, 1], 0), (256, 64, 4, 2, [2500, 90], [70, 90], 900), (256, 32, 4, 1, [100, 65], [40, 33], 0),
    (256, 32, 4, 1, [100, 65], [40, 33], 30), (128, 64, 20, 1, [2000, 700], [4, 1], 0)])
def test_many_columns(ctx, d, P, hq, hkv, lens, rows, window, half):
    """More columns than are taken 16 at a time."""
    c = Case(ctx, d + P + hq, lens, rows, P, d, hq, hkv)
    c.check(c.run(half, window), half, window)


@pytest.mark.parametrize("many", [150, 64, 65])
def test_shared_between_many_sequences(ctx, many):
    """More sequences than a wave has lanes, some of them empty, in aligned and in even shares."""
    rng = np.random.default_rng(many)
    for most in (600, 4000):
        lens = [int(x) for x in rng.integers(0, most, many)]
        lens[many // 2] = 0
        lens[-1] = most
        rows = [min(n, 1) for n in lens]
        c = Case(ctx, many, lens, rows, 64, 64, 2, 2)
        c.check(c.run())


# A lone token's weight is 2^(7 + e), e the rounding of its reference less 7; the sum holds it in fp32, the product with the
# value rounded to two fp16 terms (2^-22 of it), and the quotient rounds three times (each 2^-24): the value comes back to
LONE = 2.0 ** -22 + 3 * 2.0 ** -24


@pytest.mark.parametrize("hq", [1, 2])
def test_values_pass(ctx, hq):
    """A lone visible token has weight 1: every code times every scale comes out, to the weight's own rounding."""
    d = 256
    c = Case(ctx, 1, [1], [1], 16, d, hq, 1)
    page = c.b.table[0, 0]
    codes = np.arange(256, dtype=np.uint8)
    codes[(codes & 0x7f) == 0x7f] = 0
    c.vc[page, 0, 0] = codes
    for e in (-100, -30, -3, 0, 5, 60):
        c.vs[page, 0] = 2.0 ** e
        got = c.run()
        exp = R.VALUES[codes] * 2.0 ** e
        assert np.all(np.abs(got[0, 0] - exp) <= LONE * np.abs(exp)), e


def test_rows_of_many_columns_pass_values(ctx):
    d = 128
    c = Case(ctx, 2, [1] * 3, [1] * 3, 16, d, 40, 1)
    for s in range(3):
        page = c.b.table[s, 0]
        c.vc[page, 0, 0] = np.arange(s * 40, s * 40 + 128, dtype=np.uint8) % 0x7f
        c.vs[page, 0] = 2.0 ** (20 * s - 20)
    got = c.run()
    for s in range(3):
        page = c.b.table[s, 0]
        exp = R.VALUES[c.vc[page, 0, 0]] * np.float64(c.vs[page, 0])
        assert np.all(np.abs(got[s] - exp) <= LONE * np.abs(exp))


@pytest.mark.parametrize("hq,hkv,rows", [(4, 2, [1, 1]), (4, 2, [70, 30])])
def test_blocks_of_very_different_scales(ctx, hq, hkv, rows):
    """Keys and values whose blocks' scales lie up to 2^20 apart, in ascending, descending and mixed order: the bound is one on
    the largest block that a row sees, whose values an fp32 sum rounds by as much."""
    c = Case(ctx, 3, [400, 300], rows, 16, 64, hq, hkv)
    for s in range(2):
        for p in range(c.b.stride):
            if c.b.table[s, p] >= 0:
                c.vs[c.b.table[s, p]] = 2.0 ** ((p if s == 0 else -p) % 21 - 10)
    got = c.run()
    exp, tol = R.attend(c.kc, c.ks, c.vc, c.vs, c.b, c.q, c.scale)
    # a code loses nothing down to 2^-22 of the largest scale
    assert np.all(np.abs(got - exp) <= tol)


@pytest.mark.parametrize("rows", [[1, 1], [6, 3], [25, 10], [80, 40]])
@pytest.mark.parametrize("hq,hkv", [(2, 1), (4, 4)])
def test_non_finite_places(ctx, hq, hkv, rows):
    """NaN codes in keys and values of hidden tokens (later ones, ones before the window, bytes behind the last) leave a row
    alone; a visible one makes its row, or that element of it, NaN, and so does a query that is not finite."""
    window = 40
    c = Case(ctx, 4, [150, 90], rows, 16, 64, hq, hkv)
    clean_v, clean_k = c.vc.copy(), c.kc.copy()
    where = {"v": [(0, 149 - rows[0] // 2, 5), (1, 20, 3), (0, 100, 60)], "k": [(1, 89 - rows[1] // 3, 9), (0, 3, 1)]}
    for n, places in where.items():
        for s, t, e in places:
            (c.vc if n == "v" else c.kc)[c.b.table[s, t // 16], :, t % 16, e] = 0xff
    got = c.run(window=window)
    exp, tol = R.attend(clean_k, c.ks, clean_v, c.vs, c.b, c.q, c.scale, window)
    for s in range(2):
        for i in range(rows[s]):
            r, pos = c.b.start[s] + i, c.b.lens[s] - rows[s] + i
            see = lambda t: pos - window < t <= pos  # noqa: E731
            nan_row = any(z == s and see(t) for z, t, _ in where["k"])
            bad = [e for z, t, e in where["v"] if z == s and see(t)]
            if nan_row:
                assert np.all(np.isnan(got[r]))
                continue
            good = np.ones(64, bool)
            good[bad] = False
            assert np.all(np.isnan(got[r][:, bad]))
            assert np.all(np.abs(got[r][:, good] - exp[r][:, good]) <= tol[r][:, good])
    for bad in (np.nan, np.inf, -np.inf):
        c.vc, c.kc = clean_v.copy(), clean_k.copy()
        c.q[0, 1, 17] = bad
        got = c.run()
        assert np.all(np.isnan(got[0, 1]))
        c.q[0, 1, 17] = 0.5
        exp, tol = R.attend(c.kc, c.ks, c.vc, c.vs, c.b, c.q, c.scale)
        keep = np.ones(got.shape[:2], bool)
        keep[0, 1] = False
        assert np.all(np.abs(got - exp)[keep] <= tol[keep])


@pytest.mark.parametrize("rows", [[1, 2, 1], [40, 30, 20]])
def test_large_and_tiny_queries(ctx, rows):
    """Queries of 2^+-60 and zeros: the power of two taken off a query goes back into its scores."""
    c = Case(ctx, 5, [60, 33, 20], rows, 32, 128, 3, 1)
    c.q[0] *= 2.0 ** -60
    c.q[c.b.start[1]] *= 0
    c.q[c.b.start[2]] *= 2.0 ** 60
    c.ks[:] = np.where(np.isnan(c.ks), c.ks, 2.0 ** -6)
    got = c.run()
    exp, tol = R.attend(c.kc, c.ks, c.vc, c.vs, c.b, c.q, c.scale)
    big = c.b.start[2]
    keep = np.arange(c.b.total) != big
    assert np.all(np.abs(got - exp)[keep] <= tol[keep])
    assert np.all(np.abs(got[big] - exp[big]) <= 1e-5 * np.abs(exp[big]) + 1e-30)  # one token has all the weight


def test_negative_and_zero_scale(ctx):
    for scale in (-0.3, 0.0, 1e-30):
        for rows in ([3, 1], [50, 30]):
            c = Case(ctx, 6, [80, 45], rows, 16, 64, 2, 1)
            c.scale = scale
            c.check(c.run())


@pytest.mark.parametrize("rows", [[1, 1, 2], [33, 20, 2]])
def test_pages_outside_the_pool(ctx, rows):
    """Tokens whose table entry lies outside the pool count as not there; a row with no others gets zeros."""
    c = Case(ctx, 7, [100, 50, 2], rows, 16, 64, 4, 1)
    c.b.table[0, 1] = c.b.pages
    c.b.table[0, 4] = -2 ** 31
    c.b.table[2, 0] = 2 ** 31 - 1
    got = c.run()
    c.check(got)
    assert np.all(got[c.b.start[2]:] == 0)


@pytest.mark.parametrize("hq", [2, 20])
def test_rows_without_a_place(ctx, hq):
    """More rows than tokens; lengths beyond the bounds and the table; rows beyond max_rows."""
    c = Case(ctx, 8, [3, 20], [6, 4], 16, 64, hq, 1, behind=2)
    c.check(c.run())
    for bound, most in ((20, 4), (1000, 4), (1000, 2)):
        c = Case(ctx, 9, [32], [4], 16, 64, hq, 1)
        up_b = R.Batch(np.random.default_rng(0), [32], [4], 16)
        up_b.table = c.b.table
        up_b.lens = [1 << 30]
        batch = up_b.upload(ctx, max_rows=most, max_len=bound)
        got = c.run(batch=batch)
        c.b.lens, c.b.rows = [min(32, bound)], [most]
        c.check(got)


@pytest.mark.parametrize("pad", [1, 4])
@pytest.mark.parametrize("half", [False, True])
def test_strides(ctx, pad, half):
    for rows in ([2, 1], [40, 30]):
        c = Case(ctx, 10, [70, 40], rows, 32, 128, 6, 2)
        c.check(c.run(half, pad=pad), half)


def test_shared_pages(ctx):
    """Two sequences over the same prefix pages."""
    c = Case(ctx, 11, [96, 96, 40], [1, 17, 1], 32, 64, 2, 1)
    c.b.table[1, :2] = c.b.table[0, :2]
    c.check(c.run())


def test_short_workspace_is_refused(ctx):
    c = Case(ctx, 12, [4000], [1], 16, 64, 2, 1)
    c.upload()
    kern, batch = KV8AttentionKernel(ctx), c.b.upload(ctx)
    out = HeadRows(ctx.alloc(4 * 2 * 64), 2, 128)
    with pytest.raises(EncodingFailed):
        kern.encode(None, c.cache, batch, c.qr, out, 0.1)
    with pytest.raises(EncodingFailed):
        kern.encode(None, c.cache, batch, c.qr, out, 0.1, workspace=ctx.alloc(64))


def test_workspace_covers_every_window(ctx):
    """The bytes asked for do not depend on the window, and suffice for any."""
    c = Case(ctx, 13, [3000], [1], 16, 64, 2, 1)
    exp0 = None
    for window in (0, 1, 63, 64, 65, 500, 1000, 1025, 2900, 3000, 10 ** 6, 2 ** 32 - 1):
        got = c.run(window=window)
        if window in (0, 3000, 10 ** 6, 2 ** 32 - 1):
            exp0 = R.attend(c.kc, c.ks, c.vc, c.vs, c.b, c.q, c.scale, 0) if exp0 is None else exp0
            assert np.all(np.abs(got - exp0[0]) <= exp0[1])
        else:
            c.check(got, window=window)


@pytest.mark.parametrize("rows", [20, 90])
def test_workspace_covers_every_window_of_many_rows(ctx, rows):
    c = Case(ctx, 13, [3000], [rows], 16, 64, 2, 1)
    for window in (0, 1, 64, 65, 500, 1025, 2900, 3000, 2 ** 32 - 1):
        c.check(c.run(window=window), window=min(window, 3000))


def test_repeats_are_the_same_bits(ctx):
    for rows, hq in (([1, 1], 4), ([90, 30], 4), ([1, 1], 40), ([20, 7], 4)):
        c = Case(ctx, 14, [1500, 700], rows, 64, 128, hq, 2)
        first = c.run()
        for _ in range(3):
            assert np.array_equal(c.run(), first)


def test_captured_and_replayed_with_later_lengths(ctx):
    """A recorded call follows the lengths and tables of its replay; eager work stands between the replays."""
    for rows, hq in (([1, 1], 4), ([20, 10], 2), ([32, 30], 4)):
        c = Case(ctx, 15, [900, 300], rows, 16, 64, hq, 1)
        c.upload()
        batch = c.b.upload(ctx)
        kern = KV8AttentionKernel(ctx)
        ws = ctx.alloc(max(16, kern.workspaceBytes(c.cache, batch, hq)))
        ob = ctx.alloc(4 * c.q.size)
        out = HeadRows(ob, hq, hq * 64)
        st = ctx.stream()
        with Capture(ctx, st) as cap:
            kern.encode(st, c.cache, batch, c.qr, out, c.scale, workspace=ws)
        c.fill = np.float32(7)
        held = (c.bufs, c.qb, c.cache, c.qr)  # what the graph is bound to stays allocated; run() makes buffers of its own
        for lens in ([900, 300], [33, 300], [900, 30], [64, 64]):
            c.b.lens = lens
            batch.buffers[1].upload(np.array(lens, np.int32))
            ob.upload(np.full(c.q.size, 7, np.float32))
            cap.graph.launch(st)
            st.synchronize()
            got = ob.download(np.float32).reshape(c.q.shape)
            c.raw = got
            c.check(got.astype(np.float64))
            eager = c.run(batch=c.b.upload(ctx, max_len=900))  # the recorded call's bounds, so its cuts and bits
            assert np.array_equal(eager.astype(np.float32), got)
        cap.graph.destroy()
        del held
        st.destroy()


def test_two_streams_with_their_own_workspaces(ctx):
    cases = [Case(ctx, 16 + i, [2000 + 300 * i], [1], 32, 128, 8, 2) for i in range(2)]
    kern, streams, outs = KV8AttentionKernel(ctx), [ctx.stream(), ctx.stream()], []
    for c in cases:
        c.upload()
        batch = c.b.upload(ctx)
        outs.append((batch, ctx.alloc(kern.workspaceBytes(c.cache, batch, 8)), ctx.alloc(4 * c.q.size)))
    for _ in range(4):
        for c, st, (batch, ws, ob) in zip(cases, streams, outs):
            kern.encode(st, c.cache, batch, c.qr, HeadRows(ob, 8, 8 * 128), c.scale, workspace=ws)
    for c, st, (_, _, ob) in zip(cases, streams, outs):
        st.synchronize()
        got = ob.download(np.float32).reshape(c.q.shape)
        exp, tol = R.attend(c.kc, c.ks, c.vc, c.vs, c.b, c.q, c.scale)
        assert np.all(np.abs(got - exp) <= tol)
        st.destroy()


@pytest.mark.parametrize("rows", [1, 30, 80])
def test_cache_beyond_32_bits(ctx, rows):
    """A sequence in the last pages of a pool of more than 2^32 code bytes."""
    P, d, heads = 64, 256, 2
    pages = (1 << 32) // (P * d * heads) + 40
    c = Case(ctx, 18, [150], [rows], P, d, 4, heads)
    c.upload()
    codes = [ctx.alloc(pages * heads * P * d) for _ in range(2)]
    scales = [ctx.alloc(4 * pages * heads) for _ in range(2)]
    cache = KV8Cache(*codes, *scales, pages, heads, P, d)
    far = [pages - 1, pages - 7, pages - 2]
    for p, to in enumerate(far):
        src = c.b.table[0, p]
        for b, a, size in ((codes[0], c.kc, heads * P * d), (codes[1], c.vc, heads * P * d), (scales[0], c.ks, 4 * heads),
                           (scales[1], c.vs, 4 * heads)):
            b.upload(a[src], to * size)
    batch = c.b.upload(ctx)
    batch.buffers[0].upload(np.array(far, np.int32))
    ob = ctx.alloc(4 * c.q.size)
    kern = KV8AttentionKernel(ctx)
    ws = ctx.alloc(max(16, kern.workspaceBytes(cache, batch, 4)))
    kern.encode(None, cache, batch, c.qr, HeadRows(ob, 4, 4 * d), c.scale, workspace=ws)
    ctx.synchronize()
    got = ob.download(np.float32).reshape(c.q.shape)
    exp, tol = R.attend(c.kc, c.ks, c.vc, c.vs, c.b, c.q, c.scale)
    assert np.all(np.abs(got - exp) <= tol)
    for b in codes + scales:
        b.free()
