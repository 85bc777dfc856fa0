"""Attention over the 8-bit cache under masks (sinks, windows, trees of drafts)
against a plain 64-bit form, with the elementwise bound that kv8_ref derives."""
import numpy as np
import pytest

import draft_ref as D
import kv8_ref as R
from edgerunner_amd import Capture, Drafts, EncodingFailed, HeadRows, KV8AttentionKernel, KV8Cache

pytestmark = pytest.mark.gpu


def pool(rng, pages, heads, P, d):
    c = rng.integers(0, 256, (pages, heads, P, d)).astype(np.uint8)
    c = np.where((c & 0x7f) > 0x68, c & 0xdf, c).astype(np.uint8)  # values up to 32: scores stay moderate
    return c, (2.0 ** rng.integers(-6, -3, (pages, heads))).astype(np.float32)


class Case:
    """masks: None (causal rows), "tree", "any" (every bit by chance, some rows empty), "none", "chain"."""

    def __init__(self, ctx, seed, lens, rows, P, d, hq, hkv, masks=None, behind=0, extra_words=0):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.d, self.hq = ctx, d, hq
        self.b = R.Batch(rng, lens, rows, P, behind=behind)
        self.kc, self.ks = pool(rng, self.b.pages, hkv, P, d)
        self.vc, self.vs = pool(rng, self.b.pages, hkv, P, d)
        self.scale = d ** -0.5
        self.q = rng.standard_normal((self.b.total, hq, d)).astype(np.float32)
        # bytes behind the last token and pages of nobody are NaN codes and NaN scales
        owned = np.zeros(self.b.pages, bool)
        for s, m in enumerate(lens):
            for p in range(-(-m // P)):
                owned[self.b.table[s, p]] = True
                for c in (self.kc, self.vc):
                    c[self.b.table[s, p], :, min(P, m - p * P):] = 0x7f
        self.kc[~owned], self.vc[~owned], self.ks[~owned], self.vs[~owned] = 0xff, 0x7f, np.nan, np.nan
        self.seen = self.drafts = None
        if masks is None:
            return
        most = max(rows)
        self.n_words = -(-most // 32) + extra_words
        self.seen, self.position = [], np.full(self.b.total, -7, np.int32)
        packed = np.full((self.b.total, self.n_words), 0xffffffff, np.uint32)
        for s, (n, m) in enumerate(zip(rows, lens)):
            parent = D.tree(rng, n, chain=masks == "chain")[0] if n else np.zeros(0, np.int32)
            bits = D.lines(parent)
            at = slice(self.b.start[s], self.b.start[s] + n)
            self.position[at] = m - n + bits.sum(1) - 1
            if masks == "any":
                bits = rng.random((n, n)) < 0.5
                bits[::3] = False
            elif masks == "none":
                bits[:] = False
            self.seen.append(bits)
            packed[at] = D.words(bits, self.n_words)
        self.sb, self.pb = ctx.upload(packed), ctx.upload(self.position)
        self.drafts = Drafts(self.sb, self.n_words, position=self.pb)

    def encode(self, out, ws, batch, half, window, sinks, stream=None):
        self.kern.encode(stream, self.cache, batch, self.qr, out, self.scale, window=window, workspace=ws, outBF16=half,
                         sinks=sinks, drafts=self.drafts)

    def upload(self, pad=0):
        self.kern = KV8AttentionKernel(self.ctx)
        self.bufs = [self.ctx.upload(a) for a in (self.kc, self.vc, self.ks, self.vs)]
        self.cache = KV8Cache(*self.bufs, self.kc.shape[0], self.kc.shape[1], self.kc.shape[2], self.d)
        wide = np.zeros((self.b.total, self.hq * self.d + pad), np.float32)
        wide[:, :self.hq * self.d] = self.q.reshape(self.b.total, -1)
        self.qb = self.ctx.upload(wide)
        self.qr = HeadRows(self.qb, self.hq, self.hq * self.d + pad)

    def scratch(self, batch):
        ws = self.ctx.alloc(max(16, self.kern.workspaceBytes(self.cache, batch, self.hq)))
        ws.upload(np.full(ws.length // 4, np.nan, np.float32))  # whatever scratch holds must not matter
        return ws

    def run(self, half=False, window=0, sinks=0, pad=0, max_len=None):
        ctx, d = self.ctx, self.d
        self.upload(pad)
        batch = self.b.upload(ctx, max_len=max_len)
        t = np.uint16 if half else np.float32
        fill = np.uint16(0x1234) if half else np.float32(7)
        ob = ctx.upload(np.full((self.b.total, self.hq * d + pad), fill, t))
        self.encode(HeadRows(ob, self.hq, self.hq * d + pad), self.scratch(batch), batch, half, window, sinks)
        ctx.synchronize()
        got = ob.download(t).reshape(self.b.total, self.hq * d + pad)
        assert np.all(got[:, self.hq * d:] == fill)
        self.raw, self.fill = got[:, :self.hq * d].reshape(self.b.total, self.hq, d), fill
        return (R.bf16_to_f32(self.raw) if half else self.raw).astype(np.float64)

    def sees(self, window, sinks):
        b = self.b
        return [D.visible(m, n, window, sinks, None if self.seen is None else self.seen[s],
                          None if self.seen is None else self.position[b.start[s]:b.start[s] + n])
                for s, (n, m) in enumerate(zip(b.rows, b.lens))]

    def check(self, got, half=False, window=0, sinks=0):
        exp, tol = D.attend(self.kc, self.ks, self.vc, self.vs, self.b, self.q, self.scale, self.sees(window, sinks), half)
        nobody = np.ones(self.b.total, bool)
        for s in range(len(self.b.lens)):
            nobody[self.b.start[s]:self.b.start[s] + self.b.rows[s]] = False
        assert np.all(self.raw[nobody] == self.fill)
        err, tol = np.abs(got - exp)[~nobody], tol[~nobody]
        assert not np.isnan(err).any()
        assert np.all(err <= tol), float((err / np.maximum(tol, 1e-300)).max())
        empty = (tol == 0).all((1, 2))
        assert np.all(got[~nobody][empty] == 0)


EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 200, 260]
SHAPES = [(64, 16, 14, 2), (64, 32, 3, 3), (64, 64, 40, 1), (128, 16, 8, 2), (128, 32, 34, 2), (128, 64, 5, 5), (256, 16, 6, 2),
          (256, 32, 4, 1), (256, 64, 24, 1)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv", SHAPES)
@pytest.mark.parametrize("window,sinks", [(1, 1), (20, 4), (64, 64), (33, 100), (300, 7), (50, 0)])
def test_one_row_each(ctx, d, P, hq, hkv, window, sinks, half):
    c = Case(ctx, d + P + hq, EDGES + [0], [1] * len(EDGES) + [0], P, d, hq, hkv, behind=2)
    c.check(c.run(half, window, sinks), half, window, sinks)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (50, 65), (100, 300), (0, 5)])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows", [
    (64, 16, 4, 2, [270, 133, 0, 5, 230], [5, 8, 0, 5, 1]), (128, 32, 2, 1, [340, 8, 164], [8, 8, 2]),
    (256, 64, 3, 3, [267, 128, 1], [3, 16, 1]), (128, 16, 4, 2, [350, 77, 0, 140], [150, 33, 0, 9]),
    (64, 64, 7, 1, [331, 190], [60, 190]), (256, 32, 4, 2, [300, 65, 217], [37, 65, 17]), (64, 32, 1, 1, [400], [290]),
    (256, 16, 8, 1, [250, 130], [130, 30]), (128, 64, 16, 2, [400, 66], [100, 66]), (64, 16, 16, 1, [400, 90], [70, 20])])
def test_rows_with_sinks(ctx, d, P, hq, hkv, lens, rows, window, sinks, half):
    c = Case(ctx, d + window, lens, rows, P, d, hq, hkv, behind=1)
    c.check(c.run(half, window, sinks), half, window, sinks)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("masks", ["tree", "any"])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window,sinks", [
    (64, 16, 4, 2, [270, 33, 0, 5, 130], [5, 8, 0, 5, 1], 0, 0), (128, 32, 2, 1, [140, 8, 64], [8, 8, 2], 20, 3),
    (256, 64, 3, 3, [67, 128, 1], [3, 16, 1], 0, 0), (128, 16, 4, 2, [350, 77, 0, 40], [150, 33, 0, 9], 0, 0),
    (64, 64, 7, 1, [331, 90], [60, 90], 70, 5), (256, 32, 4, 2, [300, 65, 17], [37, 65, 17], 40, 0),
    (64, 32, 8, 1, [300, 65], [33, 31], 100, 70), (256, 16, 8, 1, [250, 130], [130, 30], 0, 0),
    (128, 64, 16, 2, [400, 66], [64, 66], 0, 0), (64, 16, 1, 1, [97, 96, 95], [32, 64, 95], 8, 1),
    (256, 64, 2, 2, [300, 40], [65, 1], 1, 1)])
def test_trees(ctx, d, P, hq, hkv, lens, rows, window, sinks, masks, half):
    c = Case(ctx, d + P + hq, lens, rows, P, d, hq, hkv, masks, behind=1, extra_words=1)
    c.check(c.run(half, window, sinks), half, window, sinks)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,window,sinks,masks", [
    (128, 64, 4, 1, [5000], [1], 1500, 4, None), (64, 16, 2, 2, [3001, 100, 0, 1500], [1, 1, 0, 1], 700, 70, None),
    (256, 32, 2, 1, [2500, 700], [3, 1], 600, 900, None), (128, 16, 4, 2, [4000, 900], [2, 2], 1000, 1, None),
    (128, 32, 6, 2, [3100, 1200, 64], [40, 20, 64], 800, 10, None), (64, 64, 8, 1, [3000], [100], 700, 130, None),
    (256, 16, 4, 2, [1700, 130], [30, 1], 900, 5, None), (64, 64, 8, 8, [30000, 9000, 3000], [1, 3, 2], 9000, 4, None),
    (128, 64, 4, 2, [5000, 900], [26, 9], 0, 0, "tree"), (64, 16, 14, 2, [3001, 100, 0, 1500], [20, 11, 0, 64], 0, 0, "tree"),
    (256, 32, 8, 4, [2500, 700], [30, 3], 900, 70, "tree"), (128, 16, 8, 1, [4000, 900], [40, 33], 0, 0, "any"),
    (256, 64, 16, 2, [3000, 500], [64, 20], 700, 4, "tree"), (64, 32, 4, 4, [9000, 700, 60], [10, 40, 60], 0, 0, "any"),
    (128, 64, 8, 8, [6000, 2000], [5, 7], 2000, 64, "tree")])
def test_split_along_the_cache(ctx, d, P, hq, hkv, lens, rows, window, sinks, masks, half):
    """Shares and pieces that begin and end around the sinks, the window and the drafts."""
    c = Case(ctx, d + P, lens, rows, P, d, hq, hkv, masks)
    c.check(c.run(half, window, sinks), half, window, sinks)


@pytest.mark.parametrize("hq,masks", [(1, "tree"), (4, "any")])
def test_the_most_drafts(ctx, hq, masks):
    c = Case(ctx, 9, [1100, 1024, 77], [1024, 1023, 64], 64, 64, hq, 1, masks)
    c.check(c.run())


@pytest.mark.parametrize("masks", ["tree", "any", "none", None])
@pytest.mark.parametrize("hq", [1, 16])
def test_no_tokens_in_front(ctx, masks, hq):
    """Trees that begin a sequence, masks that leave every row empty, and rows in front of the first token (more rows than tokens)."""
    c = Case(ctx, 10, [33, 5, 70, 1], [33, 9, 71, 4], 16, 64, hq, 1, masks)
    c.check(c.run(window=9, sinks=2), window=9, sinks=2)
    c.check(c.run())


def test_many_sequences(ctx):
    rng = np.random.default_rng(70)
    for masks, window, sinks in ((None, 300, 20), ("tree", 0, 0), ("tree", 500, 3)):
        lens = [int(x) for x in rng.integers(0, 2500, 70)]
        lens[3], lens[69] = 0, 2500
        rows = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 21, 70))]
        c = Case(ctx, 71, lens, rows, 64, 64, 6, 2, masks)
        c.check(c.run(window=window, sinks=sinks), window=window, sinks=sinks)


@pytest.mark.parametrize("rows,hq", [([1, 1], 4), ([6, 9], 2), ([80, 40], 4)])
def test_as_plain_attention(ctx, rows, hq):
    """Sinks that reach past the window, and a chain of drafts, see what a causal row does."""
    c = Case(ctx, 12, [700, 90], rows, 32, 128, hq, 2)
    c.check(c.run(window=30, sinks=700))
    c = Case(ctx, 12, [700, 90], rows, 32, 128, hq, 2, "chain")
    see = [D.visible(m, n, 0, 0) for n, m in zip(rows, [700, 90])]
    assert all(np.array_equal(a, b) for a, b in zip(see, c.sees(0, 0)))
    c.check(c.run())


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hq", [2, 32])
def test_positions_out_of_range(ctx, half, hq):
    """Positions count as no less than the first row's token and no more than the last's."""
    c = Case(ctx, 13, [200, 90], [9, 20], 16, 64, hq, 1, "tree")
    for value in (-2 ** 31, 0, 2 ** 31 - 1):
        c.position[:] = value
        c.pb.upload(c.position)
        c.check(c.run(half, 50, 3), half, 50, 3)


@pytest.mark.parametrize("rows,hq", [([4, 3], 2), ([25, 10], 2), ([80, 40], 4)])
@pytest.mark.parametrize("masks", [None, "tree", "any"])
def test_non_finite_places(ctx, rows, hq, masks):
    """NaN codes of hidden tokens leave a row alone, those of visible ones make the row, or that element of it, NaN."""
    window, sinks, lens = 40, 6, [250, 190]
    c = Case(ctx, 14, lens, rows, 16, 64, hq, 2, masks)
    kc, vc = c.kc.copy(), c.vc.copy()
    bad = {"v": [(0, 249 - rows[0] // 2, 5), (1, 20, 3), (0, 100, 60), (0, 3, 11), (1, 189, 9)],
           "k": [(1, 189 - rows[1] // 3, 9), (0, 5, 1), (0, 247, 3)]}
    for n, places in bad.items():
        for s, t, e in places:
            (c.vc if n == "v" else c.kc)[c.b.table[s, t // 16], :, t % 16, e] = 0xff
    got = c.run(window=window, sinks=sinks)
    see = c.sees(window, sinks)
    exp, tol = D.attend(kc, c.ks, vc, c.vs, c.b, c.q, c.scale, see)
    for s in range(2):
        for i in range(rows[s]):
            r = c.b.start[s] + i
            if any(z == s and see[s][i, t] for z, t, _ in bad["k"]):
                assert np.all(np.isnan(got[r]))
                continue
            good = np.ones(64, bool)
            good[[e for z, t, e in bad["v"] if z == s and see[s][i, t]]] = False
            assert np.all(np.isnan(got[r][:, ~good]))
            assert np.all(np.abs(got[r][:, good] - exp[r][:, good]) <= tol[r][:, good])


@pytest.mark.parametrize("masks,window,sinks,rows", [(None, 30, 4, [1, 2]), ("tree", 0, 0, [9, 5]), ("tree", 60, 20, [40, 70])])
def test_missing_pages_and_bounds(ctx, masks, window, sinks, rows):
    """Entries outside the pool hold no tokens, and tokens behind max_kv_len are not looked at."""
    c = Case(ctx, 15, [400, 300], rows, 16, 64, 4, 2, masks)
    c.b.table[0, 3], c.b.table[0, 24], c.b.table[1, 0] = -1, c.b.pages, -5
    c.check(c.run(window=window, sinks=sinks), window=window, sinks=sinks)
    c = Case(ctx, 16, [400, 300], rows, 16, 64, 4, 2, masks)
    got = c.run(window=window, sinks=sinks, max_len=333)
    c.b.lens = [333, 300]
    if masks:  # the windows count from positions inside the bounded sequence
        c.position = np.concatenate([np.minimum(c.position[:rows[0]], 332), c.position[rows[0]:]])
    c.check(got, window=window, sinks=sinks)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows,masks", [([1, 1], None), ([30, 20], "tree")])
def test_strided_rows(ctx, rows, masks, half):
    c = Case(ctx, 17, [900, 90], rows, 32, 128, 8, 2, masks)
    c.check(c.run(half, 100, 5, pad=9), half, 100, 5)


@pytest.mark.parametrize("masks,window,sinks", [(None, 300, 4), ("tree", 0, 0)])
def test_replayed_graph(ctx, masks, window, sinks):
    """One recorded call follows growing sequences, beside eager calls on another stream."""
    rows, lens = [7, 5], [900, 120]
    c = Case(ctx, 18, lens, rows, 64, 64, 4, 2, masks)
    c.upload()
    batch = c.b.upload(ctx)
    ws, ws2 = c.scratch(batch), c.scratch(batch)
    out, out2 = ctx.alloc(4 * 12 * 4 * 64), ctx.alloc(4 * 12 * 4 * 64)
    st, other = ctx.stream(), ctx.stream()
    with Capture(ctx, st) as cap:
        c.encode(HeadRows(out, 4, 256), ws, batch, False, window, sinks, st)
    for lens in ([900, 120], [840, 64], [512, 5], [900, 7]):
        c.b.lens = lens
        c.b.bufs[1].upload(np.array(lens, np.int32))
        out.upload(np.full(12 * 256, 7, np.float32))
        ctx.synchronize()
        cap.graph.launch(st)
        c.encode(HeadRows(out2, 4, 256), ws2, batch, False, window, sinks, other)
        st.synchronize()
        other.synchronize()
        c.raw, c.fill = out.download(np.float32).reshape(12, 4, 64), np.float32(7)
        c.check(c.raw.astype(np.float64), window=window, sinks=sinks)
        assert np.array_equal(c.raw, out2.download(np.float32).reshape(12, 4, 64))
    cap.graph.destroy()
    st.destroy()
    other.destroy()


def test_workspace_too_small(ctx):
    c = Case(ctx, 19, [5000], [1], 64, 64, 2, 1)
    c.upload()
    batch = c.b.upload(ctx)
    ws = ctx.alloc(c.kern.workspaceBytes(c.cache, batch, 2) - 4)
    out = HeadRows(ctx.alloc(4 * 128), 2, 128)
    with pytest.raises(EncodingFailed):
        c.encode(out, ws, batch, False, 1000, 4)
