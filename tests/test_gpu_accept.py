"""Acceptance of drafted tokens: the walk, and the cache that the kept ones
leave, code for code and scale for scale against a plain form."""
import numpy as np
import pytest

import draft_ref as D
import kv8_ref as R
from edgerunner_amd import Capture, Drafts, KV8AcceptKernel, KV8Cache

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, ctx, seed, lens, rows, P, d, heads, luck=0.8, tokens=1000, chain=False, behind=0, apart=3):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.heads, self.d = ctx, heads, d
        self.b = R.Batch(rng, lens, rows, P, behind=behind)
        shape = (self.b.pages, heads, P, d)
        self.before = []
        for _ in range(2):
            self.before += [rng.integers(0, 256, shape).astype(np.uint8),
                            (2.0 ** rng.integers(-apart, apart + 1, shape[:2])).astype(np.float32)]
        self.parent, self.token, self.chosen = (np.full(self.b.total, -9, np.int32) for _ in range(3))
        for s, n in enumerate(rows):
            at = slice(self.b.start[s], self.b.start[s] + n)
            self.parent[at], self.token[at] = D.tree(rng, n, tokens, chain) if n else ([], [])
            follow = rng.integers(0, tokens, n)
            for i in range(n):  # one of a row's children, mostly
                after = np.flatnonzero(self.parent[at] == i)
                if len(after) and rng.random() < luck:
                    follow[i] = self.token[at][rng.choice(after)]
            self.chosen[at] = follow

    def upload(self):
        ctx, b, S = self.ctx, self.b, len(self.b.lens)
        k, ks, v, vs = [ctx.upload(a) for a in self.before]
        self.bufs = [k, ks, v, vs]
        self.cache = KV8Cache(k, v, ks, vs, b.pages, self.heads, b.P, self.d)
        self.tree = [ctx.upload(a) for a in (self.parent, self.token, self.chosen)]
        self.drafts = Drafts(None, 0, parent=self.tree[0], token=self.tree[1])
        self.out = [ctx.upload(np.full(n, -77, np.int32)) for n in (b.total, S, S, S)]

    def encode(self, batch, stream=None):
        KV8AcceptKernel(self.ctx).encode(stream, self.cache, batch, self.drafts, self.tree[2], *self.out)

    def state(self):
        return [x.download(a.dtype).reshape(a.shape) for x, a in zip(self.bufs, self.before)], \
            [x.download(np.int32) for x in self.out]

    def expect(self, before=None):
        b, before = self.b, self.before if before is None else before
        path, count, after, left, paths = np.full(b.total, -77, np.int32), [], [], [], []
        for s, (n, m) in enumerate(zip(b.rows, b.lens)):
            at = slice(b.start[s], b.start[s] + n)
            line, t = D.walk(self.parent[at], self.token[at], self.chosen[at]) if n else ([], -1)
            path[at] = line + [-1] * (n - len(line))
            count.append(len(line))
            after.append(t)
            left.append(max(m - n + len(line), 0))
            paths.append(line)
        k, ks = D.accept(before[0], before[1], b, paths)
        v, vs = D.accept(before[2], before[3], b, paths)
        return [k, ks, v, vs], [path, np.array(count), np.array(after), np.array(left)]

    def check(self, got, exp):
        for x, y in zip(got[1], exp[1]):
            assert np.array_equal(x, y)
        for x, y in zip(got[0], exp[0]):
            # 0x7f and 0xff are both NaN
            if x.dtype == np.uint8:
                x, y = (np.where((z & 0x7f) == 0x7f, 0xff, z) for z in (x, y))
            assert np.array_equal(x, y), np.argwhere(x != y)[:5]

    def run(self):
        self.upload()
        self.encode(self.b.upload(self.ctx))
        self.ctx.synchronize()
        return self.state()


@pytest.mark.parametrize("d,P,heads", [(64, 16, 2), (64, 32, 1), (64, 64, 3), (128, 16, 1), (128, 32, 2), (128, 64, 1), (256, 16, 1),
                                       (256, 32, 2), (256, 64, 1)])
@pytest.mark.parametrize("lens,rows", [([70, 33, 0, 5, 130], [5, 8, 0, 5, 1]), ([150, 77, 0, 40], [64, 33, 0, 9]),
                                       ([331, 90], [60, 90]), ([64, 16, 17], [64, 16, 1])])
def test_trees(ctx, d, P, heads, lens, rows):
    c = Case(ctx, d + P + len(lens), lens, rows, P, d, heads, behind=2)
    c.check(c.run(), c.expect())


@pytest.mark.parametrize("luck,chain,tokens", [(1.0, False, 1000), (1.0, True, 1000), (0.0, False, 1000), (0.9, False, 2)])
def test_lucky_and_unlucky(ctx, luck, chain, tokens):
    """Everything kept, nothing but the first row, and so few tokens that siblings share them (the lowest is taken)."""
    c = Case(ctx, 3, [200, 300, 41], [40, 130, 41], 32, 64, 2, luck, tokens, chain)
    c.check(c.run(), c.expect())
    if chain:
        assert all(np.array_equal(a, b) for a, b in zip(c.state()[0], c.before))


def test_the_most_drafts(ctx):
    """Walks through rows that a wave takes 64 at a time, and moves over many pages."""
    c = Case(ctx, 4, [1500, 1024, 700], [1024, 1024, 300], 16, 64, 1, 1.0)
    for s in range(3):  # a path that leaves out every third row
        n, at = c.b.rows[s], c.b.start[s]
        line = [r for r in range(n) if r % 3 != 1]
        for a, r in zip(line, line[1:]):
            c.parent[at + r], c.chosen[at + a] = a, c.token[at + r]
    got = c.run()
    assert got[1][1].min() > 64
    c.check(got, c.expect())


def test_scales_far_apart(ctx):
    c = Case(ctx, 5, [100, 90, 80], [40, 50, 60], 16, 64, 2, 1.0, apart=30)
    c.check(c.run(), c.expect())


@pytest.mark.parametrize("lens,rows", [([33, 5, 2], [33, 9, 70]), ([1, 0, 3], [1, 4, 2])])
def test_no_tokens_in_front(ctx, lens, rows):
    """Trees that begin a sequence, and rows in front of the first token, which have no place."""
    c = Case(ctx, 6, lens, rows, 16, 64, 1, 1.0)
    c.check(c.run(), c.expect())


def test_missing_pages(ctx):
    """A token whose place or whose former place has no page is left out."""
    for s in range(8):
        c = Case(ctx, 7 + s, [100, 90], [60, 80], 16, 64, 2, 1.0)
        c.b.table[0, 3 + s % 4], c.b.table[1, 1 + s % 5] = -1, c.b.pages + s
        c.check(c.run(), c.expect())


def test_zeros_and_odd_tokens(ctx):
    """Codes of zeros move too; a negative choice ends a walk, wherever a draft holds the same."""
    c = Case(ctx, 20, [60, 50], [40, 30], 16, 64, 1, 1.0)
    for i in (0, 2):
        c.before[i][:] = np.where(c.rng.random(c.before[i].shape) < 0.5, 0x80, 0)
    c.token[c.b.start[1]:] = -5
    c.chosen[c.b.start[1]:] = -5
    got = c.run()
    assert got[1][1][1] == 1 and got[1][2][1] == -5
    c.check(got, c.expect())


def test_many_sequences(ctx):
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(1, 300, 150)]
    rows = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, 70, 150))]
    c = Case(ctx, 9, lens, rows, 32, 64, 2, behind=3)
    c.check(c.run(), c.expect())


def test_replayed_graph(ctx):
    """A recorded call follows other trees and lengths."""
    rows = [12, 0, 30]
    c = Case(ctx, 10, [100, 7, 130], rows, 32, 128, 2)
    c.upload()
    batch = c.b.upload(ctx)
    st = ctx.stream()
    with Capture(ctx, st) as cap:
        c.encode(batch, st)
    for i, lens in enumerate(([100, 7, 130], [90, 0, 129], [12, 7, 64])):
        other = Case(ctx, 30 + i, [100, 7, 130], rows, 32, 128, 2)
        c.parent, c.token, c.chosen, c.b.lens = other.parent, other.token, other.chosen, lens
        for x, a in zip(c.tree, (c.parent, c.token, c.chosen)):
            x.upload(a)
        c.b.bufs[1].upload(np.array(lens, np.int32))
        before = c.state()[0]
        ctx.synchronize()
        cap.graph.launch(st)
        st.synchronize()
        c.check(c.state(), c.expect(before))
    cap.graph.destroy()
    st.destroy()
