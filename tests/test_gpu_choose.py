"""Rules on logits and the choice against a plain 64-bit form.  A value that a rule changes is rounded once, so it is off by at
most half a step of fp32 of itself (the plain form's own 64-bit rounding adds 2^-50 of its terms, at most 2^-20 of a half step
where they cancel by less than 2^5; cancelling terms are held to 2^-50 of the largest)."""
import numpy as np
import pytest

import draft_ref as D
from edgerunner_amd import Capture, Drafts, LogitChoiceKernel, LogitRules

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, ctx, seed, vocab, rows, past=0, bias=0, allowed=False, tree=False, behind=0, penalty=None, mapped=True,
                 stride=None):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.vocab, self.rows, self.mapped = ctx, vocab, list(rows), mapped
        S, R = len(rows), sum(rows)
        self.start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.total, self.stride = R + behind, stride or vocab
        self.x = (rng.standard_normal((self.total, self.stride)) * 3).astype(np.float32)
        self.penalty = self.history = self.bias = self.allowed = self.seen = None
        if past or tree:
            self.penalty = np.stack([rng.uniform(1, 1.5, S), rng.uniform(-0.2, 1, S), rng.uniform(0, 0.3, S)], 1).astype(np.float32)
            if penalty is not None:
                self.penalty[:] = penalty
        if past:
            # tokens twice and more often, some outside the vocabulary
            self.history = (rng.random((S, past)) ** 3 * (vocab + 2) - 1).astype(np.int32)
            self.past_len = rng.integers(0, past + 1, S).astype(np.int32)
            self.past_len[0] = past
        if bias:
            self.bias_token = rng.integers(-1, min(vocab + 1, 2 * bias), (S, bias)).astype(np.int32)
            self.bias = rng.standard_normal((S, bias)).astype(np.float32) * 4
            self.bias_len = rng.integers(0, bias + 1, S).astype(np.int32)
            self.bias_len[-1] = bias
        if allowed:
            self.allowed = rng.random((self.total, vocab)) < rng.choice([0.01, 0.4, 0.95], (self.total, 1))
            self.allowed[2::5] = False
        if tree:
            self.token = rng.integers(0, vocab, self.total).astype(np.int32)
            most = max(rows)
            self.n_words = -(-most // 32) + 1
            self.seen, packed = [], np.full((self.total, self.n_words), 0xffffffff, np.uint32)
            for s, n in enumerate(rows):
                bits = D.lines(D.tree(rng, n)[0]) if n else np.zeros((0, 0), bool)
                self.seen.append(bits)
                packed[self.start[s]:self.start[s] + n] = D.words(bits, self.n_words)
            self.packed = packed

    def upload(self):
        up, S = self.ctx.upload, len(self.rows)
        self.kern = LogitChoiceKernel(self.ctx)
        self.keep = {}
        if self.penalty is not None:
            self.keep["penalty"] = up(self.penalty)
        if self.history is not None:
            self.keep |= {"history": up(self.history), "historyLen": up(self.past_len), "historyStride": self.history.shape[1]}
        if self.bias is not None:
            self.keep |= {"biasToken": up(self.bias_token), "bias": up(self.bias), "biasLen": up(self.bias_len),
                          "biasStride": self.bias.shape[1]}
        if self.allowed is not None:
            w = D.words(self.allowed)
            self.keep |= {"allowed": up(w), "allowedStride": w.shape[1]}
        where = (up(self.start), S, max(self.rows)) if self.mapped else (None, 0, 0)
        self.rules = LogitRules(*where, **self.keep)
        self.drafts = Drafts(up(self.packed), self.n_words, token=up(self.token)) if self.seen is not None else None
        self.xb = up(self.x)
        self.ws = self.ctx.alloc(self.kern.workspaceBytes(self.total, self.vocab))
        self.ws.upload(np.full(self.ws.length // 4, 0x7f800001, np.uint32))  # whatever scratch holds must not matter
        self.cb = up(np.full(self.total, -55, np.int32))
        self.ob = up(np.full((self.total, self.stride), 7, np.float32))

    def encode(self, out=True, chosen=True, stream=None, place=None):
        self.kern.encode(stream, self.xb, self.total, self.vocab, self.rules, drafts=self.drafts,
                         out=place or (self.ob if out else None), chosen=self.cb if chosen else None,
                         workspace=self.ws if chosen else None, rowStride=self.stride)

    def row(self, s, i):
        r = self.start[s] + i
        context = list(self.history[s, :self.past_len[s]]) if self.history is not None else []
        if self.seen is not None:
            context += [self.token[self.start[s] + j] for j in np.flatnonzero(self.seen[s][i])]
        bias = list(zip(self.bias_token[s], self.bias[s]))[:self.bias_len[s]] if self.bias is not None else ()
        return D.choose(self.x[r, :self.vocab], context, None if self.penalty is None else self.penalty[s], bias,
                        None if self.allowed is None else self.allowed[r])

    def check(self, out=True, chosen=True, place=None, behind=7.0):
        got = (place or self.ob).download(np.float32).reshape(self.total, self.stride)
        picks = self.cb.download(np.int32)
        of = np.full(self.total, -1)
        for s, n in enumerate(self.rows):
            for i in range(n):
                r = self.start[s] + i
                of[r] = s
                y, pick = self.row(s, i)
                if chosen:
                    assert picks[r] == pick, (r, picks[r], pick)
                if out:
                    g = got[r, :self.vocab].astype(np.float64)
                    fin = np.isfinite(y)
                    assert np.array_equal(np.isnan(g), np.isnan(y)) and np.array_equal(g[~fin & ~np.isnan(y)], y[~fin & ~np.isnan(y)])
                    big = np.abs(np.where(np.isfinite(self.x[r, :self.vocab]), self.x[r, :self.vocab], 0)) + 64
                    g, y, big = g[fin], y[fin], big[fin]
                    assert np.all(np.abs(g - y) <= D.U24 * (1 + 2.0 ** -20) * np.abs(y) + 2.0 ** -50 * big)
        assert np.all(picks[of < 0] == -55)
        if out:
            assert place or np.all(got[of < 0] == behind)
            assert place or np.all(got[:, self.vocab:] == behind)

    def run(self, **kw):
        self.upload()
        self.encode(**kw)
        self.ctx.synchronize()
        self.check(**kw)


VOCABS = [1, 3, 31, 32, 33, 1000, 1023, 1024, 1025, 4097, 32003]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("kind", [{}, {"past": 50}, {"bias": 9}, {"allowed": True}, {"past": 300, "bias": 40, "allowed": True},
                                  {"tree": True, "past": 20, "allowed": True}, {"tree": True}])
def test_rules(ctx, vocab, kind):
    rows = [5, 0, 33, 1] if kind.get("tree") else [1, 1, 0, 1, 2]
    Case(ctx, vocab, vocab, rows, behind=2, **kind).run()


@pytest.mark.parametrize("out,chosen", [(False, True), (True, False)])
@pytest.mark.parametrize("vocab", [777, 9001])
def test_one_output(ctx, vocab, out, chosen):
    Case(ctx, 2, vocab, [1, 3], past=40, bias=5, allowed=True).run(out=out, chosen=chosen)


@pytest.mark.parametrize("rows", [1, 7, 300])
def test_row_a_sequence(ctx, rows):
    Case(ctx, rows, 2050, [1] * rows, past=30, bias=3, allowed=True, mapped=False).run()


@pytest.mark.parametrize("rows,vocab", [(2, 128256), (70, 32000), (700, 5003)])
def test_sizes_of_slices(ctx, rows, vocab):
    """Few and many rows take slices of other lengths."""
    c = Case(ctx, rows, vocab, [1] * rows, past=200, bias=20, allowed=True)
    c.run()


def test_strided_and_in_place(ctx):
    c = Case(ctx, 5, 1001, [2, 3], past=20, allowed=True, stride=1007)
    c.run()
    c.upload()
    c.encode(place=c.xb)
    ctx.synchronize()
    c.check(place=c.xb)
    assert np.array_equal(c.xb.download(np.float32).reshape(c.x.shape)[:, 1001:], c.x[:, 1001:])


def test_no_rules(ctx):
    """Values keep their bits, the largest is chosen, ties go to the lowest token."""
    c = Case(ctx, 6, 5000, [1, 1, 1])
    c.x[0] = np.round(c.x[0])
    c.x[1] = -np.inf
    c.x[2, 17:] = np.float32(-0.0)
    c.x[2, :17] = -1
    c.upload()
    c.rules = None
    c.encode()
    ctx.synchronize()
    assert np.array_equal(c.ob.download(np.uint32).reshape(3, -1), c.x.view(np.uint32))
    assert list(c.cb.download(np.int32)) == [int(c.x[0].argmax()), 0, 17]


def test_penalties_that_change_nothing(ctx):
    c = Case(ctx, 7, 3000, [1, 2], past=100, penalty=(1.0, 0.0, 0.0))
    c.run()
    assert np.array_equal(c.ob.download(np.uint32).reshape(3, -1), c.x.view(np.uint32))


def test_non_finite(ctx):
    """NaN is never taken, infinities follow the formula, and what the mask hides does not count whatever it is."""
    c = Case(ctx, 8, 2000, [1] * 6, past=60, bias=20, allowed=True)
    c.x[:, ::7], c.x[1, ::3], c.x[2, 5:] = np.nan, np.inf, -np.inf
    c.x[3] = np.nan
    c.x[5] = -np.inf
    c.allowed[3:] = True
    c.run()
    assert c.cb.download(np.int32)[3] == -1 and c.cb.download(np.int32)[2] in (-1, *range(2000))


def test_nothing_left(ctx):
    c = Case(ctx, 9, 4500, [2, 1], past=10, allowed=True)
    c.allowed[:] = False
    c.run()
    assert np.all(c.cb.download(np.int32) == -1)
    # the one token that is allowed is chosen, whatever it is worth, and bits behind the vocabulary are not read
    c.allowed[:, 4499] = True
    c.x[:, 4499] = -np.inf
    c.run()
    assert np.all(c.cb.download(np.int32) == 4499)


def test_same_token_many_times(ctx):
    c = Case(ctx, 10, 300, [1, 1], past=5000, bias=50)
    c.history[:], c.bias_token[:] = 7, 7
    c.run()


def test_list_lengths_are_bounded(ctx):
    c = Case(ctx, 11, 600, [1, 1, 1], past=30, bias=8)
    c.upload()
    c.keep["historyLen"].upload(np.array([2 ** 31 - 1, -4, 30], np.int32))
    c.keep["biasLen"].upload(np.array([-1, 2 ** 31 - 1, 8], np.int32))
    c.encode()
    ctx.synchronize()
    c.past_len, c.bias_len = np.array([30, 0, 30]), np.array([0, 8, 8])
    c.check()


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 2046, 2047, 2048, 2049, 2050, 2051, 2052, 4095])
@pytest.mark.parametrize("past,bias", [(9001, 700), (4097, 300), (5, 3)])
def test_lengths_of_lists(ctx, vocab, past, bias):
    """Lists that end anywhere in a group of four, have more entries than a slice has threads, or fewer than four."""
    c = Case(ctx, vocab + past, vocab, [1] * 12, past=past, bias=bias, allowed=vocab > 2047)
    ends = [past - i for i in range(4)] + [0, 1, 2, 3, 4, 5, min(1024, past), min(4096, past)]
    c.past_len[:] = [max(n, 0) for n in ends]
    c.bias_len[:] = [bias - i % 3 for i in range(6)] + [0, 1, 2, 3, min(256, bias), min(257, bias)]
    c.run()


def test_logits_beyond_32_bits(ctx):
    """Rows whose offsets pass 2^32 bytes, in place."""
    vocab, stride, n = 5003, 1 << 26, 18
    c = Case(ctx, 12, vocab, [1] * n, past=40, bias=9, allowed=True)
    c.upload()
    far = ctx.alloc(4 * ((n - 1) * stride + vocab))
    for r in range(n):
        far.upload(c.x[r], 4 * r * stride)
    c.kern.encode(None, far, n, vocab, c.rules, out=far, chosen=c.cb, workspace=c.ws, rowStride=stride)
    ctx.synchronize()
    for r in range(n):
        c.ob.upload(far.download(np.float32, vocab, 4 * r * stride), 4 * r * vocab)
    c.check()
    far.free()


@pytest.mark.parametrize("tree", [False, True])
def test_replayed_graph(ctx, tree):
    """A recorded call follows later histories, masks and logits, beside eager calls with a workspace of their own."""
    c = Case(ctx, 12, 5001, [3, 2], past=40, bias=6, allowed=True, tree=tree)
    c.upload()
    st = ctx.stream()
    with Capture(ctx, st) as cap:
        c.encode(stream=st)
    for i in range(4):
        c.x[:] = c.rng.standard_normal(c.x.shape).astype(np.float32) * 3
        c.past_len[:] = [i * 13, 40 - i]
        c.allowed[:] = c.rng.random(c.allowed.shape) < 0.3
        c.xb.upload(c.x)
        c.keep["historyLen"].upload(c.past_len)
        c.keep["allowed"].upload(D.words(c.allowed))
        ctx.synchronize()
        cap.graph.launch(st)
        eager = Case(ctx, 20 + i, 3001, [1, 1], past=10)
        eager.run()
        st.synchronize()
        c.check()
    cap.graph.destroy()
    st.destroy()
