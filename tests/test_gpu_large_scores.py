"""Attention where scores are so large that fp32's steps are no longer small beside the powers of two that weights are
taken in.  A query has one element that is not 0, so tokens with the same key code there have exactly the same score, and the
others, an eighth lower at the least, weigh nothing: the output is the mean of the values of the tokens that have the largest.

The bound: a weight and its sum are off by an exponential (2^-22), one or two fp16 terms (2^-11, 2^-22) and the sums' and
quotients' fp32 roundings, 2 (m + 8) of 2^-24 over m tokens, and a bf16 output by half its step, 2^-8."""
import numpy as np
import pytest

import draft_ref as D
import kv8_ref as R
from edgerunner_amd import HeadRows
from test_gpu_masked_attention import Case

pytestmark = pytest.mark.gpu


def expected(c, see, half):
    exp, tol = np.zeros(c.q.shape), np.zeros(c.q.shape)
    G = c.hq // c.kc.shape[1]
    for s, (n, m) in enumerate(zip(c.b.rows, c.b.lens)):
        for hk in range(c.kc.shape[1]):
            K, _ = R.read(c.kc, c.ks, c.b, s, hk)
            V, _ = R.read(c.vc, c.vs, c.b, s, hk)
            for i in range(n):
                r = c.b.start[s] + i
                for h in range(hk * G, hk * G + G):
                    e = int(np.flatnonzero(c.q[r, h])[0])
                    score = K[:, e] * np.sign(c.q[r, h, e])
                    best = see[s][i] & (score == score[see[s][i]].max())
                    exp[r, h] = V[best].mean(0)
                    tol[r, h] = (2 * 2.0 ** -22 + (2.0 ** -11 if half else 2.0 ** -22) + 2 * (m + 8) * 2.0 ** -24) * np.abs(V[best]).mean(0)
    return exp, tol + (2.0 ** -8 * np.abs(exp) * (1 + 1e-6) if half else 0.0)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("first,last", [(20, 24), (24, 28), (28, 32), (60, 64)])
@pytest.mark.parametrize("d,P,hq,hkv,lens,rows,masks", [
    (64, 16, 4, 2, [300, 70], [3, 1], None), (128, 32, 4, 2, [700, 90], [12, 5], "tree"), (256, 64, 2, 1, [900, 130], [20, 7], "any"),
    (128, 16, 8, 8, [8200] + [100] * 31, [17] + [2] * 31, None), (64, 64, 16, 2, [400, 200], [90, 33], "tree"),
    (128, 64, 4, 1, [500, 64], [200, 64], None), (256, 16, 4, 1, [300, 200], [80, 20], "any")])
def test_large_scores(ctx, d, P, hq, hkv, lens, rows, masks, first, last, half):
    """Scores of 2^first to 2^last and above, in powers of two, under masks, and of causal rows without them too."""
    c = Case(ctx, d + P + first, lens, rows, P, d, hq, hkv, masks)
    # keys between 16 and 30 in steps of 2, of either sign, so that the largest is seen soon and often; a page's scale is 1
    c.kc[:] = np.where(c.kc == 0x7f, c.kc, c.rng.integers(0x58, 0x60, c.kc.shape) | c.rng.integers(0, 2, c.kc.shape) << 7)
    c.ks[:] = np.where(np.isnan(c.ks), c.ks, 1.0)
    at = c.rng.integers(0, d, c.q.shape[:2] + (1,))
    size = 2.0 ** c.rng.uniform(first - 4, last - 4, c.q.shape[:2]) / (c.scale * 1.4427)
    c.q[:] = 0
    np.put_along_axis(c.q, at, (size * c.rng.choice([-1, 1], size.shape)).astype(np.float32)[..., None], 2)
    see = [x.copy() for x in c.sees(0, 0)]
    if masks == "any":  # every row sees something, and something it does not
        for s in range(len(lens)):
            assert see[s].any(1).all() or lens[s] == rows[s]
    exp, tol = expected(c, see, half)
    calls = [c.run(half, 0, max(lens))]
    if masks is None:
        out = ctx.upload(np.zeros(c.q.shape, np.uint16 if half else np.float32))
        batch = c.b.upload(ctx)
        c.kern.encode(None, c.cache, batch, c.qr, HeadRows(out, hq, hq * d), c.scale, workspace=c.scratch(batch), outBF16=half)
        ctx.synchronize()
        raw = out.download(np.uint16 if half else np.float32).reshape(c.q.shape)
        calls.append((R.bf16_to_f32(raw) if half else raw).astype(np.float64))
    for got in calls:
        assert not np.isnan(got).any(), np.argwhere(np.isnan(got))[:3]
        assert np.all(np.abs(got - exp) <= tol), float((np.abs(got - exp) / np.maximum(tol, 1e-300)).max())
