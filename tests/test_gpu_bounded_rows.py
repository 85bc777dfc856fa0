"""max_rows below what a sequence has: the rows beyond it are left alone, and positions, drafts and walks count from the rest."""
import numpy as np
import pytest

from edgerunner_amd import HeadRows, LogitRules
from test_gpu_accept import Case as Accept
from test_gpu_choose import Case as Choose
from test_gpu_masked_attention import Case as Attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("masks,window,sinks", [(None, 30, 5), ("tree", 0, 0), ("any", 25, 3)])
@pytest.mark.parametrize("most,hq", [(1, 2), (7, 4), (33, 16)])
def test_attention(ctx, masks, window, sinks, most, hq):
    c = Attend(ctx, most + hq, [200, 90, 1400], [40, 5, 70], 16, 64, hq, 2, masks, behind=2)
    c.upload()
    batch = c.b.upload(ctx, max_rows=most)
    out = ctx.upload(np.full(c.q.shape, 7, np.float32))
    c.encode(HeadRows(out, hq, hq * 64), c.scratch(batch), batch, False, window, sinks)
    ctx.synchronize()
    c.raw, c.fill = out.download(np.float32).reshape(c.q.shape), np.float32(7)
    c.b.rows = [min(n, most) for n in c.b.rows]
    c.check(c.raw.astype(np.float64), window=window, sinks=sinks)


@pytest.mark.parametrize("most", [1, 6, 40, 70])
def test_acceptance(ctx, most):
    c = Accept(ctx, most, [200, 90, 140], [40, 5, 90], 16, 64, 2, 1.0, behind=2)
    c.upload()
    c.encode(c.b.upload(ctx, max_rows=most))
    ctx.synchronize()
    c.b.rows = [min(n, most) for n in c.b.rows]
    c.check(c.state(), c.expect())


@pytest.mark.parametrize("most", [1, 6, 33])
def test_rules(ctx, most):
    c = Choose(ctx, most, 3000, [40, 5, 0, 36], past=30, allowed=True, tree=True, behind=2)
    c.upload()
    c.rules = LogitRules(ctx.upload(c.start), 4, most, **c.keep)
    c.encode()
    ctx.synchronize()
    c.rows, seen = [min(n, most) for n in c.rows], c.seen
    c.seen = [s[:n, :n] for s, n in zip(seen, c.rows)]
    c.check()
