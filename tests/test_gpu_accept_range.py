"""Acceptance of drafts at the ends of its range: values next to fp32's largest,
and pages that are missing in front of ones that are there."""
import numpy as np
import pytest

from test_accept_schedule import near_the_largest
from test_gpu_accept import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("whole", [False, True])
@pytest.mark.parametrize("scales", [[120], [118, 119, 120], [-100, 0, 120]])
@pytest.mark.parametrize("d,P", [(64, 16), (64, 64), (128, 32), (256, 16)])
def test_values_past_fp32(ctx, d, P, scales, whole):
    c = near_the_largest(70 + d, P, d, scales, whole)
    c.ctx = ctx
    c.check(c.run(), c.expect())


@pytest.mark.parametrize("d,P,heads", [(64, 16, 2), (128, 16, 1), (256, 32, 2), (64, 64, 1)])
def test_pages_around_gaps(ctx, d, P, heads):
    """Every other page of the drafts' places has none in the pool."""
    for odd in (0, 1):
        c = Case(ctx, d + P + odd, [11 * P - 3, 6 * P], [9 * P, 5 * P], P, d, heads, 1.0, chain=True)
        for s, n in enumerate(c.b.rows):
            at = c.b.start[s]
            line = [0] + [r for r in range(2, n)]
            for a, r in zip(line, line[1:]):
                c.parent[at + r], c.chosen[at + a] = a, c.token[at + r]
            c.parent[at + 1] = -1
            c.b.table[s, 1 + odd::2] = -1
        exp = c.expect()
        assert list(exp[1][1]) == [9 * P - 1, 5 * P - 1]
        c.check(c.run(), exp)


@pytest.mark.parametrize("max_len", [None, 20])
def test_idle_sequences(ctx, max_len):
    """A batch without a single row: what an earlier step left in counts, tokens and lengths does not stay."""
    c = Case(ctx, 3, [33, 0, 5], [0, 0, 0], 16, 64, 2, behind=4)
    c.upload()
    full = c.b.upload(ctx, max_len=max_len)
    c.b.total = 0
    idle = c.b.upload(ctx, max_rows=0, max_len=max_len)
    for batch in (full, idle):
        for x in c.out:
            x.upload(np.full(x.length // 4, -77, np.int32))
        c.encode(batch)
        ctx.synchronize()
        cache, (path, count, after, left) = c.state()
        assert np.all(path == -77) and list(count) == [0, 0, 0] and list(after) == [-1, -1, -1]
        assert list(left) == [min(33, max_len or 33), 0, 5]
        assert all(np.array_equal(a, b) for a, b in zip(cache, c.before))
